// paged_evict.hip -- which positions a paged cache keeps, and whose pages a beam writes to (gfx950).
//
// Eviction.  Of a sequence's L > keep positions a kv head keeps the first `first`, the last
// `recent` and the m = keep - first - recent heaviest between them: those above the m-th largest
// weight T, and of those equal to T the first.  Weights are compared as integers of the same order
// (f32_key), T is found digit by digit from histograms.
//
// Kept positions move towards the front of the same pages, k-th to place k, from places that are not before
// it.  Where one block moves a kv head's rows, chunk after chunk, it reads a chunk before it
// writes it, and nothing is lost.  Blocks of their own for parts of them could overwrite each
// other's: long sequences' rows go to the workspace first, as images of the pages they will lie in.
#include <algorithm>

#include "paged_kv.hpp"
#include "topk_select.hpp"

namespace kh {

constexpr int kEvThreads = 1024;
constexpr int kEvDigit = 11;          // bits of a histogram
constexpr int kEvBins = 1 << kEvDigit;
constexpr int kEvPart = 4096;         // positions of a part of a long sequence
constexpr int kEvEach = kEvPart / kEvThreads;
constexpr int kEvMost = 16;           // weights of a thread where a block has a whole sequence's

struct EvictArgs {
  char* pool;
  int64_t block, pages;
  int nkv, ps_log2;
  int* err;
  const float* acc;
  int64_t acc_cols;
  const int64_t* len;
  const int32_t* table;
  int64_t cols, table_stride, batch, keep;
  int recent, first;
  int32_t* kept;
  float* acc_out;
  int64_t* len_out;
  // long sequences: images of the pages that the kept positions will lie in, their weights,
  // histograms of parts, and what each part begins with
  char* images;
  float* weights;
  uint16_t* hist;
  int* state;  // [batch][kv heads][2 + 2 parts]: T, the ties that are kept; kept above T and ties before each part
  int num_images, parts;
  int64_t wcols;  // weights of a kv head
};

// Positions of sequence b that weights and table reach.
__device__ __forceinline__ int64_t evict_len(const EvictArgs& a, int64_t b, bool tell) {
  const int64_t L = a.len[b], cap = min(a.acc_cols, a.cols << a.ps_log2);
  if (L >= 0 && L <= cap) return L;
  if (tell) atomicOr(a.err, 1);
  return L < 0 ? 0 : cap;
}

__device__ __forceinline__ uint32_t evict_key(float w) { return w != w ? 0xffffffffu : f32_key(w); }

// ---------------------------------------------------------------- a block a kv head
// Where position k of the kept ones comes from: its block and place; the place itself where its page is
// none of the pool (it does not move); nullptr where that is none either.
struct EvictFrom {
  const char* blk;
  int at;
};
__device__ __forceinline__ EvictFrom evict_from(const EvictArgs& a, const int32_t* __restrict__ table, int h, int from, int to) {
  int pg = table[from >> a.ps_log2], at = from;
  if (pg < 0 || pg >= a.pages) {
    atomicOr(a.err, 2);
    at = to;
    pg = table[to >> a.ps_log2];
  }
  EvictFrom x;
  x.blk = pg < 0 || pg >= a.pages ? nullptr : a.pool + ((int64_t)pg * a.nkv + h) * a.block;
  x.at = at & ((1 << a.ps_log2) - 1);
  return x;
}

// A value's codes of row r (of sixteen) of four positions, from the positions that the four
// come from: words [position / 2][h] with a position in each half.
template <int D, typename F>
__device__ __forceinline__ void evict_quad(int ps, int r, F from, uint32_t (&y)[D / 32]) {
  constexpr int HN = D / 64;
#pragma unroll
  for (int i = 0; i < 2 * HN; ++i) y[i] = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const EvictFrom x = from(e);
    if (!x.blk) continue;
    const uint32_t* w = reinterpret_cast<const uint32_t*>(x.blk + KvParts<D>::vc(ps) + (x.at >> 2) * (2 * D)) + r * (2 * HN) + (x.at >> 1 & 1) * HN;
#pragma unroll
    for (int hf = 0; hf < HN; ++hf) {
      const uint32_t u = x.at & 1 ? w[hf] >> 16 : w[hf] & 0xffffu;
      y[(e >> 1) * HN + hf] |= e & 1 ? u << 16 : u;
    }
  }
}

// Moves the kept positions k0 .. n - 1 of a kv head (n of them, s_kept[k] >= k), keys (what 1) or values
// (2) or both (3).  s_from: of a chunk.
constexpr int kEvChunk = kEvThreads;
template <int D>
__device__ __forceinline__ void evict_move(const EvictArgs& a, int64_t b, int h, int n, int k0, int what, const uint16_t* s_kept,
                                           EvictFrom* s_from) {
  using P = KvParts<D>;
  constexpr int NG = P::NG, HN = D / 64;
  const int ps = 1 << a.ps_log2, t = threadIdx.x;
  const int32_t* __restrict__ table = a.table + b * a.table_stride;
  // place k of the chunk, or nullptr
  const auto place = [&](int k, int& at) -> char* {
    const int pg = table[k >> a.ps_log2];
    at = k & (ps - 1);
    return pg < 0 || pg >= a.pages ? nullptr : a.pool + ((int64_t)pg * a.nkv + h) * a.block;
  };
  for (int c0 = k0 & ~3; c0 < n; c0 += kEvChunk) {
    const int c1 = min(c0 + kEvChunk, n), quads = (c1 - c0 + 3) >> 2;
    // the last quad's positions past the kept ones keep what they hold
    const int k = c0 + t;
    if (t < 4 * quads) s_from[t] = evict_from(a, table, h, k < c1 ? s_kept[k] : k, k);
    __syncthreads();
    if (what & 1) {
      constexpr int KC = D / 32;  // 16-byte pieces of a key's codes
      uint4 c[KC];
      uint32_t p[NG];
#pragma unroll
      for (int r = 0; r < KC; ++r) {
        const int i = r * kEvChunk + t;
        if (i < (c1 - c0) * KC) {
          const EvictFrom x = s_from[i / KC];
          if (x.blk) c[r] = *reinterpret_cast<const uint4*>(x.blk + P::kc() + x.at * (D / 2) + i % KC * 16);
        }
      }
#pragma unroll
      for (int r = 0; r < NG; ++r) {
        const int i = r * kEvChunk + t;
        if (i < (c1 - c0) * NG) {
          const EvictFrom x = s_from[i / NG];
          if (x.blk) p[r] = *reinterpret_cast<const uint32_t*>(x.blk + P::kp(ps) + (x.at * NG + i % NG) * 4);
        }
      }
      __syncthreads();
#pragma unroll
      for (int r = 0; r < KC; ++r) {
        const int i = r * kEvChunk + t;
        if (i < (c1 - c0) * KC) {
          int at;
          char* y = place(c0 + i / KC, at);
          if (y && s_from[i / KC].blk) *reinterpret_cast<uint4*>(y + P::kc() + at * (D / 2) + i % KC * 16) = c[r];
        }
      }
#pragma unroll
      for (int r = 0; r < NG; ++r) {
        const int i = r * kEvChunk + t;
        if (i < (c1 - c0) * NG) {
          int at;
          char* y = place(c0 + i / NG, at);
          if (y && s_from[i / NG].blk) *reinterpret_cast<uint32_t*>(y + P::kp(ps) + (at * NG + i % NG) * 4) = p[r];
        }
      }
    }
    if (what & 2) {
      constexpr int Q = 4;  // (quad, r) tasks of a thread: 16 rows of a quarter of the chunk
      uint32_t v[Q][2 * HN], p[NG];
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int i = q * kEvChunk + t, quad = i >> 4;
        if (quad < quads) evict_quad<D>(ps, i & 15, [&](int e) { return s_from[quad * 4 + e]; }, v[q]);
      }
#pragma unroll
      for (int j = 0; j < NG; ++j)
        if (k < c1) {
          const EvictFrom x = s_from[t];
          if (x.blk) p[j] = *reinterpret_cast<const uint32_t*>(x.blk + P::vp(ps) + (j * ps + x.at) * 4);
        }
      __syncthreads();
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int i = q * kEvChunk + t, quad = i >> 4;
        if (quad < quads) {
          int at;
          char* y = place(c0 + quad * 4, at);
          if (y) {
            uint32_t* w = reinterpret_cast<uint32_t*>(y + P::vc(ps) + (at >> 2) * (2 * D)) + (i & 15) * (2 * HN);
#pragma unroll
            for (int e = 0; e < 2 * HN; ++e) w[e] = v[q][e];
          }
        }
      }
      if (k < c1) {
        int at;
        char* y = place(k, at);
        if (y && s_from[t].blk) {
#pragma unroll
          for (int j = 0; j < NG; ++j) *reinterpret_cast<uint32_t*>(y + P::vp(ps) + (j * ps + at) * 4) = p[j];
        }
      }
    }
    __syncthreads();
  }
}

// A sequence that is not cut: its weights, and its positions as they are; parts [j0, j1) of the columns.
__device__ __forceinline__ void evict_none(const EvictArgs& a, int64_t row, int64_t L, int64_t j0, int64_t j1, int t, int nt, float* out) {
  for (int64_t j = j0 + t; j < min(j1, a.keep); j += nt) a.kept[row * a.keep + j] = j < L ? (int32_t)j : -1;
  for (int64_t j = j0 + t; j < min(j1, L); j += nt) out[j] = a.acc[row * a.acc_cols + j];
}

// Block: one kv head of one sequence, its keys or values or both (halves 2: blockIdx.z says which, and the
// block of the keys writes what else there is).  Weights stay in registers, the kept positions in LDS.
template <int D>
__global__ __launch_bounds__(kEvThreads) void evict_kernel(EvictArgs a, int halves) {
  __shared__ TopkLds<kEvThreads> sh;
  __shared__ EvictFrom s_from[kEvChunk];
  extern __shared__ __align__(16) uint16_t s_kept[];  // [keep]
  const int h = blockIdx.x, t = threadIdx.x, what = halves == 1 ? 3 : blockIdx.z == 0 ? 1 : 2;
  for (int64_t b = blockIdx.y; b < a.batch; b += gridDim.y) {
    const int64_t L = evict_len(a, b, h == 0 && t == 0 && (what & 1));
    const int64_t row = b * a.nkv + h, left = min(L, a.keep);
    const float* acc = a.acc + row * a.acc_cols;
    float* out = a.acc_out + row * a.acc_cols;
    if ((what & 1) && h == 0 && t == 0) a.len_out[b] = left;
    if (L <= a.keep) {
      if (what & 1) {
        evict_none(a, row, L, 0, max(a.acc_cols, a.keep), t, kEvThreads, out);
        for (int64_t j = L + t; j < a.acc_cols; j += kEvThreads) out[j] = 0.0f;
      }
      continue;
    }
    const int n = (int)L - a.first - a.recent, m = (int)a.keep - a.first - a.recent, each = (n + kEvThreads - 1) / kEvThreads;
    const int i0 = t * each, cnt = min(max(n - i0, 0), each);
    __syncthreads();
    if (m > 0) {
      uint32_t key[kEvMost], mx = 0, mn = 0xffffffffu;
#pragma unroll
      for (int e = 0; e < kEvMost; ++e) {
        key[e] = 0;
        if (e < cnt) {
          key[e] = evict_key(acc[a.first + i0 + e]);
          mx = max(mx, key[e]);
          mn = min(mn, key[e]);
        }
      }
      for (int i = t; i < (1 << kTopkDigit); i += kEvThreads) sh.hist[i] = 0;
      if (t == 0) sh.s_ncand = 0;
      mx = wave_max_u32(mx);
      mn = wave_min_u32(mn);
      if ((t & 63) == 0) sh.wmax[t >> 6] = mx, sh.wmin[t >> 6] = mn;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kEvThreads / 64; ++w) mx = max(mx, sh.wmax[w]), mn = min(mn, sh.wmin[w]);
      uint32_t T;
      int ties, at;
      topk_threshold<kEvThreads, kEvMost>(key, cnt, i0, m, mx, mn, sh, T, ties);
      const uint32_t take = topk_select_mask<kEvThreads, kEvMost>(key, cnt, T, ties, sh, at);
#pragma unroll
      for (int e = 0; e < kEvMost; ++e)
        if (take >> e & 1) s_kept[a.first + at++] = (uint16_t)(a.first + i0 + e);
    }
    for (int j = t; j < a.first; j += kEvThreads) s_kept[j] = (uint16_t)j;
    for (int j = t; j < a.recent; j += kEvThreads) s_kept[a.keep - a.recent + j] = (uint16_t)(L - a.recent + j);
    if (t == 0) sh.s_kk = (int)a.keep;
    __syncthreads();
    // the first one that moves: k with kept[k] > k
    int moved = (int)a.keep;
    for (int k = t; k < a.keep; k += kEvThreads)
      if (s_kept[k] != k) moved = min(moved, k);
    moved = (int)wave_min_u32((uint32_t)moved);
    if ((t & 63) == 0) atomicMin(&sh.s_kk, moved);
    __syncthreads();
    moved = sh.s_kk;
    evict_move<D>(a, b, h, (int)a.keep, moved, what, s_kept, s_from);
    if (what & 1) {
      float w[kEvMost];
#pragma unroll
      for (int e = 0; e < kEvMost; ++e) {
        const int k = e * kEvThreads + t;
        if (k < a.keep) {
          w[e] = acc[s_kept[k]];
          a.kept[row * a.keep + k] = s_kept[k];
        }
      }
      __syncthreads();
#pragma unroll
      for (int e = 0; e < kEvMost; ++e) {
        const int k = e * kEvThreads + t;
        if (k < a.keep) out[k] = w[e];
      }
      for (int64_t j = a.keep + t; j < a.acc_cols; j += kEvThreads) out[j] = 0.0f;
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- long sequences
// Four neighbouring weights from j on, of which those in [lo, hi) are asked for.
__device__ __forceinline__ void evict_four(const float* __restrict__ w, int j, int lo, int hi, uint32_t (&key)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) key[e] = j + e >= lo && j + e < hi ? evict_key(w[j + e]) : 0;
}

// Histograms of the upper digit of every part's weights.
__global__ __launch_bounds__(256) void evict_hist_kernel(EvictArgs a) {
  __shared__ uint32_t s_hist[kEvBins];
  const int part = blockIdx.x, h = blockIdx.y, t = threadIdx.x;
  for (int64_t b = blockIdx.z; b < a.batch; b += gridDim.z) {
    const int64_t L = evict_len(a, b, false), row = b * a.nkv + h;
    if (L <= a.keep || (int64_t)part * kEvPart >= L) continue;
    __syncthreads();
    for (int i = t; i < kEvBins; i += 256) s_hist[i] = 0;
    __syncthreads();
    const int lo = max(part * kEvPart, a.first), hi = min((part + 1) * kEvPart, (int)L - a.recent);
    const float* acc = a.acc + row * a.acc_cols;
#pragma unroll
    for (int c = 0; c < kEvPart / 1024; ++c) {
      uint32_t key[4];
      const int j = part * kEvPart + (c * 256 + t) * 4;
      evict_four(acc, j, lo, hi, key);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (j + e >= lo && j + e < hi) atomicAdd(&s_hist[key[e] >> (32 - kEvDigit)], 1u);
    }
    __syncthreads();
    uint32_t* to = reinterpret_cast<uint32_t*>(a.hist + (row * a.parts + part) * kEvBins);
    for (int i = t; i < kEvBins / 2; i += 256) to[i] = s_hist[2 * i] | s_hist[2 * i + 1] << 16;
  }
}

// T from the histograms and two more digits, and what each part begins with.  Block: a kv head of a
// sequence.
__global__ __launch_bounds__(kEvThreads) void evict_threshold_kernel(EvictArgs a) {
  __shared__ uint32_t hist[kEvBins];
  __shared__ int wsum[kEvThreads / 64], total, s_kk;
  __shared__ uint32_t s_bin;
  const int h = blockIdx.x, t = threadIdx.x, lane = t & 63;
  for (int64_t b = blockIdx.y; b < a.batch; b += gridDim.y) {
    const int64_t L = evict_len(a, b, false), row = b * a.nkv + h;
    if (L <= a.keep) continue;
    const float* acc = a.acc + row * a.acc_cols;
    const int lo = a.first, hi = (int)L - a.recent, parts = (int)((L + kEvPart - 1) / kEvPart);
    int* state = a.state + row * (2 + 2 * a.parts);
    uint32_t T = 0xffffffffu, mask = 0;
    int kk = (int)a.keep - a.first - a.recent;
    if (kk > 0) {
      T = 0;
      const uint32_t* from = reinterpret_cast<const uint32_t*>(a.hist + row * a.parts * kEvBins);
      uint32_t x = 0, y = 0;
#pragma unroll 8
      for (int p = 0; p < parts; ++p) {
        const uint32_t w = from[p * (kEvBins / 2) + t];
        x += w & 0xffffu;
        y += w >> 16;
      }
      hist[2 * t] = x;
      hist[2 * t + 1] = y;
      __syncthreads();
      for (int shift = 32 - kEvDigit;;) {
        // the bin of the kk-th largest: thread t owns two bins, thread 0 the highest
        const int top = kEvBins - 1 - 2 * t;
        const int n1 = (int)hist[top], n0 = (int)hist[top - 1];
        const int above = block_excl_scan(n1 + n0, wsum, &total);
        if (above < kk && kk <= above + n1 + n0) {
          s_bin = kk <= above + n1 ? top : top - 1;
          s_kk = kk - above - (kk <= above + n1 ? 0 : n1);
        }
        __syncthreads();
        T |= s_bin << shift;
        mask |= (uint32_t)(kEvBins - 1) << shift;
        kk = s_kk;
        if (shift == 0) break;
        const int next = max(shift - kEvDigit, 0);  // the last digit has some bits twice: they are T's
        for (int i = t; i < kEvBins; i += kEvThreads) hist[i] = 0;
        __syncthreads();
        constexpr int U = 4;
        for (int c = lo / 4 * 4; c < hi; c += 4 * U * kEvThreads) {
          uint32_t key[U][4];
#pragma unroll
          for (int u = 0; u < U; ++u) evict_four(acc, c + (u * kEvThreads + t) * 4, lo, hi, key[u]);
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int j = c + (u * kEvThreads + t) * 4 + e;
              if (j >= lo && j < hi && (key[u][e] & mask) == T) atomicAdd(&hist[(key[u][e] >> next) & (kEvBins - 1)], 1u);
            }
        }
        T &= ~((uint32_t)(kEvBins - 1) << next);
        shift = next;
        __syncthreads();
      }
    }
    // what lies before each part: counts of a wave's parts, then sums
    for (int p = t >> 6; p < parts; p += kEvThreads / 64) {
      int gt = 0, eq = 0;
      const int l = max(p * kEvPart, lo), u = min((p + 1) * kEvPart, hi);
#pragma unroll 4
      for (int c = 0; c < kEvPart; c += 256) {
        uint32_t key[4];
        const int j = p * kEvPart + c + lane * 4;
        evict_four(acc, j, l, u, key);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool in = j + e >= l && j + e < u;
          gt += __popcll(__ballot(in && key[e] > T));
          eq += __popcll(__ballot(in && key[e] == T));
        }
      }
      if (lane == 0) state[2 + 2 * p] = gt, state[3 + 2 * p] = eq;
    }
    __syncthreads();
    if (t < 64) {
      int g0 = 0, e0 = 0;
      for (int c = 0; c < parts; c += 64) {
        const int p = c + lane;
        const int gt = p < parts ? state[2 + 2 * p] : 0, eq = p < parts ? state[3 + 2 * p] : 0;
        const int gi = wave_incl_scan(gt), ei = wave_incl_scan(eq);
        if (p < parts) state[2 + 2 * p] = g0 + gi - gt, state[3 + 2 * p] = e0 + ei - eq;
        g0 += __builtin_amdgcn_readlane(gi, 63);
        e0 += __builtin_amdgcn_readlane(ei, 63);
      }
      if (lane == 0) state[0] = (int)T, state[1] = (int)a.keep - a.first - a.recent > 0 ? kk : 0;
    }
    __syncthreads();
  }
}

// The kept positions of a part, and their weights.
__global__ __launch_bounds__(kEvThreads) void evict_select_kernel(EvictArgs a) {
  __shared__ uint32_t uwsum[kEvThreads / 64];
  const int part = blockIdx.x, h = blockIdx.y, t = threadIdx.x;
  const int64_t j0 = (int64_t)part * kEvPart;
  for (int64_t b = blockIdx.z; b < a.batch; b += gridDim.z) {
    const int64_t L = evict_len(a, b, part == 0 && h == 0 && t == 0), row = b * a.nkv + h;
    if (part == 0 && h == 0 && t == 0) a.len_out[b] = min(L, a.keep);
    float* weights = a.weights + row * a.wcols;
    if (L <= a.keep) {
      evict_none(a, row, L, j0, part + 1 == a.parts ? max(a.acc_cols, a.keep) : j0 + kEvPart, t, kEvThreads, weights);
      continue;
    }
    if (j0 >= L) continue;
    const int* state = a.state + row * (2 + 2 * a.parts);
    const uint32_t T = (uint32_t)state[0];
    const int ties = state[1], gt0 = state[2 + 2 * part], eq0 = state[3 + 2 * part];
    const float* acc = a.acc + row * a.acc_cols;
    int32_t* kept = a.kept + row * a.keep;
    const int lo = a.first, hi = (int)L - a.recent, j = (int)j0 + t * kEvEach;
    float w[kEvEach];
    uint32_t gt = 0, eq = 0;
#pragma unroll
    for (int e = 0; e < kEvEach; ++e) {
      w[e] = j + e < L ? acc[j + e] : 0.0f;
      const uint32_t k = evict_key(w[e]);
      const bool in = j + e >= lo && j + e < hi;
      gt |= (in && k > T ? 1u : 0u) << e;
      eq |= (in && k == T ? 1u : 0u) << e;
    }
    // both counts of a part stay below 2^16
    const uint32_t before = block_excl_scan_u32(__popc(gt) | __popc(eq) << 16, uwsum);
    int e0 = eq0 + (int)(before >> 16), k0 = lo + gt0 + (int)(before & 0xffffu) + min(e0, ties);
#pragma unroll
    for (int e = 0; e < kEvEach; ++e) {
      const bool tie = eq >> e & 1;
      int k = -1;
      if ((gt >> e & 1) || (tie && e0 < ties)) k = k0++;
      if (j + e < lo) k = j + e;
      if (j + e >= hi && j + e < L) k = (int)(a.keep - (L - (j + e)));
      e0 += tie ? 1 : 0;
      if (k >= 0) kept[k] = j + e, weights[k] = w[e];
    }
    __syncthreads();
  }
}

// The first n positions of a block of a page, to another one (or to an image of one); what lies
// behind them there stays.
template <int D>
__device__ __forceinline__ void copy_positions(char* __restrict__ to, const char* __restrict__ from, int n, int ps, int t, int nt) {
  using P = KvParts<D>;
  constexpr int NG = P::NG;
  const auto words = [&](int off, int count) {
    uint32_t* y = reinterpret_cast<uint32_t*>(to + off);
    const uint32_t* x = reinterpret_cast<const uint32_t*>(from + off);
    for (int i = t; i < count; i += nt) y[i] = x[i];
  };
  const auto pieces = [&](int off, int count) {
    uint4* y = reinterpret_cast<uint4*>(to + off);
    const uint4* x = reinterpret_cast<const uint4*>(from + off);
    for (int i = t; i < count; i += nt) y[i] = x[i];
  };
  pieces(P::kc(), n * (D / 32));
  pieces(P::vc(ps), (n >> 2) * (D / 8));
  words(P::kp(ps), n * NG);
#pragma unroll
  for (int j = 0; j < NG; ++j) words(P::vp(ps) + j * ps * 4, n);
  if (n & 3) {  // of the last four positions' codes: words [r][position / 2][h], a position in each half
    uint32_t* y = reinterpret_cast<uint32_t*>(to + P::vc(ps) + (n >> 2) * (2 * D));
    const uint32_t* x = reinterpret_cast<const uint32_t*>(from + P::vc(ps) + (n >> 2) * (2 * D));
    for (int i = t; i < D / 2; i += nt) {
      const int second = i / (D / 64) & 1, there = (n & 3) - 2 * second;
      if (there <= 0) continue;
      y[i] = there >= 2 ? x[i] : (y[i] & 0xffff0000u) | (x[i] & 0xffffu);
    }
  }
}

// Images of the pages that kept positions will lie in: image i of a kv head holds positions
// i ps .. of the kept ones.  Nothing moves in an image whose last position stays.
__device__ __forceinline__ int evict_image(const EvictArgs& a, int64_t row, int64_t L, int image) {
  const int ps = 1 << a.ps_log2;
  const int64_t first = (int64_t)image << a.ps_log2;
  if (L <= a.keep || first >= a.keep) return 0;
  const int n = (int)min((int64_t)ps, a.keep - first);
  return a.kept[row * a.keep + first + n - 1] == first + n - 1 ? 0 : n;
}

template <int D>
__global__ __launch_bounds__(256) void evict_gather_kernel(EvictArgs a) {
  using P = KvParts<D>;
  constexpr int NG = P::NG, HN = D / 64;
  __shared__ EvictFrom s_from[256];
  const int h = blockIdx.y, ps = 1 << a.ps_log2, t = threadIdx.x;
  for (int64_t bi = blockIdx.x; bi < a.batch * a.num_images; bi += gridDim.x) {
    const int64_t b = bi / a.num_images, row = b * a.nkv + h;
    const int image = (int)(bi - b * a.num_images), first = image << a.ps_log2;
    const int n = evict_image(a, row, evict_len(a, b, false), image);
    if (n == 0) continue;
    const int32_t* __restrict__ table = a.table + b * a.table_stride;
    __syncthreads();
    if (t < n) s_from[t] = evict_from(a, table, h, a.kept[row * a.keep + first + t], first + t);
    __syncthreads();
    char* to = a.images + (row * a.num_images + image) * a.block;
    constexpr int KC = D / 32;  // 16-byte pieces of a key
    for (int i = t; i < n * KC; i += 256) {
      const EvictFrom x = s_from[i / KC];
      if (x.blk) *reinterpret_cast<uint4*>(to + P::kc() + i * 16) = *reinterpret_cast<const uint4*>(x.blk + P::kc() + x.at * (D / 2) + i % KC * 16);
    }
    for (int i = t; i < n * NG; i += 256) {
      const EvictFrom x = s_from[i / NG];
      if (x.blk) *reinterpret_cast<uint32_t*>(to + P::kp(ps) + i * 4) = *reinterpret_cast<const uint32_t*>(x.blk + P::kp(ps) + (x.at * NG + i % NG) * 4);
    }
    for (int i = t; i < ps * NG; i += 256) {
      const int j = i >> a.ps_log2, k = i & (ps - 1);
      if (k >= n) continue;
      const EvictFrom x = s_from[k];
      if (x.blk) *reinterpret_cast<uint32_t*>(to + P::vp(ps) + i * 4) = *reinterpret_cast<const uint32_t*>(x.blk + P::vp(ps) + (j * ps + x.at) * 4);
    }
    for (int i = t; i < (n + 3) / 4 * 16; i += 256) {
      uint32_t v[2 * HN];
      evict_quad<D>(ps, i & 15, [&](int e) { return s_from[min((i >> 4) * 4 + e, n - 1)]; }, v);
      uint32_t* w = reinterpret_cast<uint32_t*>(to + P::vc(ps)) + i * (2 * HN);
#pragma unroll
      for (int e = 0; e < 2 * HN; ++e) w[e] = v[e];
    }
  }
}

template <int D>
__global__ __launch_bounds__(256) void evict_place_kernel(EvictArgs a) {
  const int h = blockIdx.y;
  for (int64_t bi = blockIdx.x; bi < a.batch * a.num_images; bi += gridDim.x) {
    const int64_t b = bi / a.num_images, row = b * a.nkv + h, L = evict_len(a, b, false);
    const int image = (int)(bi - b * a.num_images);
    // the image's share of the weights, and of the columns behind them
    const int64_t left = min(L, a.keep), each = (a.acc_cols + a.num_images - 1) / a.num_images, to = min((image + 1) * each, a.acc_cols);
    float* out = a.acc_out + row * a.acc_cols;
    for (int64_t j = image * each + threadIdx.x; j < to; j += 256) out[j] = j < left ? a.weights[row * a.wcols + j] : 0.0f;
    const int n = evict_image(a, row, L, image);
    if (n == 0) continue;
    const int pg = a.table[b * a.table_stride + image];
    if (pg < 0 || pg >= a.pages) {
      if (threadIdx.x == 0) atomicOr(a.err, 2);
      continue;
    }
    copy_positions<D>(a.pool + ((int64_t)pg * a.nkv + h) * a.block, a.images + (row * a.num_images + image) * a.block, n,
                      1 << a.ps_log2, threadIdx.x, 256);
  }
}

template <int D>
static int evict_launch(const EvictArgs& a, bool whole, hipStream_t st) {
  const unsigned seqs = (unsigned)std::min<int64_t>(a.batch, 65535);
  if (whole) {
    // two blocks a kv head where there are few, unless one would write the weights that the other reads
    const int halves = a.acc_out != a.acc && a.batch * a.nkv < 256 ? 2 : 1;
    hipLaunchKernelGGL(evict_kernel<D>, dim3((unsigned)a.nkv, seqs, halves), dim3(kEvThreads),
                       (size_t)std::min(a.keep, a.acc_cols) * 2, st, a, halves);
    KH_LAUNCHED();
    return KH_OK;
  }
  const dim3 parts((unsigned)a.parts, (unsigned)a.nkv, seqs), images((unsigned)std::min<int64_t>(a.batch * a.num_images, 1 << 20), (unsigned)a.nkv);
  hipLaunchKernelGGL(evict_hist_kernel, parts, dim3(256), 0, st, a);
  hipLaunchKernelGGL(evict_threshold_kernel, dim3((unsigned)a.nkv, seqs), dim3(kEvThreads), 0, st, a);
  hipLaunchKernelGGL(evict_select_kernel, parts, dim3(kEvThreads), 0, st, a);
  hipLaunchKernelGGL(evict_gather_kernel<D>, images, dim3(256), 0, st, a);
  hipLaunchKernelGGL(evict_place_kernel<D>, images, dim3(256), 0, st, a);
  KH_LAUNCHED();
  return KH_OK;
}

// ---------------------------------------------------------------- beams
struct ReorderArgs {
  char* pool;
  int64_t block, pages;
  int nkv, ps_log2;
  int* err;
  const int32_t* table;
  int32_t* out;
  int64_t cols, table_stride, out_stride, batch;
  const int64_t* len;
  const int32_t* parent;
  int beams;
};

// Block: a share of one beam: of its columns, and of the kv heads whose rows it copies.  Every wave
// works the beams' pages out for itself, a beam a lane: the beams that go on from an
// earlier beam's parent (again), and those that nobody goes on from (gone), the i-th of either meeting.
template <int D>
__global__ __launch_bounds__(256) void reorder_kernel(ReorderArgs a) {
  const int lane = threadIdx.x & 63, shares = gridDim.y, share = blockIdx.y;
  for (int64_t row = blockIdx.x; row < a.batch * a.beams; row += gridDim.x) {
    const int64_t b = row / a.beams;
    const int me = (int)(row - b * a.beams);
    int p = lane;
    if (lane < a.beams) {
      p = a.parent[b * a.beams + lane];
      if (p < 0 || p >= a.beams) {
        if (share == 0) atomicOr(a.err, 4);
        p = lane;
      }
    }
    bool again = false, gone = lane < a.beams;
    for (int i = 0; i < a.beams; ++i) {
      const int q = __builtin_amdgcn_readlane(p, i);
      again = again || (i < lane && q == p);
      gone = gone && q != lane;
    }
    const uint64_t more = __ballot(again && lane < a.beams), free = __ballot(gone);
    const int from = __builtin_amdgcn_readlane(p, me);
    int own = from;
    if (more >> me & 1) {
      uint64_t f = free;
      for (int i = __popcll(more & ((1ull << me) - 1)); i > 0; --i) f &= f - 1;
      own = __builtin_ctzll(f);
    }
    int64_t L = a.len[b];
    const int64_t cap = a.cols << a.ps_log2;
    if (L < 0 || L > cap) {
      if (share == 0 && threadIdx.x == 0) atomicOr(a.err, 1);
      L = L < 0 ? 0 : cap;
    }
    const int64_t whole = L >> a.ps_log2;
    const int32_t* tf = a.table + (b * a.beams + from) * a.table_stride;
    const int32_t* to = a.table + (b * a.beams + own) * a.table_stride;
    for (int64_t c = (int64_t)share * 256 + threadIdx.x; c < a.cols; c += (int64_t)shares * 256)
      a.out[row * a.out_stride + c] = c < whole ? tf[c] : to[c];
    const int n = (int)(L & ((1 << a.ps_log2) - 1));
    if (own == from || n == 0) continue;
    const int src = tf[whole], dst = to[whole];
    if (src < 0 || src >= a.pages || dst < 0 || dst >= a.pages) {
      if (share == 0 && threadIdx.x == 0) atomicOr(a.err, 2);
      continue;
    }
    for (int h = share; h < a.nkv; h += shares)
      copy_positions<D>(a.pool + ((int64_t)dst * a.nkv + h) * a.block, a.pool + ((int64_t)src * a.nkv + h) * a.block, n,
                        1 << a.ps_log2, threadIdx.x, 256);
  }
}

// What both calls check of a page table.
static int table_args(const kh_paged_kv* c, int64_t cols, int64_t table_stride) {
  KH_CHECK_ARG(cols >= 1 && table_stride >= cols, "page table of %lld columns, %lld apart", (long long)cols,
               (long long)table_stride);
  KH_CHECK_ARG(cols <= (INT32_MAX - 64) >> c->ps_log2, "a page table of %lld columns holds 2^31 positions",
               (long long)cols);
  return KH_OK;
}

static int evict_shape(const kh_paged_kv* c, int64_t batch, int64_t keep, int64_t acc_cols) {
  KH_CHECK_ARG(c != nullptr, "null handle");
  KH_CHECK_ARG(batch >= 0 && batch < (int64_t)1 << 31, "batch %lld not in [0,2^31)", (long long)batch);
  KH_CHECK_ARG(keep >= 1 && keep < (int64_t)1 << 31, "keep %lld not in [1,2^31)", (long long)keep);
  KH_CHECK_ARG(acc_cols >= 1 && acc_cols <= INT32_MAX - 64, "weights of %lld columns", (long long)acc_cols);
  return KH_OK;
}
// One block a kv head takes its whole sequence where its weights fit in registers, and the rows do not
// take it too long.
struct EvictSpace {
  bool whole;
  int64_t parts, images;                 // of a sequence
  int64_t weights, hist, state, bytes;   // where they lie
};
static EvictSpace evict_space(const kh_paged_kv* c, int64_t batch, int64_t keep, int64_t acc_cols) {
  EvictSpace s;
  const int64_t heads = batch * c->nkv;
  s.whole = acc_cols <= kEvThreads * kEvMost && (keep <= 4096 || keep >= acc_cols || heads >= 256);
  s.parts = (acc_cols + kEvPart - 1) / kEvPart;
  s.images = std::max<int64_t>((std::min(keep, acc_cols) + c->ps - 1) >> c->ps_log2, 1);
  s.weights = keep >= acc_cols ? 0 : heads * s.images * c->block;  // nothing moves where all can be kept
  s.hist = (s.weights + heads * std::min(keep, acc_cols) * 4 + 15) / 16 * 16;
  s.state = s.hist + heads * s.parts * kEvBins * 2;
  s.bytes = s.whole ? 0 : s.state + heads * (2 + 2 * s.parts) * 4;
  return s;
}

}  // namespace kh

using namespace kh;

extern "C" int kh_paged_kv_evict_workspace(const kh_paged_kv* c, int64_t batch, int64_t keep, int64_t acc_cols,
                                           int64_t* bytes) {
  KH_CHECK_ARG(bytes != nullptr, "null output");
  const int rc = evict_shape(c, batch, keep, acc_cols);
  if (rc != KH_OK) return rc;
  *bytes = evict_space(c, batch, keep, acc_cols).bytes;
  return KH_OK;
}

extern "C" int kh_paged_kv_evict(kh_paged_kv* c, const float* acc_dev, int64_t acc_cols, const int64_t* len_dev,
                                 int64_t batch, const int32_t* table_dev, int64_t table_cols, int64_t table_stride,
                                 int64_t keep, int64_t recent, int64_t first, int32_t* kept_dev, float* acc_out_dev,
                                 int64_t* len_out_dev, void* ws_dev, int64_t ws_bytes, void* stream) {
  int rc = evict_shape(c, batch, keep, acc_cols);
  if (rc != KH_OK) return rc;
  rc = table_args(c, table_cols, table_stride);
  if (rc != KH_OK) return rc;
  KH_CHECK_ARG(recent >= 0 && first >= 0 && recent <= keep && first <= keep - recent,
               "the first %lld and the last %lld positions are more than the %lld kept", (long long)first, (long long)recent,
               (long long)keep);
  if (batch == 0) return KH_OK;
  KH_CHECK_ARG(acc_dev && len_dev && table_dev && kept_dev && acc_out_dev && len_out_dev, "null argument");
  KH_CHECK_ARG(len_out_dev != len_dev, "the new lengths need a place of their own");
  const EvictSpace sp = evict_space(c, batch, keep, acc_cols);
  const int64_t need = sp.bytes;
  if (need > 0 && (!ws_dev || ws_bytes < need)) {
    set_error("the workspace holds %lld bytes, %lld are needed", (long long)(ws_dev ? ws_bytes : 0), (long long)need);
    return KH_ERR_CAPACITY;
  }
  KH_CHECK_ARG((reinterpret_cast<uintptr_t>(ws_dev) & 15) == 0, "the workspace must be 16-byte aligned");
  KH_ON_DEVICE(c->device, "the cache");
  EvictArgs a;
  a.pool = c->pool;
  a.block = c->block;
  a.pages = c->pages;
  a.nkv = c->nkv;
  a.ps_log2 = c->ps_log2;
  a.err = c->err;
  a.acc = acc_dev;
  a.acc_cols = acc_cols;
  a.len = len_dev;
  a.table = table_dev;
  a.cols = table_cols;
  a.table_stride = table_stride;
  a.batch = batch;
  a.keep = keep;
  a.recent = (int)recent;
  a.first = (int)first;
  a.kept = kept_dev;
  a.acc_out = acc_out_dev;
  a.len_out = len_out_dev;
  char* ws = static_cast<char*>(ws_dev);
  a.images = ws;
  a.weights = reinterpret_cast<float*>(ws + sp.weights);
  a.hist = reinterpret_cast<uint16_t*>(ws + sp.hist);
  a.state = reinterpret_cast<int*>(ws + sp.state);
  a.num_images = (int)sp.images;
  a.parts = (int)sp.parts;
  a.wcols = std::min(keep, acc_cols);
  const hipStream_t st = as_stream(stream);
  return c->d == 64 ? evict_launch<64>(a, sp.whole, st) : c->d == 128 ? evict_launch<128>(a, sp.whole, st) : evict_launch<256>(a, sp.whole, st);
}

extern "C" int kh_paged_kv_reorder(kh_paged_kv* c, const int32_t* table_dev, int64_t table_cols, int64_t table_stride,
                                   const int64_t* len_dev, int64_t batch, int beams, const int32_t* parent_dev,
                                   int32_t* out_table_dev, int64_t out_stride, void* stream) {
  KH_CHECK_ARG(c != nullptr, "null handle");
  KH_CHECK_ARG(beams >= 1 && beams <= KH_MAX_BEAMS, "%d beams not in [1,%d]", beams, KH_MAX_BEAMS);
  KH_CHECK_ARG(batch >= 0 && batch < ((int64_t)1 << 31) / beams, "batch %lld", (long long)batch);
  const int rc = table_args(c, table_cols, table_stride);
  if (rc != KH_OK) return rc;
  KH_CHECK_ARG(out_stride >= table_cols, "rows of the new table %lld apart", (long long)out_stride);
  if (batch == 0) return KH_OK;
  KH_CHECK_ARG(table_dev && len_dev && parent_dev && out_table_dev, "null argument");
  KH_CHECK_ARG(out_table_dev != table_dev, "the new table needs a place of its own");
  KH_ON_DEVICE(c->device, "the cache");
  ReorderArgs a;
  a.pool = c->pool;
  a.block = c->block;
  a.pages = c->pages;
  a.nkv = c->nkv;
  a.ps_log2 = c->ps_log2;
  a.err = c->err;
  a.table = table_dev;
  a.out = out_table_dev;
  a.cols = table_cols;
  a.table_stride = table_stride;
  a.out_stride = out_stride;
  a.batch = batch;
  a.len = len_dev;
  a.parent = parent_dev;
  a.beams = beams;
  const int64_t rows = batch * beams;
  const dim3 g((unsigned)std::min<int64_t>(rows, 1 << 20), (unsigned)std::min(c->nkv, 16));
  const hipStream_t st = as_stream(stream);
  if (c->d == 64) hipLaunchKernelGGL(reorder_kernel<64>, g, dim3(256), 0, st, a);
  else if (c->d == 128) hipLaunchKernelGGL(reorder_kernel<128>, g, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(reorder_kernel<256>, g, dim3(256), 0, st, a);
  KH_LAUNCHED();
  return KH_OK;
}
