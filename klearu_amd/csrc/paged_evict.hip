// paged_evict.hip -- which positions a paged cache keeps, and whose pages a beam writes to (gfx950).
//
// Eviction.  Of a sequence's L > keep positions a kv head keeps the first `first`, the last
// `recent` and the m = keep - first - recent heaviest between them: those above the m-th largest
// weight T, and of those equal to T the first.  Weights are compared as integers of the same order
// (f32_key), T is found digit by digit from histograms.
//
// Kept positions move towards the front of the same pages, the k-th to place k, from a place that is not
// before it: a block that moves a kv head's keys (or values), chunk after chunk from the front, holds a
// chunk in registers before it writes it, and nothing is read after it was overwritten.  Where few
// kv heads keep much, such a chain takes longer than two copies: blocks of their own for pages put the rows into
// the workspace, as images of the pages that they will lie in, and others take them there.
#include <algorithm>
#include <type_traits>

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
  // long sequences: the kept weights, histograms of parts, and what was found of T
  float* weights;  // nullptr: they go to their place at once
  char* images;  // of pages of kept positions
  int num_images;
  uint16_t* hist[3];  // of each digit, [batch][kv heads][parts][bins]
  int* state;  // [batch][kv heads][4 + parts]: T's digits so far and the rank within, for one and two; weights of each part above two
  int parts;
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

// ---------------------------------------------------------------- which positions
// A sequence that is not cut: its weights, and its positions as they are; parts [j0, j1) of the columns.
__device__ __forceinline__ void evict_none(const EvictArgs& a, int64_t row, int64_t L, int64_t j0, int64_t j1, int t, int nt, float* out) {
  for (int64_t j = j0 + t; j < min(j1, a.keep); j += nt) a.kept[row * a.keep + j] = j < L ? (int32_t)j : -1;
  for (int64_t j = j0 + t; j < min(j1, L); j += nt) out[j] = a.acc[row * a.acc_cols + j];
}

// Block: one kv head of one sequence, whose weights fit in its registers: one launch, and weights are read once.  A chain of
// length, weights, histogram, candidates and places with twelve barriers bounds it, not the bytes: 12.8 us for 32 kv heads
// of 2111 positions, 15 for 256 of up to 4099.
__global__ __launch_bounds__(kEvThreads) void evict_whole_kernel(EvictArgs a) {
  __shared__ TopkLds<kEvThreads> sh;
  __shared__ uint16_t s_kept[kEvThreads * kEvMost];
  const int h = blockIdx.x, t = threadIdx.x;
  for (int64_t b = blockIdx.y; b < a.batch; b += gridDim.y) {
    const int64_t L = evict_len(a, b, h == 0 && t == 0);
    const int64_t row = b * a.nkv + h, left = min(L, a.keep);
    const float* acc = a.acc + row * a.acc_cols;
    float* out = a.acc_out + row * a.acc_cols;
    if (h == 0 && t == 0) a.len_out[b] = left;
    if (L <= a.keep) {
      evict_none(a, row, L, 0, max(a.acc_cols, a.keep), t, kEvThreads, out);
    } else {
      const int n = (int)L - a.first - a.recent, m = (int)a.keep - a.first - a.recent, each = (n + kEvThreads - 1) / kEvThreads;
      const int i0 = t * each, cnt = min(max(n - i0, 0), each);
      uint32_t key[kEvMost], mx = 0, mn = 0xffffffffu;
#pragma unroll
      for (int e = 0; e < kEvMost; ++e) key[e] = e < each ? __float_as_uint(acc[a.first + min(i0 + e, max(n - 1, 0))]) : 0;
#pragma unroll
      for (int e = 0; e < kEvMost; ++e) {
        if (e >= each) break;
        key[e] = evict_key(__uint_as_float(key[e]));
        if (e < cnt) mx = max(mx, key[e]), mn = min(mn, key[e]);
      }
      for (int i = t; i < (1 << kTopkDigit); i += kEvThreads) sh.hist[i] = 0;
      if (t == 0) sh.s_ncand = 0;
      mx = wave_max_u32(mx);
      mn = wave_min_u32(mn);
      if ((t & 63) == 0) sh.wmax[t >> 6] = mx, sh.wmin[t >> 6] = mn;
      __syncthreads();
      if (m > 0) {
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
      __syncthreads();
      float w[kEvMost];
#pragma unroll
      for (int e = 0; e < kEvMost; ++e) {
        const int k = e * kEvThreads + t;
        if (k < a.keep) {
          w[e] = acc[s_kept[k]];
          a.kept[row * a.keep + k] = s_kept[k];
        }
      }
      __syncthreads();  // out may be acc
#pragma unroll
      for (int e = 0; e < kEvMost; ++e) {
        const int k = e * kEvThreads + t;
        if (k < a.keep) out[k] = w[e];
      }
    }
    for (int64_t j = left + t; j < a.acc_cols; j += kEvThreads) out[j] = 0.0f;
    __syncthreads();
  }
}

// Long sequences: blocks of their own for parts of kEvPart positions.
//
// T has three digits, of 11, 11 and 10 bits.  A launch for each makes histograms of it, one of each
// part's weights that have T's digits before, and its blocks all find the digit before that themselves, from
// the histograms of all parts: the launches in between would take longer.  131072 positions of eight kv heads: 4.9, 6.6 and
// 8.2 us, and 10.2 of selecting (4 MB are read four times, from the caches).
constexpr int kEvShift[3] = {21, 10, 0};

struct EvictFind {
  uint32_t hist[kEvBins];
  int wsum[kEvThreads / 64], total, kk;
  uint32_t bin;
};
// The bin that holds the kk-th largest of all parts' histograms, and its rank there; x and y: of the
// thread's bins 2 t and 2 t + 1, what parts before `part` have.
__device__ __forceinline__ void evict_find(const uint16_t* hists, int parts, int part, int& kk, uint32_t& bin, uint32_t& x, uint32_t& y,
                                           EvictFind& s) {
  const int t = threadIdx.x;
  const uint32_t* from = reinterpret_cast<const uint32_t*>(hists) + t;
  uint32_t u = 0, v = 0;
#pragma unroll 8
  for (int p = 0; p < part; ++p) {
    const uint32_t w = from[(int64_t)p * (kEvBins / 2)];
    u += w & 0xffffu;
    v += w >> 16;
  }
  x = u;
  y = v;
#pragma unroll 8
  for (int p = part; p < parts; ++p) {
    const uint32_t w = from[(int64_t)p * (kEvBins / 2)];
    u += w & 0xffffu;
    v += w >> 16;
  }
  __syncthreads();
  s.hist[2 * t] = u;
  s.hist[2 * t + 1] = v;
  __syncthreads();
  // thread t looks at two bins, thread 0 at the highest
  const int top = kEvBins - 1 - 2 * t, n1 = (int)s.hist[top], n0 = (int)s.hist[top - 1];
  const int above = block_excl_scan(n1 + n0, s.wsum, &s.total);
  if (above < kk && kk <= above + n1 + n0) {
    s.bin = kk <= above + n1 ? top : top - 1;
    s.kk = kk - above - (kk <= above + n1 ? 0 : n1);
  }
  __syncthreads();
  kk = s.kk;
  bin = s.bin;
}

// What a part of a long sequence has of weights that are compared, four a thread.
struct EvictPart {
  int64_t L, row;
  int m, parts, lo, hi, j;
  __device__ __forceinline__ EvictPart(const EvictArgs& a, int64_t b, int h, int part, bool tell) {
    L = evict_len(a, b, tell);
    row = b * a.nkv + h;
    m = (int)a.keep - a.first - a.recent;
    parts = (int)((L + kEvPart - 1) / kEvPart);
    lo = a.first;
    hi = (int)(L - a.recent);
    j = part * kEvPart + (int)threadIdx.x * kEvEach;
  }
  __device__ __forceinline__ bool in(int e) const { return j + e >= lo && j + e < hi; }
};

template <int DIGIT>
__global__ __launch_bounds__(kEvThreads) void evict_hist_kernel(EvictArgs a) {
  __shared__ EvictFind s;
  const int part = blockIdx.x, h = blockIdx.y, t = threadIdx.x;
  for (int64_t b = blockIdx.z; b < a.batch; b += gridDim.z) {
    const EvictPart p(a, b, h, part, false);
    if (p.L <= a.keep || part >= p.parts || p.m == 0) continue;
    const float* acc = a.acc + p.row * a.acc_cols;
    uint32_t key[kEvEach];
#pragma unroll
    for (int e = 0; e < kEvEach; ++e) key[e] = p.in(e) ? evict_key(acc[p.j + e]) : 0;
    int* state = a.state + p.row * (4 + a.parts);
    uint32_t T = 0;
    if constexpr (DIGIT > 0) {
      int kk = DIGIT == 1 ? p.m : state[1];
      uint32_t bin, x, y;
      if (DIGIT == 2) T = (uint32_t)state[0];
      evict_find(a.hist[DIGIT - 1] + p.row * a.parts * kEvBins, p.parts, 0, kk, bin, x, y, s);
      T |= bin << kEvShift[DIGIT - 1];
      if (part == 0 && t == 0) state[2 * DIGIT - 2] = (int)T, state[2 * DIGIT - 1] = kk;
    }
    __syncthreads();
    for (int i = t; i < kEvBins; i += kEvThreads) s.hist[i] = 0;
    if (t == 0) s.total = 0;
    __syncthreads();
    int above = 0;  // of the part's, above T's digits before the last
#pragma unroll
    for (int e = 0; e < kEvEach; ++e) {
      const int shift = DIGIT == 0 ? 0 : kEvShift[DIGIT == 0 ? 0 : DIGIT - 1];
      if (p.in(e) && (DIGIT == 0 || key[e] >> shift == T >> shift)) atomicAdd(&s.hist[(key[e] >> kEvShift[DIGIT]) & (kEvBins - 1)], 1u);
      if (DIGIT == 2) above += __popcll(__ballot(p.in(e) && key[e] >> shift > T >> shift));
    }
    if (DIGIT == 2 && (t & 63) == 0) atomicAdd(&s.total, above);
    __syncthreads();
    reinterpret_cast<uint32_t*>(a.hist[DIGIT] + (p.row * a.parts + part) * kEvBins)[t] = s.hist[2 * t] | s.hist[2 * t + 1] << 16;
    if (DIGIT == 2 && t == 0) state[4 + part] = s.total;
    __syncthreads();
  }
}

// The last digit, then the kept positions of a part, and their weights.
__global__ __launch_bounds__(kEvThreads) void evict_select_kernel(EvictArgs a) {
  __shared__ EvictFind s;
  __shared__ uint32_t uwsum[kEvThreads / 64];
  __shared__ int s_gt, s_eq;
  const int part = blockIdx.x, h = blockIdx.y, t = threadIdx.x;
  for (int64_t b = blockIdx.z; b < a.batch; b += gridDim.z) {
    const EvictPart p(a, b, h, part, part == 0 && h == 0 && t == 0);
    const int64_t L = p.L, row = p.row, j0 = (int64_t)part * kEvPart;
    if (part == 0 && h == 0 && t == 0) a.len_out[b] = min(L, a.keep);
    float* weights = a.weights ? a.weights + row * a.wcols : a.acc_out + row * a.acc_cols;
    if (!a.weights)
      for (int64_t j = max(j0, min(L, a.keep)) + t; j < min(j0 + kEvPart, a.acc_cols); j += kEvThreads) weights[j] = 0.0f;
    if (L <= a.keep) {
      evict_none(a, row, L, j0, part + 1 == a.parts ? max(a.acc_cols, a.keep) : j0 + kEvPart, t, kEvThreads, weights);
      continue;
    }
    if (part >= p.parts) continue;
    const float* acc = a.acc + row * a.acc_cols;
    float w[kEvEach];
#pragma unroll
    for (int e = 0; e < kEvEach; ++e) w[e] = p.j + e < L ? acc[p.j + e] : 0.0f;
    uint32_t T = 0xffffffffu;
    int ties = 0, gt0 = 0, eq0 = 0;  // kept of those equal to T; above it and equal to it before the part
    if (p.m > 0) {
      const int* state = a.state + row * (4 + a.parts);
      uint32_t bin, x, y;
      ties = state[3];
      if (t == 0) s_gt = s_eq = 0;
      evict_find(a.hist[2] + row * a.parts * kEvBins, p.parts, part, ties, bin, x, y, s);
      T = (uint32_t)state[2] | bin;  // the digit's upper bit is the second one's last
      int gt = (2 * t > (int)bin ? (int)x : 0) + (2 * t + 1 > (int)bin ? (int)y : 0);
      for (int c = t; c < part; c += kEvThreads) gt += state[4 + c];
      gt = wave_incl_scan(gt);
      if ((t & 63) == 63) atomicAdd(&s_gt, gt);
      if (t == (int)(bin >> 1)) s_eq = (int)(bin & 1 ? y : x);
      __syncthreads();
      gt0 = s_gt;
      eq0 = s_eq;
    }
    int32_t* kept = a.kept + row * a.keep;
    uint32_t gt = 0, eq = 0;
#pragma unroll
    for (int e = 0; e < kEvEach; ++e) {
      const uint32_t k = evict_key(w[e]);
      gt |= (p.in(e) && k > T ? 1u : 0u) << e;
      eq |= (p.in(e) && k == T ? 1u : 0u) << e;
    }
    // both counts of a part stay below 2^16
    const uint32_t before = block_excl_scan_u32(__popc(gt) | __popc(eq) << 16, uwsum);
    int e0 = eq0 + (int)(before >> 16), k0 = p.lo + gt0 + (int)(before & 0xffffu) + min(e0, ties);
#pragma unroll
    for (int e = 0; e < kEvEach; ++e) {
      const bool tie = eq >> e & 1;
      int k = -1;
      if ((gt >> e & 1) || (tie && e0 < ties)) k = k0++;
      if (p.j + e < p.lo) k = p.j + e;
      if (p.j + e >= p.hi && p.j + e < L) k = (int)(a.keep - (L - (p.j + e)));
      e0 += tie ? 1 : 0;
      if (k >= 0) kept[k] = p.j + e, weights[k] = w[e];
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- moving them
template <int N>
__device__ __forceinline__ void ld_n_u32(const char* p, uint32_t* w) {
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 v = reinterpret_cast<const uint4*>(p)[i];
      w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
  }
}
template <int N>
__device__ __forceinline__ void st_n_u32(char* p, const uint32_t* w) {
  if constexpr (N == 2) {
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) reinterpret_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  }
}

// Where position k of a kv head's kept ones comes from and goes to.
struct EvictWay {
  int from, at, to;  // page and place that it comes from (its own place if that page is none; page 0 if that is none, too);
                     // its place's page, -1 where there is none
  bool moves;
};
__device__ __forceinline__ void evict_ways(const EvictArgs& a, const int32_t* __restrict__ kept, const int32_t* __restrict__ table, int n,
                                           const int (&k)[2], EvictWay (&w)[2]) {
  const int lg = a.ps_log2;
  int f[2], pf[2], pt[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) f[i] = kept[min(k[i], n - 1)];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    f[i] = k[i] < n ? f[i] : k[i];  // places past the kept ones keep what they hold
    pf[i] = table[f[i] >> lg];
    pt[i] = table[k[i] >> lg];
  }
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bool from = (uint32_t)pf[i] < (uint64_t)a.pages, to = (uint32_t)pt[i] < (uint64_t)a.pages;
    w[i].moves = f[i] != k[i];
    bad = bad || (w[i].moves && !(from && to));
    w[i].from = from ? pf[i] : to ? pt[i] : 0;
    w[i].at = (from ? f[i] : k[i]) & ((1 << lg) - 1);
    w[i].to = to ? pt[i] : -1;
  }
  if (bad) atomicOr(a.err, 2);
}

// Rows of a page (or image), as the kernels that move them see them: positions i of a chunk come from from(i)
// (a block and a place) and go to to(i) (a block, nullptr for none) at place at(i).  A thread's pieces
// are loaded together, without branches, and written behind `between`.
template <int D, int NT, int CHUNK, typename F, typename G, typename A, typename B>
__device__ __forceinline__ void move_keys(int t, int ps, int count, F from, G to, A at, B between) {
  using P = KvParts<D>;
  constexpr int NG = P::NG, KC = D / 32, H = CHUNK * KC / NT, HP = CHUNK / NT;
  uint32_t c[H][4], p[HP][NG];
#pragma unroll
  for (int r = 0; r < H; ++r) {
    const int i = r * NT + t, k = min(i / KC, count - 1);
    int place;
    const char* x = from(k, place);
    ld_n_u32<4>(x + P::kc() + place * (D / 2) + i % KC * 16, c[r]);
  }
#pragma unroll
  for (int r = 0; r < HP; ++r) {
    int place;
    const char* x = from(min(r * NT + t, count - 1), place);
    ld_n_u32<NG>(x + P::kp(ps) + place * NG * 4, p[r]);
  }
  between();
#pragma unroll
  for (int r = 0; r < H; ++r) {
    const int i = r * NT + t, k = i / KC;
    char* y = k < count ? to(k) : nullptr;
    if (y) st_n_u32<4>(y + P::kc() + at(k) * (D / 2) + i % KC * 16, c[r]);
  }
#pragma unroll
  for (int r = 0; r < HP; ++r) {
    const int k = r * NT + t;
    char* y = k < count ? to(k) : nullptr;
    if (y) st_n_u32<NG>(y + P::kp(ps) + at(k) * NG * 4, p[r]);
  }
}
// Values: words [quad][row of sixteen][position / 2][h] of two positions' codes each.  Of the last quad's
// positions those past `count` are the caller's, too.
template <int D, int NT, int CHUNK, typename F, typename G, typename A, typename B>
__device__ __forceinline__ void move_values(int t, int ps, int count, F from, G to, A at, B between) {
  using P = KvParts<D>;
  constexpr int NG = P::NG, HN = D / 64, Q = CHUNK * 4 / NT, HP = CHUNK / NT;
  const int quads = (count + 3) >> 2;
  uint32_t v[Q][2 * HN], p[HP][NG];
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const int i = q * NT + t, r = i & 15, quad = min(i >> 4, quads - 1);
    uint32_t w[4][HN];
    int place[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const char* x = from(quad * 4 + e, place[e]);
      ld_n_u32<HN>(x + P::vc(ps) + (place[e] >> 2) * (2 * D) + (r * 2 + (place[e] >> 1 & 1)) * (HN * 4), w[e]);
    }
#pragma unroll
    for (int hf = 0; hf < HN; ++hf)
#pragma unroll
      for (int e = 0; e < 4; e += 2)
        v[q][(e >> 1) * HN + hf] = (place[e] & 1 ? w[e][hf] >> 16 : w[e][hf] & 0xffffu) |
                                   (place[e + 1] & 1 ? w[e + 1][hf] & 0xffff0000u : w[e + 1][hf] << 16);
  }
#pragma unroll
  for (int r = 0; r < HP; ++r) {
    int place;
    const char* x = from(min(r * NT + t, count - 1), place);
#pragma unroll
    for (int j = 0; j < NG; ++j) p[r][j] = *reinterpret_cast<const uint32_t*>(x + P::vp(ps) + (j * ps + place) * 4);
  }
  between();
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const int i = q * NT + t, quad = i >> 4;
    char* y = nullptr;
    if (quad < quads) {
#pragma unroll
      for (int e = 3; e >= 0; --e) y = quad * 4 + e < count && to(quad * 4 + e) ? to(quad * 4 + e) : y;
    }
    if (y) st_n_u32<2 * HN>(y + P::vc(ps) + (at(quad * 4) >> 2) * (2 * D) + (i & 15) * (8 * HN), v[q]);
  }
#pragma unroll
  for (int r = 0; r < HP; ++r) {
    const int k = r * NT + t;
    char* y = k < count ? to(k) : nullptr;
    if (y) {
#pragma unroll
      for (int j = 0; j < NG; ++j) *reinterpret_cast<uint32_t*>(y + P::vp(ps) + (j * ps + at(k)) * 4) = p[r][j];
    }
  }
}

// Block: the keys (blockIdx.z 0) or the values of a kv head, chunk after chunk.  A chunk is a chain of kept positions, pages and
// rows, so it is as long as the registers allow; 256 kv heads that keep 1024 of 64: 17.2 us, a block for each kind of
// 16-byte pieces, which each look their rows up, 25.9.
template <int D>
__global__ __launch_bounds__(kEvThreads) void evict_move_kernel(EvictArgs a) {
  constexpr int CHUNK = (D == 256 ? 1 : 2) * kEvThreads;
  __shared__ int s_from[2 * kEvThreads], s_to[2 * kEvThreads];
  __shared__ uint8_t s_at[2 * kEvThreads];
  const int h = blockIdx.x, t = threadIdx.x, ps = 1 << a.ps_log2;
  char* pool = a.pool + h * a.block;
  const int64_t apart = a.nkv * a.block;
  for (int64_t b = blockIdx.y; b < a.batch; b += gridDim.y) {
    if (evict_len(a, b, false) <= a.keep) continue;
    const int n = (int)a.keep;
    const int32_t* __restrict__ kept = a.kept + (b * a.nkv + h) * a.keep;
    const int32_t* __restrict__ table = a.table + b * a.table_stride;
    for (int c0 = 0; c0 < n; c0 += CHUNK) {
      const int count = min(CHUNK, n - c0);
      EvictWay w[2];
      int k[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) k[i] = c0 + min(i * kEvThreads + t, (count + 3 & ~3) - 1);
      evict_ways(a, kept, table, n, k, w);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (i * kEvThreads + t >= (count + 3 & ~3)) break;
        s_from[i * kEvThreads + t] = w[i].from;
        s_at[i * kEvThreads + t] = (uint8_t)w[i].at;
        s_to[i * kEvThreads + t] = w[i].moves ? w[i].to : -1;
      }
      __syncthreads();
      const auto from = [&](int i, int& place) -> const char* {
        place = s_at[i];
        return pool + s_from[i] * apart;
      };
      const auto to = [&](int i) -> char* { return s_to[i] < 0 ? nullptr : pool + s_to[i] * apart; };
      const auto at = [&](int i) { return (c0 + i) & (ps - 1); };
      const auto between = [] { __syncthreads(); };
      if (blockIdx.z == 0) move_keys<D, kEvThreads, CHUNK>(t, ps, count, from, to, at, between);
      else move_values<D, kEvThreads, CHUNK>(t, ps, count, from, to, at, between);
      lds_barrier();  // the tables are read; what is written need not have arrived
    }
  }
}

// Block: the keys (blockIdx.z 0) or the values of a kv head's positions kEvCopy c .., into images of the pages that
// they will lie in, or from there.  Nothing moves where the last of them stays.
constexpr int kEvCopy = 256;
template <int D, bool BACK>
__global__ __launch_bounds__(kEvCopy) void evict_copy_kernel(EvictArgs a) {
  __shared__ int s_from[kEvCopy], s_to[kEvCopy];
  __shared__ uint8_t s_at[kEvCopy];
  const int h = blockIdx.y, ps = 1 << a.ps_log2, t = threadIdx.x, chunks = (int)((a.keep + kEvCopy - 1) / kEvCopy);
  char* pool = a.pool + h * a.block;
  const int64_t apart = a.nkv * a.block;
  for (int64_t bi = blockIdx.x; bi < a.batch * chunks; bi += gridDim.x) {
    const int64_t b = bi / chunks, row = b * a.nkv + h;
    const int c0 = (int)(bi - b * chunks) * kEvCopy, n = (int)a.keep, count = min(kEvCopy, n - c0);
    const int32_t* __restrict__ kept = a.kept + row * a.keep;
    if (evict_len(a, b, false) <= n || kept[c0 + count - 1] == c0 + count - 1) continue;
    EvictWay w[2];
    const int k[2] = {c0 + min(t, (count + 3 & ~3) - 1), c0};
    evict_ways(a, kept, a.table + b * a.table_stride, n, k, w);
    __syncthreads();
    s_from[t] = w[0].from;
    s_at[t] = (uint8_t)w[0].at;
    s_to[t] = w[0].to;
    __syncthreads();
    char* images = a.images + row * a.num_images * a.block;
    const auto page = [&](int i) { return s_to[i] < 0 ? nullptr : pool + s_to[i] * apart; };
    const auto moved = [&](int i, int& place) -> const char* {
      place = s_at[i];
      return pool + s_from[i] * apart;
    };
    const auto at = [&](int i) { return (c0 + i) & (ps - 1); };
    const auto image = [&](int i) { return images + ((c0 + i) >> a.ps_log2) * a.block; };
    const auto held = [&](int i, int& place) -> const char* {
      place = at(i);
      return image(i);
    };
    const auto copy = [&](auto from, auto to) {
      if (blockIdx.z == 0) move_keys<D, kEvCopy, kEvCopy>(t, ps, count, from, to, at, [] {});
      else move_values<D, kEvCopy, kEvCopy>(t, ps, count, from, to, at, [] {});
    };
    if constexpr (BACK) copy(held, page);
    else copy(moved, image);
  }
}

// The kept weights of long sequences whose places other parts still read, and zeros behind them.
__global__ __launch_bounds__(256) void evict_weights_kernel(EvictArgs a) {
  const int h = blockIdx.y;
  const int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x;
  for (int64_t b = blockIdx.z; b < a.batch; b += gridDim.z) {
    const int64_t row = b * a.nkv + h, left = min(evict_len(a, b, false), a.keep);
    if (j < a.acc_cols) a.acc_out[row * a.acc_cols + j] = j < left ? a.weights[row * a.wcols + j] : 0.0f;
  }
}

template <int D>
static int evict_launch(const EvictArgs& a, bool whole, bool chain, hipStream_t st) {
  const unsigned seqs = (unsigned)std::min<int64_t>(a.batch, 65535);
  if (whole) {
    hipLaunchKernelGGL(evict_whole_kernel, dim3((unsigned)a.nkv, seqs), dim3(kEvThreads), 0, st, a);
  } else {
    const dim3 parts((unsigned)a.parts, (unsigned)a.nkv, seqs);
    hipLaunchKernelGGL(evict_hist_kernel<0>, parts, dim3(kEvThreads), 0, st, a);
    hipLaunchKernelGGL(evict_hist_kernel<1>, parts, dim3(kEvThreads), 0, st, a);
    hipLaunchKernelGGL(evict_hist_kernel<2>, parts, dim3(kEvThreads), 0, st, a);
    hipLaunchKernelGGL(evict_select_kernel, parts, dim3(kEvThreads), 0, st, a);
    if (a.weights)
      hipLaunchKernelGGL(evict_weights_kernel, dim3((unsigned)((a.acc_cols + 255) / 256), (unsigned)a.nkv, seqs), dim3(256), 0, st, a);
  }
  if (a.keep >= a.acc_cols) {  // nothing is cut, nothing moves
  } else if (chain) {
    hipLaunchKernelGGL(evict_move_kernel<D>, dim3((unsigned)a.nkv, seqs, 2), dim3(kEvThreads), 0, st, a);
  } else {
    const dim3 g((unsigned)std::min<int64_t>(a.batch * ((a.keep + kEvCopy - 1) / kEvCopy), 1 << 20), (unsigned)a.nkv, 2);
    hipLaunchKernelGGL((evict_copy_kernel<D, false>), g, dim3(kEvCopy), 0, st, a);
    hipLaunchKernelGGL((evict_copy_kernel<D, true>), g, dim3(kEvCopy), 0, st, a);
  }
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

// Block: a share of one beam: of its columns, and, a wave each, of the kv heads' keys and values that it copies.  64 x 8 beams of eight kv
// heads of 128 with half a page of 64 each: 10.2 us (a row of pieces after the other: 15.5).  The chain of parents, tables and
// rows takes 2.9, as four beams show; the rest are rounds: 94 registers leave five waves a SIMD for eight of them, and those that
// have nothing to copy take their places, too.  Every wave
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
    // 64 positions at a time; in the last four those past n keep what the place has
    const int wave = threadIdx.x >> 6, ps = 1 << a.ps_log2;
    for (int task = share * 4 + wave; task < 2 * a.nkv; task += shares * 4) {
      const char* x = a.pool + ((int64_t)src * a.nkv + (task >> 1)) * a.block;
      char* y = a.pool + ((int64_t)dst * a.nkv + (task >> 1)) * a.block;
      for (int c0 = 0; c0 < n; c0 += 64) {
        const auto source = [&](int i, int& place) -> const char* {
          place = c0 + i;
          return place < n ? x : y;
        };
        const auto to = [&](int i) { return y; };
        const auto at = [&](int i) { return c0 + i; };
        if (task & 1) move_values<D, 64, 64>(lane, ps, min(n - c0, 64), source, to, at, [] {});
        else move_keys<D, 64, 64>(lane, ps, min(n - c0, 64), source, to, at, [] {});
      }
    }
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

// Whether two tables of the same rows and columns share an element: each one's rows come in order and apart.
static bool tables_meet(const int32_t* a, int64_t a_stride, const int32_t* b, int64_t b_stride, int64_t rows, int64_t cols) {
  if (!ranges_meet(a, ((rows - 1) * a_stride + cols) * 4, b, ((rows - 1) * b_stride + cols) * 4)) return false;
  for (int64_t i = 0, j = 0; i < rows && j < rows;) {
    const int32_t *x = a + i * a_stride, *y = b + j * b_stride;
    if (ranges_meet(x, cols * 4, y, cols * 4)) return true;
    if (x < y) ++i;
    else ++j;
  }
  return false;
}

static int evict_shape(const kh_paged_kv* c, int64_t batch, int64_t keep, int64_t acc_cols) {
  KH_CHECK_ARG(c != nullptr, "null handle");
  KH_CHECK_ARG(batch >= 0 && batch < (int64_t)1 << 31, "batch %lld not in [0,2^31)", (long long)batch);
  KH_CHECK_ARG(keep >= 1 && keep < (int64_t)1 << 31, "keep %lld not in [1,2^31)", (long long)keep);
  KH_CHECK_ARG(acc_cols >= 1 && acc_cols <= INT32_MAX - 64, "weights of %lld columns", (long long)acc_cols);
  return KH_OK;
}
// How a call is cut, and its workspace: one block a kv head selects where a sequence's weights fit in its
// registers, and two (keys and values) move where there are enough of them or little is kept.  Whole calls that halve
// 128-wide sequences, such a chain / two copies, in us:
//   kv heads   keep 1024     2048          4096          8192
//        8     22.8 / 23.5   27.2 / 26.2   41.1 / 29.6   64.7 / 35.5
//       32     23.5 / 25.3   28.4 / 33.5   42.9 / 40.1   68.3 / 56.6
//       64     24.3 / 28.6   30.0 / 38.6   45.3 / 55.3   73.6 / 88.0
//      128     26.4 / 35.5   36.9 / 53.0   57.4 / 89.5   113 / 186
// 64-wide heads (62.0 / 60.9 at 64 of 8192) and 256-wide ones (30.9 / 28.6 at 8 of 2048) change sides at the same sizes.
struct EvictSpace {
  bool whole, chain;
  int64_t parts, images, weights, hist, state, bytes;
};
static EvictSpace evict_space(const kh_paged_kv* c, int64_t batch, int64_t keep, int64_t acc_cols) {
  EvictSpace s;
  const int64_t heads = batch * c->nkv, most = std::min(keep, acc_cols);
  s.whole = acc_cols <= kEvThreads * kEvMost;
  s.chain = keep >= acc_cols || heads >= 64 || keep <= 2048;
  s.parts = (acc_cols + kEvPart - 1) / kEvPart;
  s.images = (most + c->ps - 1) >> c->ps_log2;
  if (heads > ((int64_t)1 << 46) / acc_cols) {  // more than a GPU's weights: no workspace is large enough
    s.weights = s.hist = s.state = 0;
    s.bytes = s.whole ? 0 : INT64_MAX;
    return s;
  }
  s.weights = s.chain ? 0 : heads * s.images * c->block;
  s.hist = s.weights + (s.whole ? 0 : (heads * most * 4 + 15) / 16 * 16);
  s.state = s.hist + (s.whole ? 0 : 2 * heads * s.parts * kEvBins * 2);  // two digits' at a time
  s.bytes = s.state + (s.whole ? 0 : heads * (4 + s.parts) * 4);
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
  KH_CHECK_ARG(!ranges_meet(len_dev, batch * 8, len_out_dev, batch * 8), "the new lengths need a place of their own");
  const EvictSpace sp = evict_space(c, batch, keep, acc_cols);
  const int64_t need = sp.bytes;
  if (need > 0 && (!ws_dev || ws_bytes < need)) {
    set_error("the workspace holds %lld bytes, %lld are needed", (long long)(ws_dev ? ws_bytes : 0), (long long)need);
    return KH_ERR_CAPACITY;
  }
  KH_CHECK_ARG((reinterpret_cast<uintptr_t>(ws_dev) & 15) == 0, "the workspace must be 16-byte aligned");
  // at most 2^59 bytes: more heads have no workspace
  const int64_t all = batch * c->nkv * acc_cols;
  const bool in_place = acc_out_dev == acc_dev;
  KH_CHECK_ARG(in_place || !ranges_meet(acc_dev, all * 4, acc_out_dev, all * 4),
               "the weights and their new place overlap and are not the same");
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
  a.num_images = (int)sp.images;
  a.weights = in_place ? reinterpret_cast<float*>(ws + sp.weights) : nullptr;
  a.hist[0] = a.hist[2] = reinterpret_cast<uint16_t*>(ws + sp.hist);
  a.hist[1] = a.hist[0] + batch * c->nkv * sp.parts * kEvBins;
  a.state = reinterpret_cast<int*>(ws + sp.state);
  a.parts = (int)sp.parts;
  a.wcols = std::min(keep, acc_cols);
  const hipStream_t st = as_stream(stream);
  return c->d == 64    ? evict_launch<64>(a, sp.whole, sp.chain, st)
         : c->d == 128 ? evict_launch<128>(a, sp.whole, sp.chain, st)
                       : evict_launch<256>(a, sp.whole, sp.chain, st);
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
  KH_CHECK_ARG(table_stride < INT64_MAX / 8 / (batch * beams) && out_stride < INT64_MAX / 8 / (batch * beams),
               "tables of rows %lld and %lld apart", (long long)table_stride, (long long)out_stride);
  KH_CHECK_ARG(!tables_meet(table_dev, table_stride, out_table_dev, out_stride, batch * beams, table_cols),
               "the new table needs a place of its own");
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
  const dim3 g((unsigned)std::min<int64_t>(rows, 1 << 20), (unsigned)std::min((c->nkv + 1) / 2, 16));
  const hipStream_t st = as_stream(stream);
  if (c->d == 64) hipLaunchKernelGGL(reorder_kernel<64>, g, dim3(256), 0, st, a);
  else if (c->d == 128) hipLaunchKernelGGL(reorder_kernel<128>, g, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(reorder_kernel<256>, g, dim3(256), 0, st, a);
  KH_LAUNCHED();
  return KH_OK;
}
