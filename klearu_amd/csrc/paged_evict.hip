// paged_evict.hip -- which positions a paged cache keeps, and whose pages a beam writes to (gfx950).
//
// Eviction.  Of a sequence's L > keep positions a kv head keeps the first `first`, the last
// `recent` and the m = keep - first - recent heaviest between them: those above the m-th largest
// weight T, and of those equal to T the first.  Weights are compared as integers of the same order
// (f32_key), T is found digit by digit from histograms, and one ascending pass writes the kept positions.
//
// Kept positions move towards the front of the same pages, so a place may be written before another
// block has read it: their rows go to the workspace first, as images of the pages that they will
// lie in, and from there to the pages.
#include <algorithm>

#include "paged_kv.hpp"

namespace kh {

constexpr int kEvThreads = 1024;
constexpr int kEvDigit = 11;  // bits of a histogram
constexpr int kEvEach = 4;    // neighbouring positions of a thread

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
  char* ws;
  int images;  // pages of a sequence's kept positions
};

// Positions of sequence b that weights and table reach.
__device__ __forceinline__ int64_t evict_len(const EvictArgs& a, int64_t b, bool tell) {
  const int64_t L = a.len[b], cap = min(a.acc_cols, a.cols << a.ps_log2);
  if (L >= 0 && L <= cap) return L;
  if (tell) atomicOr(a.err, 1);
  return L < 0 ? 0 : cap;
}

__device__ __forceinline__ uint32_t evict_key(float w) { return w != w ? 0xffffffffu : f32_key(w); }

struct EvictLds {
  uint32_t hist[1 << kEvDigit];
  int wsum[kEvThreads / 64];
  uint32_t uwsum[kEvThreads / 64];
  int total, kk;
  uint32_t prefix, mask, mx, mn;
};

// The m-th largest key (m >= 1) of w[0 .. n - 1], and how many of the keys equal to it are among the first m.
__device__ __forceinline__ void evict_threshold(const float* __restrict__ w, int n, int m, EvictLds& s, uint32_t& T, int& ties) {
  uint32_t mx = 0, mn = 0xffffffffu;
  for (int j = threadIdx.x; j < n; j += kEvThreads) {
    const uint32_t k = evict_key(w[j]);
    mx = max(mx, k);
    mn = min(mn, k);
  }
  if (threadIdx.x == 0) s.mx = 0, s.mn = 0xffffffffu;
  __syncthreads();
  mx = wave_max_u32(mx);
  mn = wave_min_u32(mn);
  if ((threadIdx.x & 63) == 0) atomicMax(&s.mx, mx), atomicMin(&s.mn, mn);
  __syncthreads();
  mx = s.mx;
  mn = s.mn;
  // digits below the bits that all keys share
  int hi = mx == mn ? -1 : 31 - __clz(mx ^ mn);
  uint32_t mask = hi < 0 ? 0xffffffffu : hi >= 31 ? 0u : ~((2u << hi) - 1u), prefix = mx & mask;
  int kk = m;
  while (hi >= 0) {
    const int lo = max(0, hi - (kEvDigit - 1)), bins = 2 << (hi - lo);
    for (int i = threadIdx.x; i < bins; i += kEvThreads) s.hist[i] = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < n; j += kEvThreads) {
      const uint32_t k = evict_key(w[j]);
      if ((k & mask) == prefix) atomicAdd(&s.hist[(k >> lo) & (bins - 1)], 1u);
    }
    __syncthreads();
    // thread t owns bins [top - per, top), thread 0 the highest
    const int per = (bins + kEvThreads - 1) / kEvThreads, top = bins - (int)threadIdx.x * per, bot = max(top - per, 0);
    int mine = 0;
    for (int j = bot; j < top; ++j) mine += (int)s.hist[j];
    const int above = block_excl_scan(mine, s.wsum, &s.total);
    if (top > 0 && above < kk && kk <= above + mine) {
      int cum = above;
      for (int j = top - 1; j >= bot; --j) {
        if (cum + (int)s.hist[j] >= kk) {
          s.kk = kk - cum;
          s.prefix = prefix | (uint32_t)j << lo;
          s.mask = mask | (uint32_t)(bins - 1) << lo;
          break;
        }
        cum += (int)s.hist[j];
      }
    }
    __syncthreads();
    kk = s.kk;
    prefix = s.prefix;
    mask = s.mask;
    hi = lo - 1;
    __syncthreads();
  }
  T = prefix;
  ties = kk;
}

// Block: one kv head of one sequence.
__global__ __launch_bounds__(kEvThreads) void evict_select_kernel(EvictArgs a) {
  __shared__ EvictLds s;
  const int h = blockIdx.x;
  for (int64_t b = blockIdx.y; b < a.batch; b += gridDim.y) {
    const int64_t L = evict_len(a, b, h == 0 && threadIdx.x == 0);
    const int64_t row = b * a.nkv + h;
    const float* acc = a.acc + row * a.acc_cols;
    float* out = a.acc_out + row * a.acc_cols;
    int32_t* kept = a.kept + row * a.keep;
    const int64_t left = min(L, a.keep);
    if (h == 0 && threadIdx.x == 0) a.len_out[b] = left;
    if (L <= a.keep) {
      for (int64_t j = threadIdx.x; j < L; j += kEvThreads) kept[j] = (int32_t)j, out[j] = acc[j];
      for (int64_t j = L + threadIdx.x; j < a.keep; j += kEvThreads) kept[j] = -1;
    } else {
      const int n = (int)L - a.first - a.recent, m = (int)a.keep - a.first - a.recent;
      uint32_t T = 0xffffffffu;
      int ties = 0;
      if (m > 0) evict_threshold(acc + a.first, n, m, s, T, ties);
      for (int j = threadIdx.x; j < a.first; j += kEvThreads) kept[j] = j, out[j] = acc[j];
      int at = a.first, eq = 0;  // positions kept, and ties met, before the chunk
      if (m > 0) {
        constexpr int C = kEvThreads * kEvEach;
        for (int c = 0; c < n; c += C) {
          float w[kEvEach];
          uint32_t gt = 0, same = 0;
#pragma unroll
          for (int e = 0; e < kEvEach; ++e) {
            const int j = c + (int)threadIdx.x * kEvEach + e;
            w[e] = 0.0f;
            if (j < n) {
              w[e] = acc[a.first + j];
              const uint32_t k = evict_key(w[e]);
              gt |= (k > T ? 1u : 0u) << e;
              same |= (k == T ? 1u : 0u) << e;
            }
          }
          // both counts of a chunk stay below 2^16
          const uint32_t mine = __popc(gt) | __popc(same) << 16;
          const uint32_t before = block_excl_scan_u32(mine, s.uwsum);
          if (threadIdx.x == kEvThreads - 1) s.total = (int)(before + mine);
          int e0 = eq + (int)(before >> 16), k0 = at + (int)(before & 0xffffu) + min(e0, ties) - min(eq, ties);
#pragma unroll
          for (int e = 0; e < kEvEach; ++e) {
            const bool tie = same >> e & 1;
            if ((gt >> e & 1) || (tie && e0 < ties)) {
              kept[k0] = a.first + c + (int)threadIdx.x * kEvEach + e;
              out[k0] = w[e];
              ++k0;
            }
            e0 += tie ? 1 : 0;
          }
          __syncthreads();
          const uint32_t all = (uint32_t)s.total;
          const int eq1 = eq + (int)(all >> 16);
          at += (int)(all & 0xffffu) + min(eq1, ties) - min(eq, ties);
          eq = eq1;
        }
      }
      const int to = (int)a.keep - a.recent, from = (int)L - a.recent;
      for (int c = 0; c < a.recent; c += kEvThreads) {
        const int i = c + (int)threadIdx.x;
        const float w = i < a.recent ? acc[from + i] : 0.0f;
        __syncthreads();
        if (i < a.recent) kept[to + i] = from + i, out[to + i] = w;
      }
      __syncthreads();
    }
    for (int64_t j = left + threadIdx.x; j < a.acc_cols; j += kEvThreads) out[j] = 0.0f;
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
  __shared__ const char* s_blk[256];  // of each position: its block, and its place there
  __shared__ int s_at[256];
  const int h = blockIdx.y, ps = 1 << a.ps_log2, t = threadIdx.x;
  for (int64_t bi = blockIdx.x; bi < a.batch * a.images; bi += gridDim.x) {
    const int64_t b = bi / a.images, row = b * a.nkv + h;
    const int image = (int)(bi - b * a.images), first = image << a.ps_log2;
    const int n = evict_image(a, row, evict_len(a, b, false), image);
    if (n == 0) continue;
    const int32_t* __restrict__ table = a.table + b * a.table_stride;
    __syncthreads();
    if (t < n) {
      int p = a.kept[row * a.keep + first + t], pg = table[p >> a.ps_log2];
      if (pg < 0 || pg >= a.pages) {  // it does not move: the place keeps what it holds
        atomicOr(a.err, 2);
        p = first + t;
        pg = table[image];
        if (pg < 0 || pg >= a.pages) pg = 0;  // nor is it written
      }
      s_blk[t] = a.pool + ((int64_t)pg * a.nkv + h) * a.block;
      s_at[t] = p & (ps - 1);
    }
    __syncthreads();
    char* to = a.ws + (row * a.images + image) * a.block;
    constexpr int KC = D / 32;  // 16-byte pieces of a key
    for (int i = t; i < n * KC; i += 256) {
      const int k = i / KC, c = i - k * KC;
      *reinterpret_cast<uint4*>(to + P::kc() + i * 16) =
          *reinterpret_cast<const uint4*>(s_blk[k] + P::kc() + s_at[k] * (D / 2) + c * 16);
    }
    for (int i = t; i < n * NG; i += 256) {
      const int k = i / NG, j = i - k * NG;
      *reinterpret_cast<uint32_t*>(to + P::kp(ps) + i * 4) =
          *reinterpret_cast<const uint32_t*>(s_blk[k] + P::kp(ps) + (s_at[k] * NG + j) * 4);
    }
    for (int i = t; i < n * NG; i += 256) {
      const int j = i / n, k = i - j * n;
      *reinterpret_cast<uint32_t*>(to + P::vp(ps) + (j * ps + k) * 4) =
          *reinterpret_cast<const uint32_t*>(s_blk[k] + P::vp(ps) + (j * ps + s_at[k]) * 4);
    }
    // words [quad][r][position / 2][h] of two positions' codes each
    for (int i = t; i < (n + 3) / 4 * (D / 2); i += 256) {
      const int quad = i / (D / 2), w = i - quad * (D / 2), hf = w & (HN - 1), second = w / HN & 1, r = w / (2 * HN);
      uint32_t x[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int k = min(quad * 4 + 2 * second + e, n - 1), at = s_at[k];
        x[e] = *reinterpret_cast<const uint16_t*>(s_blk[k] + P::vc(ps) + (at >> 2) * (2 * D) +
                                                  (((r * 2 + (at >> 1 & 1)) * HN + hf) * 2 + (at & 1)) * 2);
      }
      *reinterpret_cast<uint32_t*>(to + P::vc(ps) + i * 4) = x[0] | x[1] << 16;
    }
  }
}

template <int D>
__global__ __launch_bounds__(256) void evict_place_kernel(EvictArgs a) {
  const int h = blockIdx.y;
  for (int64_t bi = blockIdx.x; bi < a.batch * a.images; bi += gridDim.x) {
    const int64_t b = bi / a.images, row = b * a.nkv + h;
    const int image = (int)(bi - b * a.images);
    const int n = evict_image(a, row, evict_len(a, b, false), image);
    if (n == 0) continue;
    const int pg = a.table[b * a.table_stride + image];
    if (pg < 0 || pg >= a.pages) {
      if (threadIdx.x == 0) atomicOr(a.err, 2);
      continue;
    }
    copy_positions<D>(a.pool + ((int64_t)pg * a.nkv + h) * a.block, a.ws + (row * a.images + image) * a.block, n,
                      1 << a.ps_log2, threadIdx.x, 256);
  }
}

template <int D>
static int evict_move(const EvictArgs& a, hipStream_t st) {
  const dim3 g((unsigned)std::min<int64_t>(a.batch * a.images, 1 << 20), (unsigned)a.nkv);
  hipLaunchKernelGGL(evict_gather_kernel<D>, g, dim3(256), 0, st, a);
  hipLaunchKernelGGL(evict_place_kernel<D>, g, dim3(256), 0, st, a);
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
// Nothing is evicted, and no page image is needed, where the weights have no more columns than are kept.
static int64_t evict_images(const kh_paged_kv* c, int64_t keep, int64_t acc_cols) {
  return keep >= acc_cols ? 0 : (keep + c->ps - 1) >> c->ps_log2;
}

}  // namespace kh

using namespace kh;

extern "C" int kh_paged_kv_evict_workspace(const kh_paged_kv* c, int64_t batch, int64_t keep, int64_t acc_cols,
                                           int64_t* bytes) {
  KH_CHECK_ARG(bytes != nullptr, "null output");
  const int rc = evict_shape(c, batch, keep, acc_cols);
  if (rc != KH_OK) return rc;
  *bytes = batch * c->nkv * evict_images(c, keep, acc_cols) * c->block;
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
  const int64_t images = evict_images(c, keep, acc_cols), need = batch * c->nkv * images * c->block;
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
  a.ws = static_cast<char*>(ws_dev);
  a.images = (int)images;
  const hipStream_t st = as_stream(stream);
  hipLaunchKernelGGL(evict_select_kernel, dim3((unsigned)c->nkv, (unsigned)(batch < 65535 ? batch : 65535)), dim3(kEvThreads), 0,
                     st, a);
  KH_LAUNCHED();
  if (images == 0) return KH_OK;
  return c->d == 64 ? evict_move<64>(a, st) : c->d == 128 ? evict_move<128>(a, st) : evict_move<256>(a, st);
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
