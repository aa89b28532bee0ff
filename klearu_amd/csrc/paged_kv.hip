// paged_kv.hip -- a paged K/V cache held in 4 bits: appending rows with the
// position rotation applied on the way, and reading rows back (gfx950).
//
// Thirty-two neighbouring values x of a head share
//   m = min x rounded down to BF16,  s = (max x - m) / 15 rounded up to BF16
// and each is held as c = rint((x - m) / s), 0..15, and stands for s c + m: with
// m below every value and 15 s above every distance from it, no value is
// clipped and each is off by at most s / 2.  Differences and quotients are f32
// with one rounding each, so the codes are a function of x alone.  A group that
// holds a value that is not finite, or of 2^100 and more, has s = NaN, m = 0 and
// stands for NaN: no infinity ever enters the cache, and none comes of its sums.
#include <new>

#include "paged_kv.hpp"

namespace kh {

constexpr int kKvThreads = 256;
constexpr int kSeqLds = 1025;  // offsets staged in LDS for the search of a row's sequence

// BF16 bits of x rounded towards minus infinity, and of x >= 0 towards plus infinity.
__device__ __forceinline__ uint32_t bf16_down(float x) {
  const uint32_t u = __float_as_uint(x);
  return (u & 0x80000000u) ? (u + 0xffffu) >> 16 : u >> 16;
}
__device__ __forceinline__ uint32_t bf16_up(float x) { return (__float_as_uint(x) + 0xffffu) >> 16; }

// minimum | scale << 16 of a group with range [lo, hi]; bad: it stands for NaN.
__device__ __forceinline__ uint32_t kv_pair(float lo, float hi, bool bad) {
  const uint32_t m = bf16_down(lo);
  const uint32_t s = bf16_up(__fdiv_rn(__fsub_rn(hi, __uint_as_float(m << 16)), 15.0f));
  return bad ? 0x7fc00000u : m | s << 16;  // s >= 0: hi >= m
}
__device__ __forceinline__ uint32_t kv_code(float x, uint32_t pair) {
  const float s = __uint_as_float(pair & 0xffff0000u), m = __uint_as_float(pair << 16);
  if (!(s > 0.0f)) return 0;
  const float q = rintf(__fdiv_rn(__fsub_rn(x, m), s));
  return (uint32_t)fminf(fmaxf(q, 0.0f), 15.0f);
}
__device__ __forceinline__ bool too_large(float x) { return (__float_as_uint(x) & 0x7fffffffu) >= 0x71800000u; }  // 2^100

struct KvRows {
  char* pool;
  int64_t block, pages;
  int nkv, ps_log2;
  int* err;
  const int64_t *off, *start;
  const int32_t* table;
  int64_t batch, rows, cols, table_stride;
};

// Where row t of head h lies: its block, and its place in the page (-1: the
// row lies in no sequence, or its place is not in the cache, which is recorded).
__device__ __forceinline__ int kv_place(const KvRows& a, const int64_t* off, int64_t t, int h, char** blk,
                                        int64_t* pos) {
  const int64_t b = seq_of_row(off, a.batch, t);
  if (b < 0) return -1;
  const int64_t p = a.start[b] + (t - off[b]);
  const int64_t col = p >> a.ps_log2;
  if (p < 0 || col >= a.cols) {
    atomicOr(a.err, 1);
    return -1;
  }
  const int64_t pg = a.table[b * a.table_stride + col];
  if (pg < 0 || pg >= a.pages) {
    atomicOr(a.err, 2);
    return -1;
  }
  *pos = p;
  *blk = a.pool + (pg * a.nkv + h) * a.block;
  return (int)(p & ((1 << a.ps_log2) - 1));
}

// The offsets the block searches: an LDS copy where they fit.
__device__ __forceinline__ const int64_t* stage_off(const KvRows& a, int64_t* lds) {
  if (a.batch >= kSeqLds) return a.off;
  for (int i = threadIdx.x; i <= a.batch; i += blockDim.x) lds[i] = a.off[i];
  __syncthreads();
  return lds;
}

struct AppendArgs {
  KvRows r;
  const void *k, *v;
  int64_t ks, kh, vs, vh;
  const int64_t* pos;  // rotary positions of the rows, or nullptr: their places in the cache
  const float2* table;
  int64_t max_pos;
  int rot, half_layout;
  int* rope_err;
  int kvec, vvec;  // 16-byte loads
};

// The key's elements d .. d + 7 after the rotation, in f32.
template <typename T>
__device__ __forceinline__ void rotated8(const T* __restrict__ x, int d, int rot, int half_layout, bool vec,
                                         const float2* __restrict__ tab, float (&f)[8]) {
  load8(x + d, vec, f);
  if (d >= rot) return;
  if (!half_layout) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (d + 2 * i >= rot) break;
      const float2 cs = tab[(d >> 1) + i];
      const float x0 = f[2 * i], x1 = f[2 * i + 1];
      f[2 * i] = x0 * cs.x - x1 * cs.y;
      f[2 * i + 1] = x1 * cs.x + x0 * cs.y;
    }
    return;
  }
  const int half = rot >> 1;
  if ((half & 7) == 0) {  // the whole piece on one side of the pairs
    const bool second = d >= half;
    float o[8];
    load8(x + (second ? d - half : d + half), vec, o);
    tab += second ? d - half : d;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 cs = tab[i];
      f[i] = second ? f[i] * cs.x + o[i] * cs.y : f[i] * cs.x - o[i] * cs.y;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int e = d + i;
    if (e >= rot) break;
    const bool second = e >= half;
    const float o = load_f32(x + (second ? e - half : e + half));
    const float2 cs = tab[second ? e - half : e];
    f[i] = second ? f[i] * cs.x + o * cs.y : f[i] * cs.x - o * cs.y;
  }
}

// Blocks with blockIdx.y = 0 append keys, D / 8 lanes a row with eight
// neighbouring values each (four lanes share a group); the others append
// values, D / 4 lanes a row with the four values of one u16 each (the sixteen
// lanes of a DPP row share two groups).
template <typename T, int D>
__global__ __launch_bounds__(kKvThreads) void kv_append_kernel(AppendArgs a) {
  __shared__ int64_t s_off[kSeqLds];
  constexpr int NG = D / kKvGroup, HN = D / 64;
  using P = KvParts<D>;
  const int64_t* off = stage_off(a.r, s_off);
  const int ps = 1 << a.r.ps_log2;
  const int64_t units = a.r.rows * a.r.nkv;
  if (blockIdx.y == 0) {
    constexpr int L = D / 8, R = kKvThreads / L;
    const int c = threadIdx.x % L, j = c >> 2, g = c & 3;
    for (int64_t u = (int64_t)blockIdx.x * R + threadIdx.x / L; u < units; u += (int64_t)gridDim.x * R) {
      const int64_t t = u / a.r.nkv;
      const int h = (int)(u - t * a.r.nkv);
      char* blk = nullptr;
      int64_t p = 0;
      int at = kv_place(a.r, off, t, h, &blk, &p);
      const float2* tab = a.table;
      if (tab && at >= 0) {
        if (a.pos) p = a.pos[t];
        if (p < 0 || p >= a.max_pos) {
          atomicOr(a.rope_err, 1);
          at = -1;
        } else
          tab += p * (a.rot >> 1);
      }
      float f[8];
      // the lanes of a group take the same way: `at` is the row's
      if (at < 0) continue;
      const T* x = static_cast<const T*>(a.k) + t * a.ks + h * a.kh;
      if (tab) rotated8(x, 8 * c, a.rot, a.half_layout, a.kvec, tab, f);
      else load8(x + 8 * c, a.kvec, f);
      float lo = f[0], hi = f[0];
      int bad = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        lo = fminf(lo, f[i]);
        hi = fmaxf(hi, f[i]);
        bad |= too_large(f[i]);
      }
      lo = fminf(lo, dppf<kDppQuadSwap1>(lo));
      hi = fmaxf(hi, dppf<kDppQuadSwap1>(hi));
      bad |= dpp<kDppQuadSwap1>(bad);
      lo = fminf(lo, dppf<kDppQuadSwap2>(lo));
      hi = fmaxf(hi, dppf<kDppQuadSwap2>(hi));
      bad |= dpp<kDppQuadSwap2>(bad);
      const uint32_t pair = kv_pair(lo, hi, bad != 0);
      uint32_t w = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) w |= kv_code(f[i], pair) << (4 * i);
      *reinterpret_cast<uint32_t*>(blk + P::kc() + at * (D / 2) + (g * NG + j) * 4) = w;
      if (g == 0) *reinterpret_cast<uint32_t*>(blk + P::kp(ps) + (at * NG + j) * 4) = pair;
    }
  } else {
    constexpr int L = D / 4, R = kKvThreads / L;
    const int c = threadIdx.x % L, r = c & 15, hf = c >> 4;
    for (int64_t u = (int64_t)blockIdx.x * R + threadIdx.x / L; u < units; u += (int64_t)gridDim.x * R) {
      const int64_t t = u / a.r.nkv;
      const int h = (int)(u - t * a.r.nkv);
      char* blk = nullptr;
      int64_t p = 0;
      int at = kv_place(a.r, off, t, h, &blk, &p);
      if (a.table && at >= 0) {  // a row without a rotation is not appended at all
        if (a.pos) p = a.pos[t];
        if (p < 0 || p >= a.max_pos) at = -1;
      }
      if (at < 0) continue;
      const T* x = static_cast<const T*>(a.v) + t * a.vs + h * a.vh + 64 * hf + r;
      float f[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) f[n] = load_f32(x + 16 * n);
      uint32_t w = 0;
      uint32_t pairs[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float lo = fminf(f[2 * q], f[2 * q + 1]), hi = fmaxf(f[2 * q], f[2 * q + 1]);
        int bad = too_large(f[2 * q]) || too_large(f[2 * q + 1]);
        lo = fminf(lo, dppf<kDppQuadSwap1>(lo));
        hi = fmaxf(hi, dppf<kDppQuadSwap1>(hi));
        bad |= dpp<kDppQuadSwap1>(bad);
        lo = fminf(lo, dppf<kDppQuadSwap2>(lo));
        hi = fmaxf(hi, dppf<kDppQuadSwap2>(hi));
        bad |= dpp<kDppQuadSwap2>(bad);
        lo = fminf(lo, dppf<kDppRowHalfMirror>(lo));
        hi = fmaxf(hi, dppf<kDppRowHalfMirror>(hi));
        bad |= dpp<kDppRowHalfMirror>(bad);
        lo = fminf(lo, dppf<kDppRowMirror>(lo));
        hi = fmaxf(hi, dppf<kDppRowMirror>(hi));
        bad |= dpp<kDppRowMirror>(bad);
        pairs[q] = kv_pair(lo, hi, bad != 0);
        w |= kv_code(f[2 * q], pairs[q]) << (8 * q);
        w |= kv_code(f[2 * q + 1], pairs[q]) << (8 * q + 4);
      }
      uint16_t* vc = reinterpret_cast<uint16_t*>(blk + P::vc(ps));
      vc[((((at >> 2) * 16 + r) * 2 + ((at >> 1) & 1)) * HN + hf) * 2 + (at & 1)] = (uint16_t)w;
      if (r < 2) *reinterpret_cast<uint32_t*>(blk + P::vp(ps) + ((2 * hf + r) * ps + at) * 4) = r ? pairs[1] : pairs[0];
    }
  }
}

struct GatherArgs {
  KvRows r;
  void *k, *v;
};

// The inverse walk, eight neighbouring values a lane.
template <typename T, int D>
__global__ __launch_bounds__(kKvThreads) void kv_gather_kernel(GatherArgs a) {
  __shared__ int64_t s_off[kSeqLds];
  constexpr int NG = D / kKvGroup, HN = D / 64, L = D / 8, R = kKvThreads / L;
  using P = KvParts<D>;
  const int64_t* off = stage_off(a.r, s_off);
  const int ps = 1 << a.r.ps_log2;
  const int c = threadIdx.x % L, j = c >> 2;
  const int64_t units = a.r.rows * a.r.nkv;
  for (int64_t u = (int64_t)blockIdx.x * R + threadIdx.x / L; u < units; u += (int64_t)gridDim.x * R) {
    const int64_t t = u / a.r.nkv;
    const int h = (int)(u - t * a.r.nkv);
    char* blk = nullptr;
    int64_t p = 0;
    const int at = kv_place(a.r, off, t, h, &blk, &p);
    if (at < 0) continue;
    float f[8];
    if (blockIdx.y == 0) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(blk + P::kc() + at * (D / 2) + ((c & 3) * NG + j) * 4);
      const uint32_t pr = *reinterpret_cast<const uint32_t*>(blk + P::kp(ps) + (at * NG + j) * 4);
      const float s = __uint_as_float(pr & 0xffff0000u), m = __uint_as_float(pr << 16);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = s * (float)((w >> (4 * i)) & 15) + m;
    } else {
      // d = 8 c + i = 64 hf + 16 n + r: one nibble of eight neighbouring r
      const int hf = c >> 3, n = (c >> 1) & 3, r0 = 8 * (c & 1);
      const uint16_t* vc = reinterpret_cast<const uint16_t*>(blk + P::vc(ps));
      const uint32_t pr = *reinterpret_cast<const uint32_t*>(blk + P::vp(ps) + (j * ps + at) * 4);
      const float s = __uint_as_float(pr & 0xffff0000u), m = __uint_as_float(pr << 16);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t w = vc[((((at >> 2) * 16 + r0 + i) * 2 + ((at >> 1) & 1)) * HN + hf) * 2 + (at & 1)];
        f[i] = s * (float)((w >> (4 * n)) & 15) + m;
      }
    }
    T* y = static_cast<T*>(blockIdx.y == 0 ? a.k : a.v) + u * D + 8 * c;
    store8(y, true, f);
  }
}

template <typename T>
static void append_launch(int d, const AppendArgs& a, dim3 g, hipStream_t st) {
  if (d == 64) hipLaunchKernelGGL((kv_append_kernel<T, 64>), g, dim3(kKvThreads), 0, st, a);
  else if (d == 128) hipLaunchKernelGGL((kv_append_kernel<T, 128>), g, dim3(kKvThreads), 0, st, a);
  else hipLaunchKernelGGL((kv_append_kernel<T, 256>), g, dim3(kKvThreads), 0, st, a);
}
template <typename T>
static void gather_launch(int d, const GatherArgs& a, dim3 g, hipStream_t st) {
  if (d == 64) hipLaunchKernelGGL((kv_gather_kernel<T, 64>), g, dim3(kKvThreads), 0, st, a);
  else if (d == 128) hipLaunchKernelGGL((kv_gather_kernel<T, 128>), g, dim3(kKvThreads), 0, st, a);
  else hipLaunchKernelGGL((kv_gather_kernel<T, 256>), g, dim3(kKvThreads), 0, st, a);
}

// The arguments every call over rows of sequences checks.
static int rows_args(const kh_paged_kv* c, int dtype, int64_t rows, const int64_t* off, int64_t batch,
                     const int64_t* start, const int32_t* table, int64_t cols, int64_t table_stride, KvRows* r) {
  KH_CHECK_ARG(c != nullptr, "null handle");
  KH_CHECK_ARG(dtype == KH_DT_F32 || dtype == KH_DT_BF16, "dtype %d: f32 and BF16 are supported", dtype);
  KH_CHECK_ARG(rows >= 0 && batch >= 0, "rows %lld, batch %lld", (long long)rows, (long long)batch);
  KH_CHECK_ARG(rows <= (int64_t)1 << 40, "too many rows");
  KH_CHECK_ARG(rows == 0 || batch == 0 || (off && start && table), "null argument");
  KH_CHECK_ARG(cols >= 1 && table_stride >= cols, "page table of %lld columns, %lld apart", (long long)cols,
               (long long)table_stride);
  r->pool = c->pool;
  r->block = c->block;
  r->pages = c->pages;
  r->nkv = c->nkv;
  r->ps_log2 = c->ps_log2;
  r->err = c->err;
  r->off = off;
  r->start = start;
  r->table = table;
  r->batch = batch;
  r->rows = rows;
  r->cols = cols;
  r->table_stride = table_stride;
  return KH_OK;
}

}  // namespace kh

using namespace kh;

extern "C" int kh_paged_kv_destroy(kh_paged_kv* c) {
  if (!c) return KH_OK;
  dev_free(c->pool);
  dev_free(c->err);
  delete c;
  return KH_OK;
}

extern "C" int kh_paged_kv_create(int num_kv_heads, int head_dim, int page_size, int64_t num_pages,
                                  kh_paged_kv** out) {
  KH_CHECK_ARG(out != nullptr, "null output");
  *out = nullptr;
  KH_CHECK_ARG(num_kv_heads >= 1 && num_kv_heads <= 4096, "num_kv_heads %d not in [1,4096]", num_kv_heads);
  KH_CHECK_ARG(num_pages >= 1 && num_pages <= INT32_MAX, "num_pages %lld not in [1,2^31)", (long long)num_pages);
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) {
    set_error("head_dim %d not in {64, 128, 256}", head_dim);
    return KH_ERR_UNSUPPORTED;
  }
  int lg = 4;
  while (lg < 8 && (1 << lg) != page_size) ++lg;
  if ((1 << lg) != page_size) {
    set_error("page_size %d not in {16, 32, 64, 128, 256}", page_size);
    return KH_ERR_UNSUPPORTED;
  }
  kh_paged_kv* c = new (std::nothrow) kh_paged_kv;
  if (!c) {
    set_error("out of host memory");
    return KH_ERR_ALLOC;
  }
  c->nkv = num_kv_heads;
  c->d = head_dim;
  c->ps = page_size;
  c->ps_log2 = lg;
  c->pages = num_pages;
  c->block = kv_block_bytes(page_size, head_dim);
  const auto fill = [&]() -> int {
    KH_HIP(hipGetDevice(&c->device));
    const size_t bytes = (size_t)num_pages * num_kv_heads * c->block;
    c->pool = static_cast<char*>(dev_alloc(bytes));
    c->err = static_cast<int*>(dev_alloc(sizeof(int)));
    if (!c->pool || !c->err) return KH_ERR_ALLOC;
    // zeroed: places that were never written stand for 0, so that no bit
    // pattern but the format's own is ever read
    KH_HIP(hipMemset(c->pool, 0, bytes));
    KH_HIP(hipMemset(c->err, 0, sizeof(int)));
    KH_HIP(hipStreamSynchronize(nullptr));
    return KH_OK;
  };
  const int rc = fill();
  if (rc != KH_OK) {
    kh_paged_kv_destroy(c);
    return rc;
  }
  *out = c;
  return KH_OK;
}

extern "C" int kh_paged_kv_status(const kh_paged_kv* c) {
  KH_CHECK_ARG(c != nullptr, "null handle");
  KH_ON_DEVICE(c->device, "the cache");
  KH_HIP(hipDeviceSynchronize());
  int bad = 0;
  KH_HIP(hipMemcpy(&bad, c->err, sizeof(int), hipMemcpyDeviceToHost));
  if (!bad) return KH_OK;
  KH_HIP(hipMemset(c->err, 0, sizeof(int)));
  set_error("%s%s", (bad & 1) ? "a position lay outside its sequence's page table; " : "",
            (bad & 2) ? "a page id lay outside the pool; " : "");
  return KH_ERR_ARG;
}

extern "C" int kh_paged_kv_append(kh_paged_kv* c, const kh_rope* rope, int dtype, const void* k_dev,
                                  int64_t k_row_stride, int64_t k_head_stride, const void* v_dev,
                                  int64_t v_row_stride, int64_t v_head_stride, int64_t rows, const int64_t* off_dev,
                                  int64_t batch, const int64_t* start_dev, const int64_t* pos_dev,
                                  const int32_t* table_dev, int64_t table_cols, int64_t table_stride, void* stream) {
  AppendArgs a;
  const int rc = rows_args(c, dtype, rows, off_dev, batch, start_dev, table_dev, table_cols, table_stride, &a.r);
  if (rc != KH_OK) return rc;
  if (rope) {
    KH_CHECK_ARG(rope->rot <= c->d, "the rotation takes %d elements, a head has %d", rope->rot, c->d);
    KH_CHECK_ARG(rope->device == c->device, "the rotation lives on device %d, the cache on %d", rope->device,
                 c->device);
  }
  KH_CHECK_ARG(k_row_stride >= 0 && k_head_stride >= 0 && v_row_stride >= 0 && v_head_stride >= 0,
               "negative stride");
  KH_CHECK_ARG(!pos_dev || rope, "rotary positions without a rotation");
  if (rows == 0 || batch == 0) return KH_OK;
  KH_CHECK_ARG(k_dev && v_dev, "null argument");
  KH_ON_DEVICE(c->device, "the cache");
  a.k = k_dev;
  a.v = v_dev;
  a.ks = k_row_stride;
  a.kh = k_head_stride;
  a.vs = v_row_stride;
  a.vh = v_head_stride;
  a.pos = pos_dev;
  a.table = rope ? rope->table : nullptr;
  a.max_pos = rope ? rope->max_pos : 0;
  a.rot = rope ? rope->rot : 0;
  a.half_layout = rope && rope->layout == KH_ROPE_HALF ? 1 : 0;
  a.rope_err = rope ? rope->err : nullptr;
  a.kvec = aligned16(k_dev, dtype, k_row_stride, k_head_stride) ? 1 : 0;
  a.vvec = aligned16(v_dev, dtype, v_row_stride, v_head_stride) ? 1 : 0;
  const int64_t per = kKvThreads / (c->d / 4);
  const int64_t blocks = (rows * c->nkv + per - 1) / per;
  const dim3 g((unsigned)(blocks < 16384 ? blocks : 16384), 2);
  if (dtype == KH_DT_F32) append_launch<float>(c->d, a, g, as_stream(stream));
  else append_launch<uint16_t>(c->d, a, g, as_stream(stream));
  KH_LAUNCHED();
  return KH_OK;
}

extern "C" int kh_paged_kv_gather(const kh_paged_kv* c, int dtype, int64_t rows, const int64_t* off_dev,
                                  int64_t batch, const int64_t* start_dev, const int32_t* table_dev,
                                  int64_t table_cols, int64_t table_stride, void* k_dev, void* v_dev, void* stream) {
  GatherArgs a;
  const int rc = rows_args(c, dtype, rows, off_dev, batch, start_dev, table_dev, table_cols, table_stride, &a.r);
  if (rc != KH_OK) return rc;
  if (rows == 0 || batch == 0) return KH_OK;
  KH_CHECK_ARG(k_dev && v_dev, "null argument");
  KH_CHECK_ARG(((reinterpret_cast<uintptr_t>(k_dev) | reinterpret_cast<uintptr_t>(v_dev)) & 15) == 0,
               "outputs must be 16-byte aligned");
  KH_ON_DEVICE(c->device, "the cache");
  a.k = k_dev;
  a.v = v_dev;
  const int64_t per = kKvThreads / (c->d / 8);
  const int64_t blocks = (rows * c->nkv + per - 1) / per;
  const dim3 g((unsigned)(blocks < 16384 ? blocks : 16384), 2);
  if (dtype == KH_DT_F32) gather_launch<float>(c->d, a, g, as_stream(stream));
  else gather_launch<uint16_t>(c->d, a, g, as_stream(stream));
  KH_LAUNCHED();
  return KH_OK;
}
