// paged_weights.hip -- the attention weight that cached positions get, added up (gfx950).
//
//   acc[j] += sum_i exp(c q_i . k_j - lse_i)   over the rows i (and query heads) that see position j
//
// The log-sum-exps are known, so positions are independent of each other: a wave holds the keys of
// its positions in registers and runs the rows over them; nothing is joined, and each
// sum has one owner and one order.  With group sums A_g = sum_{d in g} q_d c_d of the codes, which
// are exact BF16 numbers,
//   log2(e) (c q . k - lse) = sum_g (c' s_g) A_g + [sum_g m_g (c' Q_g) - lse'],   Q_g = sum_{d in g} q_d
// where the bracket is one more matrix product, of the BF16 minima with three BF16 terms of c' Q_g
// and of lse' (three hold all bits of an f32; c' = c log2 e).
//
// Scores come out of the matrix core with positions along lanes and rows along registers, so a
// sum over rows stays in its lane until the end.
#include <algorithm>
#include <cmath>

#include "paged_frag.hpp"

namespace kh {

constexpr int kWtWaves = 4;
constexpr float kWtNone = 0x1p100f;  // a log-sum-exp whose rows add nothing

struct WtArgs {
  const char* pool;
  int64_t block, pages;
  int nkv, ps_log2;
  int* err;
  const void* q;
  int64_t qs, qh;
  const int64_t *off, *len;
  int64_t batch, rows;
  const int32_t* table;
  int64_t cols, table_stride;
  int nh, gs;
  float c1;  // scale * log2(e)
  int causal;
  int64_t window;
  const float* lse;
  float* acc;
  int64_t acc_cols;
  int qvec;
};

// A tile of 16 rows (of the heads of a kv head, row after row) as first operands: the
// queries' terms, slots (0,4,1,5,2,6,3,7) of eight neighbouring elements as codes2 gives the codes, and the bracket's.
template <int D, typename T>
struct WtRows {
  static constexpr int NG = D / kKvGroup, NQ = sizeof(T) == 4 ? 3 : 1;
  uint4 q[NG][NQ], base;
  __device__ __forceinline__ void load(const WtArgs& a, int64_t o0, int nr, int h, int tile, int lane) {
    const int g = lane >> 4, rr = tile * 16 + (lane & 15);
    const bool inside = rr < nr;
    const int i = (int)((uint32_t)(inside ? rr : 0) / (uint32_t)a.gs);
    const int head = h * a.gs + ((inside ? rr : 0) - i * a.gs);
    const int64_t t = o0 + i;
    const T* x = static_cast<const T*>(a.q) + t * a.qs + head * a.qh;
    Raw8<T> raw[NG];
#pragma unroll
    for (int j = 0; j < NG; ++j) raw[j].load(x + 32 * j + 8 * g, a.qvec);
    const float lse = a.lse[t * a.nh + head];
    const bool on = inside && !__builtin_isinf(lse);
    float e[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      float f[8];
      raw[j].get(f);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = on ? f[k] : 0.0f;
      const float s[8] = {f[0], f[4], f[1], f[5], f[2], f[6], f[3], f[7]};
      terms8<NQ>(s, q[j]);
      e[j] = a.c1 * across_groups_sum(((f[0] + f[1]) + (f[2] + f[3])) + ((f[4] + f[5]) + (f[6] + f[7])));
    }
    uint4 tm[3];
    terms8<3>(e, tm);
    const float l0 = on ? -lse * kLog2e : -kWtNone;
    const float t0 = bf16_to_f32(f32_to_bf16(l0)), t1 = bf16_to_f32(f32_to_bf16(l0 - t0)), t2 = l0 - t0 - t1;
    const uint4 tl = make_uint4(cvt_bf16x2(t0, t1), cvt_bf16x2(t2, 0.0f), 0, 0);
    base = g == 0 ? tm[0] : g == 1 ? tm[1] : g == 2 ? tm[2] : tl;
  }
};

// The keys of 16 positions as second operands, a position a column.
template <int D>
struct WtKeys {
  static constexpr int NG = D / kKvGroup;
  uint4 c[NG], m;
  float s[NG];
  __device__ __forceinline__ void put(const uint32_t (&w)[NG], const uint32_t (&p)[NG], float c1, int g) {
    uint32_t e[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      c[j] = make_uint4(codes2<0>(w[j], 0), codes2<0>(w[j], 1), codes2<0>(w[j], 2), codes2<0>(w[j], 3));
      s[j] = c1 * __uint_as_float(p[j] & 0xffff0000u);
      e[j] = p[j] & 0xffffu;
    }
    m = g == 3 ? make_uint4(0x3f803f80u, 0x00003f80u, 0, 0)
               : make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
  }
};

// Block: 4 waves with NPT tiles of 16 positions each, of one kv head of one sequence.
template <int D, typename T, int NPT>
__global__ __launch_bounds__(64 * kWtWaves) void paged_weights_kernel(WtArgs a) {
  using P = KvParts<D>;
  constexpr int NG = D / kKvGroup, NQ = WtRows<D, T>::NQ, BP = 16 * NPT * kWtWaves;
  const int lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = blockIdx.y, ps = 1 << a.ps_log2;
  const int64_t cap = a.cols << a.ps_log2;
  for (int64_t b = blockIdx.z; b < a.batch; b += gridDim.z) {
    const int32_t* __restrict__ table = a.table + b * a.table_stride;
    int64_t o0 = a.off[b], o1 = a.off[b + 1], L = a.len[b];
    o0 = o0 < 0 ? 0 : o0;
    o1 = o1 > a.rows ? a.rows : o1;
    if (o1 <= o0) continue;
    const int n = (int)(o1 - o0), nr = n * a.gs;
    if (L < 0 || L > min(cap, a.acc_cols)) {
      if (threadIdx.x == 0) atomicOr(a.err, 1);
      L = L < 0 ? 0 : min(L, cap);
    }
    const int64_t before = L - n;  // the first row's position
    const int E = (int)min(L, a.acc_cols);
    float* acc = a.acc + (b * a.nkv + h) * a.acc_cols;
    for (int64_t pb = blockIdx.x; pb * BP < E; pb += gridDim.x) {
      const int base = (int)(pb * BP) + wave * 16 * NPT;
      WtKeys<D> x[NPT];
      int rlo[NPT], rhi[NPT];  // the rows (times heads) that see the lane's position
      float sum[NPT], old[NPT];
      uint32_t all_lo = 0, all_hi = 0x7fffffffu, some_lo = 0x7fffffffu, some_hi = 0;
#pragma unroll
      for (int t = 0; t < NPT; ++t) {
        const int tok = base + 16 * t, j = tok + col;
        sum[t] = old[t] = 0.0f;
        rlo[t] = 0;
        rhi[t] = 0x7fffffff;  // a column that is no position: its sum goes nowhere
        int64_t lo = a.causal ? max(j - before, (int64_t)0) : 0;
        int64_t hi = a.window > 0 ? min(j + a.window - before, (int64_t)n) : n;
        if (hi <= lo) lo = hi = 0;
        uint32_t w[NG], p[NG];
#pragma unroll
        for (int k = 0; k < NG; ++k) w[k] = p[k] = 0;
        if (__ballot(j < E && hi > lo)) {  // tables need not name pages that no row sees
          const int pg = __builtin_amdgcn_readfirstlane(table[tok >> a.ps_log2]);
          if (pg >= 0 && pg < a.pages) {
            const char* blk = a.pool + ((int64_t)pg * a.nkv + h) * a.block;
            const int at = (tok & (ps - 1)) + col;
            ld_words<NG>(blk + P::kc() + at * (D / 2) + g * NG * 4, w);
            ld_words<NG>(blk + P::kp(ps) + at * NG * 4, p);
            if (j < E) {
              old[t] = acc[j];
              some_lo = min(some_lo, hi > lo ? (uint32_t)(lo * a.gs) : 0x7fffffffu);
              some_hi = max(some_hi, (uint32_t)(hi * a.gs));
            }
          } else {
            if (lane == 0) atomicOr(a.err, 2);
            lo = hi = 0;
          }
        } else {
          lo = hi = 0;
        }
        if (j < E) {
          rlo[t] = (int)(lo * a.gs);
          rhi[t] = (int)(hi * a.gs);
        }
        all_lo = max(all_lo, (uint32_t)rlo[t]);
        all_hi = min(all_hi, (uint32_t)rhi[t]);
        x[t].put(w, p, a.c1, g);
      }
      all_lo = wave_max_u32(all_lo);
      all_hi = wave_min_u32(all_hi);
      some_lo = wave_min_u32(some_lo);
      some_hi = wave_max_u32(some_hi);
      for (int rt = (int)(some_lo >> 4); rt * 16 < (int)some_hi; ++rt) {
        WtRows<D, T> r;
        r.load(a, o0, nr, h, rt, lane);
        const bool whole = rt * 16 >= (int)all_lo && min(rt * 16 + 16, nr) <= (int)all_hi;
#pragma unroll
        for (int t = 0; t < NPT; ++t) {
          const kh_f32x4 zero = {0, 0, 0, 0};
          kh_f32x4 y = mfma16(r.base, x[t].m, zero);
#pragma unroll
          for (int j = 0; j < NG; ++j) {
            kh_f32x4 c = zero;
#pragma unroll
            for (int k = NQ - 1; k >= 0; --k) c = mfma16(r.q[j][k], x[t].c[j], c);
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = fmaf(x[t].s[j], c[i], y[i]);
          }
          float w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_exp2f(y[i]);
          if (!whole) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int rr = rt * 16 + 4 * g + i;
              w[i] = rr >= rlo[t] && rr < rhi[t] ? w[i] : 0.0f;
            }
          }
          sum[t] += (w[0] + w[1]) + (w[2] + w[3]);
        }
      }
#pragma unroll
      for (int t = 0; t < NPT; ++t) {
        const int j = base + 16 * t + col;
        const float s = across_groups_sum(sum[t]);
        if (g == 0 && j < E && rhi[t] > rlo[t]) acc[j] = old[t] + s;
      }
    }
  }
}

template <int D, typename T>
static int wt_launch(const WtArgs& a, int64_t max_len, hipStream_t st) {
  constexpr int NPT = 2, BP = 16 * NPT * kWtWaves;
  const int64_t most = std::min(std::min(max_len, a.acc_cols), a.cols << a.ps_log2);
  const dim3 g((unsigned)std::max<int64_t>(std::min<int64_t>((most + BP - 1) / BP, 65535), 1), (unsigned)a.nkv,
               (unsigned)std::min<int64_t>(a.batch, 65535));
  hipLaunchKernelGGL((paged_weights_kernel<D, T, NPT>), g, dim3(64 * kWtWaves), 0, st, a);
  KH_LAUNCHED();
  return KH_OK;
}
template <typename T>
static int wt_launch_d(int d, const WtArgs& a, int64_t max_len, hipStream_t st) {
  if (d == 64) return wt_launch<64, T>(a, max_len, st);
  if (d == 128) return wt_launch<128, T>(a, max_len, st);
  return wt_launch<256, T>(a, max_len, st);
}

static int wt_shape(const kh_paged_kv* c, int dtype, int64_t rows, int64_t batch, int num_heads, int64_t max_rows,
                    int64_t max_len) {
  KH_CHECK_ARG(c != nullptr, "null handle");
  KH_CHECK_ARG(dtype == KH_DT_F32 || dtype == KH_DT_BF16, "dtype %d: f32 and BF16 are supported", dtype);
  KH_CHECK_ARG(rows >= 0 && rows < (int64_t)1 << 31 && batch >= 0 && batch < (int64_t)1 << 31,
               "rows %lld, batch %lld not in [0,2^31)", (long long)rows, (long long)batch);
  KH_CHECK_ARG(num_heads >= c->nkv && num_heads % c->nkv == 0 && num_heads <= 65536,
               "num_heads %d is no multiple of the cache's %d", num_heads, c->nkv);
  KH_CHECK_ARG(rows * (num_heads / c->nkv) < ((int64_t)1 << 31) - 64, "%lld rows of %d heads: too many for one call",
               (long long)rows, num_heads);
  KH_CHECK_ARG(max_rows >= 0 && max_len >= 0, "max_rows %lld, max_len %lld", (long long)max_rows, (long long)max_len);
  return KH_OK;
}

}  // namespace kh

using namespace kh;

extern "C" int kh_paged_kv_weights_workspace(const kh_paged_kv* c, int dtype, int64_t rows, int64_t batch,
                                             int num_heads, int64_t max_rows, int64_t max_len, int64_t* bytes) {
  KH_CHECK_ARG(bytes != nullptr, "null output");
  const int rc = wt_shape(c, dtype, rows, batch, num_heads, max_rows, max_len);
  if (rc != KH_OK) return rc;
  *bytes = 0;
  return KH_OK;
}

extern "C" int kh_paged_kv_weights(const kh_paged_kv* c, int dtype, const void* q_dev, int64_t q_row_stride,
                                   int64_t q_head_stride, int num_heads, int64_t rows, const int64_t* off_dev,
                                   int64_t batch, const int64_t* len_dev, const int32_t* table_dev,
                                   int64_t table_cols, int64_t table_stride, int64_t max_rows, int64_t max_len,
                                   float scale, int causal, int64_t window, const float* lse_dev, float* acc_dev,
                                   int64_t acc_cols, void* ws_dev, int64_t ws_bytes, void* stream) {
  const int rc = wt_shape(c, dtype, rows, batch, num_heads, max_rows, max_len);
  if (rc != KH_OK) return rc;
  KH_CHECK_ARG(table_cols >= 1 && table_stride >= table_cols, "page table of %lld columns, %lld apart",
               (long long)table_cols, (long long)table_stride);
  KH_CHECK_ARG(table_cols <= (INT32_MAX - 64) >> c->ps_log2, "a page table of %lld columns holds 2^31 positions",
               (long long)table_cols);
  KH_CHECK_ARG(std::isfinite(scale * kLog2e) && scale > 0, "scale must be positive and finite");
  KH_CHECK_ARG(window >= 0 && (window == 0 || causal), "a window (%lld) needs causal attention", (long long)window);
  KH_CHECK_ARG(q_row_stride >= 0 && q_head_stride >= 0, "negative stride");
  KH_CHECK_ARG(acc_cols >= 1, "weights of %lld columns", (long long)acc_cols);
  if (rows == 0 || batch == 0) return KH_OK;
  KH_CHECK_ARG(q_dev && off_dev && len_dev && table_dev && lse_dev && acc_dev, "null argument");
  KH_ON_DEVICE(c->device, "the cache");
  WtArgs a;
  a.pool = c->pool;
  a.block = c->block;
  a.pages = c->pages;
  a.nkv = c->nkv;
  a.ps_log2 = c->ps_log2;
  a.err = c->err;
  a.q = q_dev;
  a.qs = q_row_stride;
  a.qh = q_head_stride;
  a.off = off_dev;
  a.len = len_dev;
  a.batch = batch;
  a.rows = rows;
  a.table = table_dev;
  a.cols = table_cols;
  a.table_stride = table_stride;
  a.nh = num_heads;
  a.gs = num_heads / c->nkv;
  a.c1 = scale * kLog2e;
  a.causal = causal ? 1 : 0;
  a.window = window <= INT32_MAX ? window : 0;  // wider than a table hides nothing
  a.lse = lse_dev;
  a.acc = acc_dev;
  a.acc_cols = acc_cols;
  a.qvec = aligned16(q_dev, dtype, q_row_stride, q_head_stride) ? 1 : 0;
  return dtype == KH_DT_F32 ? wt_launch_d<float>(c->d, a, max_len, as_stream(stream))
                            : wt_launch_d<uint16_t>(c->d, a, max_len, as_stream(stream));
}
