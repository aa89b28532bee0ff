// paged_weights.hip -- the attention weight that cached positions get, added up (gfx950).
//
//   acc[j] += sum_i exp(c q_i . k_j - lse_i)   over the rows i (and query heads) that see position j
//
// The log-sum-exps are known, so positions are independent of each other: nothing is carried
// from one to the next, and each sum has one owner and one order.
//
// Scores come from the f16 matrix core without a rounding of either side that an f32 would not have:
// with codes c, scale s and minimum m of a group, k = s (c - 8) + m + 8 s, where s (c - 8) has 11
// significant bits, as f16 has, and
//   q . k = sum_g [sum_{d in g} q_d s_g (c_d - 8)] + sum_g m_g Q_g + sum_g 8 s_g Q_g,   Q_g = sum_{d in g} q_d
// is one chain of products, the last two sums with Q_g in three f16 terms.  A position's numbers are scaled by
// a power of two of its own, and a row's by one of its own, or by one for its tile of 16 rows where those are within
// 2^7 of each other.  What falls below f16's smallest number is lost, towards zero: less than 2^-32 of the largest number of a
// position or row, of a row that shares its scale less than 2^-25 of its own.  f32 rows take three terms; BF16 rows
// take one, which has all bits of elements down to 2^-25 of the row's largest (2^-18 with a shared scale).
//
// log2 e is rounded in c = scale log2 e and once more for the log-sum-exps: all rows share an error of 1.3e-8 lse and of up
// to 7e-8 of the score in the exponent, the size of an f32 score's own rounding.  Sums of a prompt of 4096 come out 6.7e-8
// off, 3.9e-8 in plain f32.
//
// Rows lie along the registers of a product and positions along its lanes, so that a sum over
// rows stays in its lane until the end.
#include <algorithm>
#include <cmath>

#include "paged_frag.hpp"

namespace kh {

constexpr int kWtWaves = 4;
constexpr float kWtNone = 0x1p100f;  // a log-sum-exp whose rows add nothing
constexpr float kWtLarge = 0x1p60f;    // scales up to it have finite products
constexpr int kWtNew = 3;               // steps whose time a share's next block of rows costs
constexpr int kWtNear = 7;           // powers of two between the largest and the smallest row of a tile with one scale

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
  // many rows: shares of a kv head's steps, their sums [batch][kv heads][shares][reach], and which of those a share has
  float* sums;
  int2* range;
  int shares;
  int64_t reach;
};

typedef _Float16 kh_f16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ kh_f32x4 mfma16h(const uint4& a, const uint4& b, kh_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(kh_f16x8, a), __builtin_bit_cast(kh_f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t f16x2(float x, float y) {
  const kh_f16x2 h = {(_Float16)x, (_Float16)y};
  return __builtin_bit_cast(uint32_t, h);
}
// Eight f32 in f16 terms: x = t[0] + t[1] + ..., each towards zero (one instruction a pair): three
// leave less than 2^-30 of x, or than f16's smallest number.
template <int NT>
__device__ __forceinline__ void terms8h(const float (&f)[8], uint4 (&t)[NT]) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = f[i];
#pragma unroll
  for (int k = 0; k < NT; ++k) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(r[2 * i], r[2 * i + 1]));
      const kh_f16x2 h = __builtin_bit_cast(kh_f16x2, w[i]);
      r[2 * i] -= (float)h.x;
      r[2 * i + 1] -= (float)h.y;
    }
    t[k] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
// The power of two that a number's exponent is, between 2^lo and 2^hi; 0 and subnormals: 2^lo.
__device__ __forceinline__ int exponent_of(float x) { return (int)(__float_as_uint(x) >> 23 & 0xff) - 127; }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// A tile of 16 rows (of the heads of a kv head, row after row) as first operands, lane by lane.
template <int D, typename T>
struct WtRows {
  static constexpr int NG = D / kKvGroup, NQ = sizeof(T) == 4 ? 3 : 1;
  static constexpr int NB = NG == 8 ? 2 : 1;  // operands of the sums over groups: eight numbers each
  static constexpr int NF = NG * NQ + NB;
  uint4 x[NF];      // the groups' terms, slots (0,4,1,5,2,6,3,7) of eight elements as codes_f16 gives codes; sums
  float r, nl;      // of row lane % 16: its scale, and minus its log-sum-exp in powers of two
  bool one;         // all rows have the first one's scale
  // `between` runs while the rows' loads are on their way.
  template <typename F>
  __device__ __forceinline__ void load(const WtArgs& a, int64_t o0, int nr, int h, int tile, int lane, F between) {
    const int g = lane >> 4, rr = tile * 16 + (lane & 15);
    const bool inside = rr < nr;
    const int i = (int)((uint32_t)(inside ? rr : 0) / (uint32_t)a.gs);
    const int head = h * a.gs + ((inside ? rr : 0) - i * a.gs);
    const int64_t t = o0 + i;
    const T* q = static_cast<const T*>(a.q) + t * a.qs + head * a.qh;
    Raw8<T> raw[NG];
#pragma unroll
    for (int j = 0; j < NG; ++j) raw[j].load(q + 32 * j + 8 * g, a.qvec);
    const float lse = a.lse[t * a.nh + head];
    between();
    const bool on = inside && !__builtin_isinf(lse);
    nl = on ? -lse * kLog2e : -kWtNone;
    uint32_t top = 0;  // of the row's finite elements, as an f32's bits
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      raw[j].keep(on);
      top = max(top, raw[j].largest());
    }
    if (__ballot(top >= 0x7f800000u)) {
      top = 0;
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        float f[8];
        raw[j].get(f);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t y = __float_as_uint(f[k]) & 0x7fffffffu;
          top = y < 0x7f800000u ? max(top, y) : top;
        }
      }
    }
    top = across_groups_max_u32(top);
    // elements below 2^9, so that sums of 32 are below 2^14
    int e = min(max((int)(top >> 23) - 135, -100), 118);
    const int most = (int)wave_max_u32((uint32_t)(top > 0 ? e + 128 : 0)) - 128;
    one = __ballot(top > 0 && e < most - kWtNear) == 0;
    if (one) e = max(most, -100);
    r = pow2(e);
    const float down = pow2(-e);
    float sums[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      float f[8];
      raw[j].get(f);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] *= down;
      const float s[8] = {f[0], f[4], f[1], f[5], f[2], f[6], f[3], f[7]};
      uint4 tm[NQ];
      terms8h<NQ>(s, tm);
#pragma unroll
      for (int k = 0; k < NQ; ++k) x[j * NQ + k] = tm[k];
      sums[j] = across_groups_sum(((f[0] + f[1]) + (f[2] + f[3])) + ((f[4] + f[5]) + (f[6] + f[7])));
    }
    if constexpr (NB == 1) {
#pragma unroll
      for (int j = 0; j < 4; ++j) sums[j + NG] = sums[j];  // NG is 4 or 2: of eight numbers, the minima's and the scales'
    }
    uint4 tm[3];
    terms8h<3>(sums, tm);
    const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int k = 0; k < NB; ++k) x[NG * NQ + k] = g == 0 ? tm[0] : g == 1 ? tm[1] : g == 2 ? tm[2] : zero;
  }
};

// The keys of 16 positions as second operands, a position a column: groups g0 .. g0 + N - 1 of the
// codes w, all of the pairs p; f: the position's scale, times c1.
template <int D, int N>
__device__ __forceinline__ void wt_unpack(const uint32_t (&w)[N], const uint32_t (&p)[D / kKvGroup], int g0, float c1, int g,
                                          uint4 (&c)[N], uint4 (&b)[D == 256 ? 2 : 1], float& f) {
  constexpr int NG = D / kKvGroup, NB = NG == 8 ? 2 : 1;
  float top = 0.0f;
#pragma unroll
  for (int j = 0; j < NG; ++j)  // a NaN is passed over
    top = fmaxf(top, fmaxf(8.0f * __uint_as_float(p[j] & 0xffff0000u), __builtin_fabsf(__uint_as_float(p[j] << 16))));
  const int e = max(exponent_of(top) - 13, -100);
  const float down = pow2(-e);
  f = c1 * pow2(e);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const uint32_t pj = N == NG ? p[j] : g0 == 0 ? p[j] : p[j + NG - N];
    const _Float16 s1 = (_Float16)(__uint_as_float(pj & 0xffff0000u) * down);
    const kh_f16x2 s2 = {s1, s1}, off = {(_Float16)-24.0f, (_Float16)-24.0f};
    uint32_t v[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) v[n] = __builtin_bit_cast(uint32_t, (codes_f16(w[j], n) + off) * s2);
    c[j] = make_uint4(v[0], v[1], v[2], v[3]);
  }
  uint32_t mh[NG / 2], sh[NG / 2];  // minima and 8 scales, pairs of groups
#pragma unroll
  for (int j = 0; j < NG / 2; ++j) {
    mh[j] = f16x2(__uint_as_float(p[2 * j] << 16) * down, __uint_as_float(p[2 * j + 1] << 16) * down);
    sh[j] = f16x2(__uint_as_float(p[2 * j] & 0xffff0000u) * down * 8.0f, __uint_as_float(p[2 * j + 1] & 0xffff0000u) * down * 8.0f);
  }
  if constexpr (NG == 2) b[0] = make_uint4(mh[0], sh[0], 0, 0);
  if constexpr (NG == 4) b[0] = make_uint4(mh[0], mh[1], sh[0], sh[1]);
  if constexpr (NG == 8) {
    b[0] = make_uint4(mh[0], mh[1], mh[2], mh[3]);
    b[1] = make_uint4(sh[0], sh[1], sh[2], sh[3]);
  }
  // three terms: the lanes' last group has none
  const uint32_t some = g == 3 ? 0 : 0xffffffffu;
#pragma unroll
  for (int k = 0; k < NB; ++k) b[k] = make_uint4(b[k].x & some, b[k].y & some, b[k].z & some, b[k].w & some);
}
// The two scales together: products of powers of two, so that it does not matter which rows share one.
__device__ __forceinline__ float wt_scale(float f, float r) { return fminf(f * r, 0x1.fffffep127f); }
// The weights of four rows for the lane's position.
__device__ __forceinline__ void wt_weights(const kh_f32x4& y, float f, const float (&r)[4], const float (&nl)[4], float (&w)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_exp2f(fmaf(y[i], wt_scale(f, r[i]), nl[i]));
}

// A sequence of the call.
struct WtSeq {
  const int32_t* table;
  int64_t o0, before;  // its first row; that row's position
  int n, nr, E;        // rows, times heads; positions that are added up
};
// Of rows o0 .. o1 - 1 and L cached positions, as off and len have them.
__device__ __forceinline__ bool wt_seq(const WtArgs& a, int64_t b, int64_t o0, int64_t o1, int64_t L, bool tell, WtSeq& s) {
  const int64_t cap = a.cols << a.ps_log2;
  o0 = o0 < 0 ? 0 : o0;
  o1 = o1 > a.rows ? a.rows : o1;
  if (o1 <= o0) return false;
  if (L < 0 || L > min(cap, a.acc_cols)) {
    if (tell) atomicOr(a.err, 1);
    L = L < 0 ? 0 : min(L, cap);
  }
  s.table = a.table + b * a.table_stride;
  s.o0 = o0;
  s.n = (int)(o1 - o0);
  s.nr = s.n * a.gs;
  s.before = L - s.n;
  s.E = (int)min(L, a.acc_cols);
  return true;
}
__device__ __forceinline__ bool wt_seq(const WtArgs& a, int64_t b, bool tell, WtSeq& s) {
  return wt_seq(a, b, a.off[b], a.off[b + 1], a.len[b], tell, s);
}
// The first position that some row of a sequence sees; the last one is E - 1.
__device__ __forceinline__ int wt_first(const WtArgs& a, const WtSeq& s) {
  return a.window > 0 ? (int)min(max(s.before - a.window + 1, (int64_t)0), (int64_t)s.E) : 0;
}
// The rows (times heads) that see position j: [lo, hi).
__device__ __forceinline__ void wt_span(const WtArgs& a, const WtSeq& s, int j, int& lo, int& hi) {
  const int64_t x = a.causal ? max(j - s.before, (int64_t)0) : 0;
  const int64_t y = a.window > 0 ? min(j + a.window - s.before, (int64_t)s.n) : s.n;
  const bool some = y > x;
  lo = some ? (int)(x * a.gs) : 0;
  hi = some ? (int)(y * a.gs) : 0;
}

// Leaves the weights of rows that see the lane's position, and that add anything: 0 times a NaN is one.
__device__ __forceinline__ void wt_hide(int r0, int g, int lo, int hi, const float (&nl)[4], float (&w)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int rr = r0 + 4 * g + i;
    w[i] = rr >= lo && rr < hi && nl[i] != -kWtNone ? w[i] : 0.0f;
  }
}

// ---------------------------------------------------------------- few rows
// Positions are taken in steps of 16 NPT.  A kv head's steps, of 64 sequences after each other, are cut in shares of
// the same length for waves, since contexts have every length.  A wave keeps a tile of rows, and the loads of
// a step are under way while it works on the step before.
//
// 64 contexts of up to 4095, four kv heads of 64, eight BF16 rows each: 16.5 us (1.3 TB/s).  Bounded by instructions: 90
// for the keys of 16 positions, 400 where a wave turns to other rows (a step a wave, without shares: 36 us;
// every eighth step of a sequence a wave: 22).  One sequence of 2000, 32 heads of 128: 7.5 us, the chain of lengths, table, keys.
template <int D, typename T, int NPT>
__global__ __launch_bounds__(64 * kWtWaves) void paged_weights_kernel(WtArgs a) {
  using R = WtRows<D, T>;
  using P = KvParts<D>;
  constexpr int NG = R::NG, NB = R::NB, STEP = 16 * NPT;
  const int lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = blockIdx.y, ps = 1 << a.ps_log2;
  struct Step {
    uint32_t w[NPT][NG], p[NPT][NG];
    int pg[NPT];
    float old[NPT];
  };
  const uint32_t share = blockIdx.x * kWtWaves + wave, shares = gridDim.x * kWtWaves;
  for (int64_t c = blockIdx.z * (int64_t)64; c < a.batch; c += gridDim.z * (int64_t)64) {
    // lane i: of sequence c + i the rows, the length and the steps, and of those up to it
    int64_t o0 = 0, o1 = 0, L = 0;
    int of = 0;
    if (c + lane < a.batch) {
      o0 = a.off[c + lane];
      o1 = a.off[c + lane + 1];
      L = a.len[c + lane];
      WtSeq s;
      if (wt_seq(a, c + lane, o0, o1, L, share == 0 && h == 0, s)) of = (s.E + STEP - 1) / STEP - wt_first(a, s) / STEP;
    }
    const int64_t upto = ((int64_t)wave_incl_scan(of >> 16) << 16) + wave_incl_scan(of & 0xffff);
    const auto lane_of = [](int64_t v, int i) {
      return (int64_t)__builtin_amdgcn_readlane((int)(v >> 32), i) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, i);
    };
    const int64_t total = lane_of(upto, 63);
    int64_t from = total * share / shares, left = total * (share + 1) / shares - from;
    if (left == 0) continue;
    for (int i = __builtin_ctzll(__ballot(upto > from)); left > 0; ++i) {
      const int n = __builtin_amdgcn_readlane(of, i);
      if (n == 0) continue;
      const int64_t before = lane_of(upto, i) - n, b = c + i;
      WtSeq s;
      wt_seq(a, b, lane_of(o0, i), lane_of(o1, i), lane_of(L, i), false, s);
      // positions that some row sees: tables need not name pages of others
      const int x0 = wt_first(a, s), x1 = s.E;
      const int skip = (int)(from - before), steps = (int)min((int64_t)(n - skip), left);
      const int first = (x0 / STEP + skip) * STEP;
      left -= steps;
      from = before + n;
      float* acc = a.acc + (b * a.nkv + h) * a.acc_cols;
      for (int tile = 0; tile * 16 < s.nr; ++tile) {
        // lane i holds the page of the i-th of 64 tiles of positions
        int pages = 0;
        const auto find = [&](int i) {
          const int64_t tok = first + (int64_t)(i * NPT + lane) * 16;
          pages = tok < x1 && tok + 16 > x0 ? s.table[max(tok, (int64_t)x0) >> a.ps_log2] : 0;
          if (tok < x1 && tok + 16 > x0 && (pages < 0 || pages >= a.pages)) {
            atomicOr(a.err, 2);
            pages = -1;
          }
        };
        const auto fetch = [&](int i, Step& k) {
#pragma unroll
          for (int t = 0; t < NPT; ++t) {
            const int tok = first + i * STEP + 16 * t;
            k.pg[t] = __builtin_amdgcn_readlane(pages, i * NPT + t & 63);
            const char* blk = a.pool + ((int64_t)max(k.pg[t], 0) * a.nkv + h) * a.block;
            const int at = (tok & (ps - 1)) + col;
            ld_words<NG>(blk + P::kc() + at * (D / 2) + g * NG * 4, k.w[t]);
            ld_words<NG>(blk + P::kp(ps) + at * NG * 4, k.p[t]);
            k.old[t] = acc[min(tok + col, s.E - 1)];
          }
        };
        R q;
        Step now, next;
        find(0);
        q.load(a, s.o0, s.nr, h, tile, lane, [&] { fetch(0, now); });
        float r[4], nl[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          r[i] = __shfl(q.r, 4 * g + i);
          nl[i] = __shfl(q.nl, 4 * g + i);
        }
        // positions that all of the tile's rows see
        const int r0 = tile * 16, r1 = min(r0 + 16, s.nr);
        const int64_t t0 = s.before + (uint32_t)r0 / (uint32_t)a.gs, t1 = s.before + (uint32_t)(r1 - 1) / (uint32_t)a.gs;
        const int64_t all0 = a.window > 0 ? max(t1 - a.window + 1, (int64_t)0) : 0, all1 = a.causal ? t0 + 1 : s.E;
        for (int i = 0; i < steps; ++i) {
          if (i + 1 < steps) {
            if (((i + 1) * NPT & 63) == 0) find(i + 1);
            fetch(i + 1, next);
          }
          const int base = first + i * STEP;
          uint32_t nan = 0;
#pragma unroll
          for (int t = 0; t < NPT; ++t)
#pragma unroll
            for (int k = 0; k < NG; ++k) nan = max(nan, now.p[t][k]);
          const bool whole = base >= all0 && min(base + STEP, s.E) <= all1 && __ballot(nan >= 0x7f800000u) == 0;
#pragma unroll
          for (int t = 0; t < NPT; ++t) {
            uint4 c[NG], sums[NB];
            float f, w[4];
            wt_unpack<D, NG>(now.w[t], now.p[t], 0, a.c1, g, c, sums, f);
            kh_f32x4 y = {0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < NB; ++k) y = mfma16h(q.x[NG * R::NQ + k], sums[k], y);
#pragma unroll
            for (int j = 0; j < NG; ++j)
#pragma unroll
              for (int k = R::NQ - 1; k >= 0; --k) y = mfma16h(q.x[j * R::NQ + k], c[j], y);
            wt_weights(y, f, r, nl, w);
            const int j = base + 16 * t + col;
            if (!whole) {
              int lo, hi;
              wt_span(a, s, j, lo, hi);
              wt_hide(r0, g, lo, hi, nl, w);
            }
            const float sum = across_groups_sum((w[0] + w[1]) + (w[2] + w[3]));
            if (g == 0 && j < s.E && now.pg[t] >= 0 && sum != 0.0f) acc[j] = now.old[t] + sum;
          }
          now = next;
        }
      }
    }
  }
}

// ---------------------------------------------------------------- many rows
// A wave keeps RT tiles of rows, and the waves of a block run the same positions: a step's 128
// (64) are unpacked once for all of them, to LDS as operands, while the step before is worked on.  The
// waves' sums of a step meet in LDS, and as many threads as positions add them up in the order of the waves.
//
// A kv head's steps, of all its blocks of rows after each other, are cut in shares of the same length for blocks, since
// a causal mask leaves blocks of rows unlike numbers of them and since each new block of rows costs a share as
// much as some steps (its rows become operands).  A share has sums of its own in the workspace;
// a second kernel adds those to acc in the order of the shares.
//
// 4096 causal BF16 rows of 32 heads of 128 over eight: 106 us and 6 for the second kernel, 650 TFLOP/s of q k, in a stream
// of calls; the first hundred calls after a pause take 122 and 6.
// Bounded by what is not a product: exponentials and sums take 14 instructions for a tile's five products, and the
// waves of a SIMD hardly hide one in the other's (11200 cycles a step of 128 positions, 5100 of them products).  Measured on the way:
// parts of 512 positions for each block of rows 220 us, equal shares 170, operands asked for a tile ahead and
// shares weighed with what a block of rows costs 126, unpacking between products 123; four waves with twice the rows 155, two
// blocks of four waves a compute unit 140.
template <int D, typename T>
struct WtShape {
  using R = WtRows<D, T>;
  static constexpr int NW = 8, KEYS = D == 256 ? 64 : 128, TK = KEYS / 16;
  static constexpr int PARTS = NW / TK, NGW = R::NG / PARTS;  // waves that unpack a tile, and groups that each takes
  static constexpr int RT = R::NF <= 7 ? 4 : R::NF <= 13 ? 2 : 1;
  static constexpr int RB = 16 * RT * NW;                 // rows of a block
  static constexpr int NK = R::NG + R::NB;                // operands of a tile of positions
  static constexpr int kStep = TK * NK * 1024;            // bytes of a step
  static constexpr int kLds = 2 * kStep + 2 * KEYS * 4 + 2 * NW * KEYS * 4;  // and the scales, and the waves' sums
};

template <int D, typename T>
__global__ __launch_bounds__((64 * WtShape<D, T>::NW), 2) void paged_weights_tiles_kernel(WtArgs a) {
  using R = WtRows<D, T>;
  using S = WtShape<D, T>;
  using P = KvParts<D>;
  constexpr int NG = R::NG, NB = R::NB, NW = S::NW, KEYS = S::KEYS, TK = S::TK, RT = S::RT, RB = S::RB, NK = S::NK;
  constexpr int NGW = S::NGW;
  extern __shared__ __align__(16) char s_buf[];
  float* s_f = reinterpret_cast<float*>(s_buf + 2 * S::kStep);  // [2][KEYS]
  float* s_sum = s_f + 2 * KEYS;                                // [2][NW][KEYS]
  __shared__ int s_state[2][TK];  // of a step's tiles: 1 where a key holds a NaN or has a large scale, 2 and 3 where there is no page
  const int lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15, tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ps = 1 << a.ps_log2, utile = wave / S::PARTS, ugroup = wave % S::PARTS * NGW;
  // the kv head varies fastest: there are eight XCDs, and each keeps its heads' pages
  const int h = (int)(blockIdx.x % (uint32_t)a.nkv), share = (int)(blockIdx.x / (uint32_t)a.nkv);
  for (int64_t b = blockIdx.y; b < a.batch; b += gridDim.y) {
    WtSeq s;
    if (!wt_seq(a, b, tid == 0 && blockIdx.x == 0, s)) continue;
    const int nrb = (int)(((int64_t)s.nr + RB - 1) / RB);
    // positions [x, y) that some of rows r0 .. r1 - 1 see, and the steps that hold them
    const auto seen = [&](int r0, int r1, int& x, int& y) {
      const int64_t q0 = s.before + (uint32_t)r0 / (uint32_t)a.gs, q1 = s.before + ((uint32_t)r1 - 1) / (uint32_t)a.gs;
      const int64_t lo = a.window > 0 ? max(q0 - a.window + 1, (int64_t)0) : 0;
      const int64_t hi = min(a.causal ? q1 + 1 : (int64_t)s.E, (int64_t)s.E);
      x = hi > lo ? (int)lo : 0;
      y = hi > lo ? (int)hi : 0;
    };
    const auto steps = [&](int rb, int& x, int& y) {
      seen(rb * RB, (int)min((int64_t)rb * RB + RB, (int64_t)s.nr), x, y);
      return (y + KEYS - 1) / KEYS - x / KEYS;
    };
    // a sequence longer than the guess is one share
    const int shares = a.shares > 1 && s.E <= a.reach ? a.shares : 1;
    if (share >= shares) continue;
    int rb = 0;              // the share's first block of rows,
    int64_t from = 0, left;  // how many of its steps (and kWtNew) others have, and how many are the share's
    if (shares == 1) {
      left = INT64_MAX;
    } else {
      const auto count = [&](int c) {
        int x, y;
        const int of = c + lane < nrb ? steps(c + lane, x, y) : 0;
        return of > 0 ? of + kWtNew : 0;
      };
      int n = count(0), upto = wave_incl_scan(n);
      int64_t total = __builtin_amdgcn_readlane(upto, 63);
      for (int c = 64; c < nrb; c += 64) total += __builtin_amdgcn_readlane(wave_incl_scan(count(c)), 63);
      from = total * (uint32_t)share / (uint32_t)shares;
      left = total * (uint32_t)(share + 1) / (uint32_t)shares - from;
      for (;;) {
        const uint64_t here = __ballot(upto > from);
        if (left == 0 || here) {
          const int i = here ? __builtin_ctzll(here) : 0;
          rb += i;
          from -= __builtin_amdgcn_readlane(upto - n, i);
          break;
        }
        from -= __builtin_amdgcn_readlane(upto, 63);
        rb += 64;
        n = count(rb);
        upto = wave_incl_scan(n);
      }
    }
    float* out = a.acc + (b * a.nkv + h) * a.acc_cols;
    if (shares > 1) {
      const int64_t row = (b * a.nkv + h) * a.shares + share;
      out = a.sums + row * a.reach;
      int p0 = 0x7fffffff, p1 = 0;
      int64_t n = left, skip = from;
      for (int i = rb; n > 0; ++i) {
        int x, y;
        const int of = steps(i, x, y);
        if (of == 0) continue;
        const int i0 = (int)min(skip, (int64_t)of), i1 = (int)min(skip + n, (int64_t)of);
        if (i1 > i0) {
          p0 = min(p0, (x / KEYS + i0) * KEYS);
          p1 = max(p1, min((x / KEYS + i1) * KEYS, s.E));
        }
        n -= of + kWtNew - skip;
        skip = 0;
      }
      p0 = min(p0, p1);  // a share may have no steps
      if (tid == 0) a.range[row] = make_int2(p0, p1);
      if (tid < KEYS)
        for (int j = p0 + tid; j < p1; j += KEYS) out[j] = 0.0f;
    }
    // sums go to out[j], by the same thread each time
    for (; rb < nrb && left > 0; ++rb) {
      int tlo, thi;
      const int of = steps(rb, tlo, thi);
      if (of == 0) continue;
      const int sb = tlo / KEYS + (int)min(from, (int64_t)of), se = tlo / KEYS + (int)(left < of - from ? from + left : of);
      left -= of + kWtNew - from;
      from = 0;
      if (se <= sb) continue;
      const int w0 = (rb * NW + wave) * RT * 16;  // the wave's first row
      // positions that some of the wave's rows see, and those that all of them see
      uint32_t lo = 0x7fffffffu, hi = 0, all_lo = 0, all_hi = 0x7fffffffu;
      if (w0 < s.nr) {
        const int64_t i0 = (uint32_t)w0 / (uint32_t)a.gs, i1 = (uint32_t)(min(w0 + RT * 16, s.nr) - 1) / (uint32_t)a.gs;
        const int64_t L = s.before + s.n, q0 = s.before + i0, q1 = s.before + i1;
        const int64_t x = a.window > 0 ? max(q0 - a.window + 1, (int64_t)0) : 0, xa = a.window > 0 ? max(q1 - a.window + 1, (int64_t)0) : 0;
        const int64_t y = a.causal ? min(q1 + 1, L) : L, ya = a.causal ? min(q0 + 1, L) : L;
        if (y > x) lo = (uint32_t)x, hi = (uint32_t)y;
        all_lo = (uint32_t)xa;
        all_hi = (uint32_t)max(ya, (int64_t)0);
      }
      __syncthreads();  // the last block of rows is done with LDS

      // lane i holds the page of the wave's tile of the i-th of 64 steps
      int pages = 0;
      const auto find = [&](int st) {
        const int tok = (int)((uint32_t)(st + lane) * KEYS) + utile * 16;
        pages = tok + 16 > tlo && tok < thi ? s.table[max(tok, tlo) >> a.ps_log2] : 0;
        if (tok + 16 > tlo && tok < thi && (pages < 0 || pages >= a.pages)) {
          atomicOr(a.err, 2);
          pages = -1;
        }
      };
      // of a step's tile: what it holds, and its page
      struct Tile {
        uint32_t w[NGW], p[NG];
        int pg;
      } now, next;
      const auto load = [&](int st, Tile& k) {
        k.pg = __builtin_amdgcn_readlane(pages, (st - sb) & 63);
        const int tok = st * KEYS + utile * 16;
        const char* blk = a.pool + ((int64_t)max(k.pg, 0) * a.nkv + h) * a.block;
        const int at = (tok & (ps - 1)) + col;
        ld_n<NGW>(blk + P::kc() + at * (D / 2) + (g * NG + ugroup) * 4, k.w);
        ld_words<NG>(blk + P::kp(ps) + at * NG * 4, k.p);
      };
      // without branches, so that it can lie between products: all waves of a tile write what the tile has one of
      const auto unpack = [&](int st, const Tile& k) {
        char* to = s_buf + (st & 1) * S::kStep + utile * NK * 1024 + lane * 16;
        float f;
        uint4 c[NGW], bb[NB];
        wt_unpack<D, NGW>(k.w, k.p, ugroup, a.c1, g, c, bb, f);
#pragma unroll
        for (int i = 0; i < NGW; ++i) *reinterpret_cast<uint4*>(to + (ugroup + i) * 1024) = c[i];
#pragma unroll
        for (int i = 0; i < NB; ++i) *reinterpret_cast<uint4*>(to + (NG + i) * 1024) = bb[i];
        s_f[(st & 1) * KEYS + utile * 16 + col] = f;
        uint32_t nan = 0;
#pragma unroll
        for (int i = 0; i < NG; ++i) nan = max(nan, k.p[i]);
        const uint64_t rare = __ballot(nan >= 0x7f800000u || f > kWtLarge);
        s_state[st & 1][utile] = (k.pg >> 31 & 2) | ((uint32_t)rare | (uint32_t)(rare >> 32) ? 1 : 0);
      };
      find(sb);
      load(sb, now);

      R q[RT];
      float nl[RT][4], r[RT];
      bool one = true;
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        q[t].load(a, s.o0, s.nr, h, w0 / 16 + t, lane, [] {});
        r[t] = __shfl(q[t].r, 0);
        one = one && q[t].one && r[t] <= kWtLarge;
      }
#pragma unroll
      for (int t = 0; t < RT; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) nl[t][i] = __shfl(q[t].nl, 4 * g + i);
      }
      unpack(sb, now);
      if (sb + 1 < se) load(sb + 1, now);

      float old = 0.0f;  // what out holds of a step's positions
      const auto add = [&](int st) {
        const float* x = s_sum + (st & 1) * NW * KEYS + tid;
        float w = 0.0f;
#pragma unroll
        for (int k = 0; k < NW; ++k) w += x[k * KEYS];
        const int j = st * KEYS + tid;
        if (j < s.E && w != 0.0f) out[j] = old + w;
      };
      for (int st = sb; st < se; ++st) {
        __syncthreads();
        if (tid < KEYS) {
          if (st > sb) add(st - 1);
          old = out[min(st * KEYS + tid, s.E - 1)];
        }
        const int first = st * KEYS;
        const char* buf = s_buf + (st & 1) * S::kStep + lane * 16;
        const float* fs = s_f + (st & 1) * KEYS;
        float* sums = s_sum + ((st & 1) * NW + wave) * KEYS;
        int state = 0;
#pragma unroll
        for (int k = 0; k < TK; ++k) state |= s_state[st & 1][k];
        state = __builtin_amdgcn_readfirstlane(state);
        if (st + 2 < se) {
          if (((st + 2 - sb) & 63) == 0) find(st + 2);
          load(st + 2, next);
        }
        // The next step goes to the other buffer (after the last one, what nobody reads).
        const auto scores = [&](int k, kh_f32x4 (&y)[RT]) {
#pragma unroll
          for (int t = 0; t < RT; ++t) y[t] = kh_f32x4{0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            const uint4 c = *reinterpret_cast<const uint4*>(buf + (k * NK + NG + i) * 1024);
#pragma unroll
            for (int t = 0; t < RT; ++t) y[t] = mfma16h(q[t].x[NG * R::NQ + i], c, y[t]);
          }
#pragma unroll
          for (int j = 0; j < NG; ++j) {
            const uint4 c = *reinterpret_cast<const uint4*>(buf + (k * NK + j) * 1024);
#pragma unroll
            for (int i = R::NQ - 1; i >= 0; --i)
#pragma unroll
              for (int t = 0; t < RT; ++t) y[t] = mfma16h(q[t].x[j * R::NQ + i], c, y[t]);
          }
        };
        if (first >= (int)hi || first + KEYS <= (int)lo) {  // the wave's rows see nothing of it
          unpack(st + 1, now);
#pragma unroll
          for (int i = lane; i < KEYS; i += 64) sums[i] = 0.0f;
        } else if (one && state == 0 && first >= (int)all_lo && first + KEYS <= (int)all_hi) {
          // Every row sees every position.  A tile's products lie between the rest of the work of the tile before
          // (the first one's between the unpacking), and an operand of the next tile is asked for as soon as this
          // tile's is used: the compiler would ask for it just before it is needed, and wait.
          const auto at = [](int o) { return o < NB ? NG + o : o - NB; };
          const auto operand = [&](int k, int o) { return *reinterpret_cast<const uint4*>(buf + (k * NK + at(o)) * 1024); };
          uint4 c[NK];
#pragma unroll
          for (int o = 0; o < NK; ++o) c[o] = operand(0, o);
          kh_f32x4 y[2][RT];
          float f[2], sum = 0.0f;
          const auto finish = [&](int k, int t) {
            const float fr = f[k & 1] * r[t];  // finite: see `one` and the tiles' states
            float w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_exp2f(fmaf(y[k & 1][t][i], fr, nl[t][i]));
            sum = t == 0 ? (w[0] + w[1]) + (w[2] + w[3]) : sum + ((w[0] + w[1]) + (w[2] + w[3]));
          };
          __builtin_amdgcn_sched_barrier(0);
          unpack(st + 1, now);
#pragma unroll
          for (int k = 0; k < TK; ++k) {
            f[k & 1] = fs[k * 16 + col];
#pragma unroll
            for (int o = 0; o < NK; ++o) {
              constexpr int NQ = R::NQ;
#pragma unroll
              for (int i = o < NB ? 0 : NQ - 1; i >= 0; --i)
#pragma unroll
                for (int t = 0; t < RT; ++t)
                  y[k & 1][t] = mfma16h(q[t].x[o < NB ? NG * NQ + o : at(o) * NQ + i], c[o], o == 0 ? kh_f32x4{0, 0, 0, 0} : y[k & 1][t]);
              if (k + 1 < TK) c[o] = operand(k + 1, o);
              if (k > 0) {
#pragma unroll
                for (int t = 0; t < RT; ++t)
                  if (t * NK / RT == o) finish(k - 1, t);
                if (o == NK - 1) sums[(k - 1) * 16 + col] = across_groups_sum(sum);
              }
#pragma unroll
              for (int i = 0; i < RT * (o < NB ? 1 : NQ); ++i) {
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                if (k == 0) __builtin_amdgcn_sched_group_barrier(0x402, 7, 0);
                else __builtin_amdgcn_sched_group_barrier(0x402, 4, 0);
              }
              if (k > 0 || o == NK - 1) __builtin_amdgcn_sched_barrier(0);
            }
          }
#pragma unroll
          for (int t = 0; t < RT; ++t) finish(TK - 1, t);
          sums[(TK - 1) * 16 + col] = across_groups_sum(sum);
        } else {
          unpack(st + 1, now);
          for (int k = 0; k < TK; ++k) {
            const int j0 = first + k * 16;
            float sum = 0.0f;
            if (j0 < (int)hi && j0 + 16 > (int)lo && s_state[st & 1][k] < 2) {
              const float f = fs[k * 16 + col];
              const bool whole = j0 >= (int)all_lo && j0 + 16 <= (int)all_hi && s_state[st & 1][k] == 0;
              int from = 0, to = 0;
              if (!whole) wt_span(a, s, j0 + col, from, to);
              kh_f32x4 y[RT];
              scores(k, y);
#pragma unroll
              for (int t = 0; t < RT; ++t) {
                float w[4], rt[4] = {r[t], r[t], r[t], r[t]};
                if (!one) {
#pragma unroll
                  for (int i = 0; i < 4; ++i) rt[i] = __shfl(q[t].r, 4 * g + i);
                }
                wt_weights(y[t], f, rt, nl[t], w);
                if (!whole) wt_hide(w0 + 16 * t, g, from, to, nl[t], w);
                sum += (w[0] + w[1]) + (w[2] + w[3]);
              }
              sum = across_groups_sum(sum);
            }
            sums[k * 16 + col] = sum;
          }
        }
        now = next;
      }
      __syncthreads();
      if (tid < KEYS) add(se - 1);
    }
  }
}

// Adds the shares' sums to acc: each wave those of a quarter of the shares, in their order, then the four.
__global__ __launch_bounds__(256) void paged_weights_join_kernel(WtArgs a) {
  __shared__ float part[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, each = (a.shares + 3) / 4;
  for (int64_t b = blockIdx.z; b < a.batch; b += gridDim.z) {
    WtSeq s;
    if (!wt_seq(a, b, false, s) || s.E > a.reach || (int64_t)blockIdx.x * 64 >= s.E) continue;
    const int64_t row = b * a.nkv + blockIdx.y, j = (int64_t)blockIdx.x * 64 + lane;
    const float* sums = a.sums + row * a.shares * a.reach + j;
    const int2* range = a.range + row * a.shares;
    float w = 0.0f;
    for (int c0 = wave * each; c0 < min((wave + 1) * each, a.shares); c0 += 64) {
      const int n = min(min((wave + 1) * each, a.shares) - c0, 64);
      const int2 p = range[c0 + min(lane, n - 1)];
#pragma unroll 8
      for (int c = 0; c < n; ++c) {
        const int x = __builtin_amdgcn_readlane(p.x, c), y = __builtin_amdgcn_readlane(p.y, c);
        const float v = sums[(c0 + c) * a.reach];
        w += j >= x && j < y ? v : 0.0f;
      }
    }
    part[wave][lane] = w;
    __syncthreads();
    w = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
    if (wave == 0 && j < s.E && w != 0.0f) a.acc[row * a.acc_cols + j] += w;
    __syncthreads();
  }
}

// How a call is cut.
struct WtPlan {
  bool many;
  int shares;
  int64_t reach;
};
static int wt_block_rows(int d, int dtype) {
  if (dtype == KH_DT_F32) return d == 64 ? WtShape<64, float>::RB : d == 128 ? WtShape<128, float>::RB : WtShape<256, float>::RB;
  return d == 64 ? WtShape<64, uint16_t>::RB : d == 128 ? WtShape<128, uint16_t>::RB : WtShape<256, uint16_t>::RB;
}
static int wt_step(int d) { return d == 64 ? WtShape<64, float>::KEYS : d == 128 ? WtShape<128, float>::KEYS : WtShape<256, float>::KEYS; }
constexpr int64_t kWtFill = 256;      // blocks of many rows that the chip holds at once
constexpr int64_t kWtFew = 1024;      // blocks of few rows
constexpr int64_t kWtMost = 1 << 26;  // sums of shares
static WtPlan wt_plan(const kh_paged_kv* c, int dtype, int nh, int64_t rows, int64_t batch, int64_t max_rows, int64_t max_len) {
  WtPlan p;
  const int64_t gs = nh / c->nkv, rb = wt_block_rows(c->d, dtype), keys = wt_step(c->d);
  max_rows = std::min(max_rows, rows);
  max_len = std::max<int64_t>(std::min<int64_t>(max_len, INT32_MAX - 64), 1);
  p.many = max_rows * gs > 16;
  p.reach = (max_len + 63) / 64 * 64;
  // the number of shares that lets the rounds of blocks on the chip end first
  const int64_t heads = batch * c->nkv, steps = (max_rows * gs + rb - 1) / rb * ((max_len + keys - 1) / keys);
  int64_t least = INT64_MAX;
  p.shares = 1;
  for (int64_t n = 1; n <= kWtFill && n <= steps && (n == 1 || n * heads <= std::min(4 * kWtFill, kWtMost / p.reach)); ++n) {
    const int64_t time = (heads * n + kWtFill - 1) / kWtFill * ((steps + n - 1) / n + 2 * kWtNew);
    if (time < least) least = time, p.shares = (int)n;
  }
  return p;
}
static int64_t wt_space(const WtPlan& p, int64_t heads) {
  return p.many && p.shares > 1 ? heads * p.shares * (p.reach * 4 + 8) : 0;
}

template <int D, typename T>
static int wt_launch(const WtArgs& a, bool many, int64_t max_len, hipStream_t st) {
  const unsigned seqs = (unsigned)std::min<int64_t>(a.batch, 65535);
  if (!many) {
    constexpr int NPT = 2, BP = 16 * NPT * kWtWaves;
    const int64_t most = std::min(std::min(max_len, a.acc_cols), a.cols << a.ps_log2);
    // as many waves as the chip holds at once, if there are steps for them
    const int64_t groups = std::min<int64_t>((a.batch + 63) / 64, 65535);
    const int64_t blocks = std::min((most + BP - 1) / BP * std::min<int64_t>(a.batch, 64), std::max<int64_t>(kWtFew / (a.nkv * groups), 1));
    const dim3 g((unsigned)std::max<int64_t>(blocks, 1), (unsigned)a.nkv, (unsigned)groups);
    hipLaunchKernelGGL((paged_weights_kernel<D, T, NPT>), g, dim3(64 * kWtWaves), 0, st, a);
  } else {
    hipLaunchKernelGGL((paged_weights_tiles_kernel<D, T>), dim3((unsigned)((int64_t)a.shares * a.nkv), seqs),
                       dim3((64 * WtShape<D, T>::NW)), (WtShape<D, T>::kLds), st, a);
    if (a.shares > 1)
      hipLaunchKernelGGL(paged_weights_join_kernel, dim3((unsigned)(a.reach / 64), (unsigned)a.nkv, seqs), dim3(256), 0, st, a);
  }
  KH_LAUNCHED();
  return KH_OK;
}
template <typename T>
static int wt_launch_d(int d, const WtArgs& a, bool many, int64_t max_len, hipStream_t st) {
  if (d == 64) return wt_launch<64, T>(a, many, max_len, st);
  if (d == 128) return wt_launch<128, T>(a, many, max_len, st);
  return wt_launch<256, T>(a, many, max_len, st);
}

template <int D>
static int wt_allow_lds() {
  KH_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&paged_weights_tiles_kernel<D, float>),
                             hipFuncAttributeMaxDynamicSharedMemorySize, WtShape<D, float>::kLds));
  KH_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&paged_weights_tiles_kernel<D, uint16_t>),
                             hipFuncAttributeMaxDynamicSharedMemorySize, WtShape<D, uint16_t>::kLds));
  return KH_OK;
}
int paged_weights_prepare(int d) { return d == 64 ? wt_allow_lds<64>() : d == 128 ? wt_allow_lds<128>() : wt_allow_lds<256>(); }

static int wt_shape(const kh_paged_kv* c, int dtype, int64_t rows, int64_t batch, int num_heads, int64_t max_rows,
                    int64_t max_len) {
  KH_CHECK_ARG(c != nullptr, "null handle");
  KH_CHECK_ARG(dtype == KH_DT_F32 || dtype == KH_DT_BF16, "dtype %d: f32 and BF16 are supported", dtype);
  KH_CHECK_ARG(rows >= 0 && rows < (int64_t)1 << 31 && batch >= 0 && batch < (int64_t)1 << 31,
               "rows %lld, batch %lld not in [0,2^31)", (long long)rows, (long long)batch);
  KH_CHECK_ARG(num_heads >= c->nkv && num_heads % c->nkv == 0 && num_heads <= 65536,
               "num_heads %d is no multiple of the cache's %d", num_heads, c->nkv);
  KH_CHECK_ARG(rows * (num_heads / c->nkv) < ((int64_t)1 << 31) - 1024, "%lld rows of %d heads: too many for one call",
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
  if (rows && batch) *bytes = wt_space(wt_plan(c, dtype, num_heads, rows, batch, max_rows, max_len), batch * c->nkv);
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
  KH_CHECK_ARG(table_cols <= (INT32_MAX - 256) >> c->ps_log2, "a page table of %lld columns holds 2^31 positions",
               (long long)table_cols);
  KH_CHECK_ARG(std::isfinite(scale * kLog2e) && scale > 0, "scale must be positive and finite");
  KH_CHECK_ARG(window >= 0 && (window == 0 || causal), "a window (%lld) needs causal attention", (long long)window);
  KH_CHECK_ARG(q_row_stride >= 0 && q_head_stride >= 0, "negative stride");
  KH_CHECK_ARG(acc_cols >= 1, "weights of %lld columns", (long long)acc_cols);
  if (rows == 0 || batch == 0) return KH_OK;
  KH_CHECK_ARG(q_dev && off_dev && len_dev && table_dev && lse_dev && acc_dev, "null argument");
  const WtPlan p = wt_plan(c, dtype, num_heads, rows, batch, max_rows, max_len);
  const int64_t need = wt_space(p, batch * c->nkv);
  if (need > 0 && (!ws_dev || ws_bytes < need)) {
    set_error("the workspace holds %lld bytes, %lld are needed", (long long)(ws_dev ? ws_bytes : 0), (long long)need);
    return KH_ERR_CAPACITY;
  }
  KH_CHECK_ARG((reinterpret_cast<uintptr_t>(ws_dev) & 15) == 0, "the workspace must be 16-byte aligned");
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
  a.sums = static_cast<float*>(ws_dev);
  a.range = reinterpret_cast<int2*>(a.sums + batch * c->nkv * p.shares * p.reach);
  a.shares = p.shares;
  a.reach = p.reach;
  return dtype == KH_DT_F32 ? wt_launch_d<float>(c->d, a, p.many, max_len, as_stream(stream))
                            : wt_launch_d<uint16_t>(c->d, a, p.many, max_len, as_stream(stream));
}
