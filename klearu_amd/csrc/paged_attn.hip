// paged_attn.hip -- attention over the paged 4-bit cache (gfx950).
//
// For row i of a sequence with n new rows and L cached positions (the new rows'
// own among them), at position p = L - n + i:
//   o = sum_j softmax_j(scale q . k_j) v_j,  lse = log sum_j exp(scale q . k_j)
// over the positions j that the row sees: j < L, with `causal` j <= p, with a
// window w also j > p - w.  A row that sees nothing gives 0 and -inf.
//
// The codes go into the matrix cores as they are, as BF16 numbers B + c.  For BF16 rows B is
// 16: a nibble three bits up behind the bits 0x418.  f32 rows convert the codes (B = 0): their
// bits do not last through sums of the size of 16s.  With group sums A_g = sum_d q_d (B + c_d)
//   q . k = sum_g s_g A_g + sum_g (m_g - B s_g) Q_g,   Q_g = sum_{d in g} q_d
// where the second sum is one more product, of the (s, m) pairs as they lie in
// the page with (-B Q_g, Q_g) in three BF16 terms.  Values alike, with R the
// rounded products p_j s_jg that the matrix core takes:
//   o_d = sum_j R_jg (B + c_jd) - B sum_j R_jg + sum_j p_j m_jg
// where the rounding of R cancels in the Bs.  The middle sum is one more
// product with ones, per group: a group that stands for NaN touches no other.
//
// Row tiles are 16 rows of one kv head: the queries of its heads, of one
// sequence.  Scores come out of the matrix core with positions along registers
// and rows along lanes, which is the layout that the second product takes its P
// in when the positions of a step are numbered 4 g + i and 16 + 4 g + i; nothing
// is exchanged between lanes but the running maximum.
//
// Few rows (paged_rows_kernel) are bound by the cache's bytes where it is long and by a
// chain of some 6.5 us where it is short: launch, lengths, pages, codes, one step, the
// join of the waves.  32 heads of 128, BF16: eight sequences of 2048 positions (84 MB)
// 25.4 us, 131072 positions of 8 kv heads (168 MB) 48.0 + 4.6 us of join (3.5 TB/s; a copy
// runs at 4.8, read and write), 64 positions 7 us.  16 of 32 heads, f32, 2000 positions:
// 11.8 + 3.9 us (parts are cut as if all heads had work: blocks of unlisted heads stay idle).
// 16 heads of 256 over 8, eight sequences of 2048: 21.6 + 4.0 us, f32 27.5 + 4.1; no step is
// loaded ahead there, the sums and a step fill the registers.  Many f32 rows run here too: 1024
// causal rows of 32 heads of 128 over 8 take 130 us, each tile unpacks its positions for itself
// and every product has three or more terms.  Many BF16 rows: below.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "mfma.hpp"
#include "paged_kv.hpp"

namespace kh {

// Waves of a block, and waves that a SIMD's registers hold.
template <int D, typename T>
struct PaShape {
  static constexpr bool kF32 = sizeof(T) == 4;
  static constexpr int NW = D == (kF32 ? 64 : 128) ? 8 : 4;
  static constexpr int kPerSimd = D == 256 || (kF32 && D == 128) ? 1 : D == 64 && !kF32 ? 3 : 2;
  static constexpr int kAhead = D == 256 ? 0 : 1;        // steps loaded ahead of the one that is worked on
  static constexpr int kFill = 256 * 4 * kPerSimd / NW;  // blocks that the chip holds at once
  static constexpr int kOS = D + 4;                      // floats between rows in LDS: other banks for each
  static constexpr int kLds = NW * 16 * (kOS + 2) * 4;
};
constexpr int kPaStep = 32;        // positions a wave takes at a time
constexpr int kPaMaxSplit = 128;  // parts of a row that the join takes: two a lane
constexpr int kPaFine = 1024;     // positions up to which BF16 rows hold their weights in two terms
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

struct PaArgs {
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
  const int32_t* heads;
  int nsel, nh, gs;
  float c1;  // scale * log2(e)
  int causal;
  int64_t window;
  void* out;
  int64_t os, oh;
  float* lse;
  float* part_o;
  float2* part_ml;
  int nsplit, tiles;
  int share;  // 0, or the parts that a kv head's sequences get by their lengths, up to nsplit each
  int qvec, ovec;
  char* un;  // unpacked positions (tiles of many rows): un_steps steps of each sequence
  uint32_t* un_nan;
  int un_steps;
};

template <int N>
__device__ __forceinline__ void ld_words(const char* p, uint32_t (&w)[N]) {
  if constexpr (N == 2) {
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

// Eight neighbouring elements as they lie in memory.
template <typename T>
struct Raw8 {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p, bool vec) {
    if (vec) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
      float f[8];
      load8(p, false, f);
      put(f);
    }
  }
  __device__ __forceinline__ void put(const float (&f)[8]) {
    if constexpr (sizeof(T) == 4) {
      w[0] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
      w[1] = make_uint4(__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7]));
    } else {
      w[0] = make_uint4(__float_as_uint(f[0]) >> 16 | __float_as_uint(f[1]), __float_as_uint(f[2]) >> 16 | __float_as_uint(f[3]),
                        __float_as_uint(f[4]) >> 16 | __float_as_uint(f[5]), __float_as_uint(f[6]) >> 16 | __float_as_uint(f[7]));
    }
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    if constexpr (sizeof(T) == 4) {
      f[0] = __uint_as_float(w[0].x); f[1] = __uint_as_float(w[0].y); f[2] = __uint_as_float(w[0].z); f[3] = __uint_as_float(w[0].w);
      f[4] = __uint_as_float(w[1].x); f[5] = __uint_as_float(w[1].y); f[6] = __uint_as_float(w[1].z); f[7] = __uint_as_float(w[1].w);
    } else {
      f[0] = bf16_lo(w[0].x); f[1] = bf16_hi(w[0].x); f[2] = bf16_lo(w[0].y); f[3] = bf16_hi(w[0].y);
      f[4] = bf16_lo(w[0].z); f[5] = bf16_hi(w[0].z); f[6] = bf16_lo(w[0].w); f[7] = bf16_hi(w[0].w);
    }
  }
};

__device__ __forceinline__ kh_f32x4 mfma16(const uint4& a, const uint4& b, kh_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(a), as_bf16x8(b), c, 0, 0, 0);
}

// Two codes (nibble n of each half of w) as BF16 numbers BIAS + c: two instructions a pair
// behind the bits of 16, where a nibble counts ones three bits up, four by conversion.  The bias
// leaves the sums again, with the rounding errors of numbers of its size.  Errors of 150 drawn
// calls against 64 bits: f32 rows with 16 up to 1.2e-6 of the result where plain f32 has 4e-7,
// with 0 up to 4.7e-7 at 1 to 3 % more time (1024 f32 rows of 32 heads of 128: 132 us, 129 with
// 16); log-sum-exps of BF16 rows with 128 up to 2.3e-6, with 16 below 1e-6 at 1 to 2 %.
template <int BIAS>
__device__ __forceinline__ uint32_t codes2(uint32_t w, int n) {
  if constexpr (BIAS == 16) return ((n == 0 ? w << 3 : w >> (4 * n - 3)) & 0x00780078u) | 0x41804180u;
  const uint32_t x = (n & 1 ? w >> 4 : w) & 0x0f0f0f0fu;
  return cvt_bf16x2((float)(x >> (n & 2 ? 8 : 0) & 0xffu), (float)(x >> (n & 2 ? 24 : 16) & 0xffu));
}

// Eight f32 in BF16 terms: x = t[0] + t[1] + ... to 8 more bits each.
template <int NT>
__device__ __forceinline__ void terms8(const float (&f)[8], uint4 (&t)[NT]) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = f[i];
#pragma unroll
  for (int k = 0; k < NT; ++k) {
    t[k] = make_uint4(cvt_bf16x2(r[0], r[1]), cvt_bf16x2(r[2], r[3]), cvt_bf16x2(r[4], r[5]), cvt_bf16x2(r[6], r[7]));
    if (k + 1 < NT) {
      r[0] -= bf16_lo(t[k].x); r[1] -= bf16_hi(t[k].x); r[2] -= bf16_lo(t[k].y); r[3] -= bf16_hi(t[k].y);
      r[4] -= bf16_lo(t[k].z); r[5] -= bf16_hi(t[k].z); r[6] -= bf16_lo(t[k].w); r[7] -= bf16_hi(t[k].w);
    }
  }
}

// c plus the two BF16 numbers of w.
__device__ __forceinline__ float add2(uint32_t w, float c) {
  typedef __bf16 v2 __attribute__((ext_vector_type(2)));
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2, w), __builtin_bit_cast(v2, 0x3f803f80u), c, false);
}

// Over the four lanes of a column, one in each group of sixteen: a row of
// sixteen is exchanged with its neighbour, then halves of the wave.
template <typename F>
__device__ __forceinline__ float across_groups(float v, F f) {
  const uint32_t u = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t w = __float_as_uint(f(__uint_as_float(a[0]), __uint_as_float(a[1])));
  const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float across_groups_max(float v) {
  return across_groups(v, [](float x, float y) { return fmaxf(x, y); });
}
__device__ __forceinline__ float across_groups_sum(float v) {
  return across_groups(v, [](float x, float y) { return x + y; });
}

__device__ __forceinline__ uint32_t across_groups_or(uint32_t u) {
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t w = a[0] | a[1];
  const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return b[0] | b[1];
}

// a times the lane's row's (of sixteen) lane N of s; c plus a times the quad's lane N of s.
template <int N>
__device__ __forceinline__ float mul_row(float a, uint32_t s) {
  return a * __int_as_float(__builtin_amdgcn_mov_dpp((int)s, 0x150 + N, 0xf, 0xf, true));
}
template <int N>
__device__ __forceinline__ float fma_quad(float a, uint32_t s, float c) {
  return fmaf(__int_as_float(__builtin_amdgcn_mov_dpp((int)s, N * 0x55, 0xf, 0xf, true)), a, c);
}

// What a wave holds of 32 positions, two tiles of 16.
template <int D>
struct PaStepData {
  static constexpr int NG = D / kKvGroup, HN = D / 64;
  uint32_t kw[2][NG];      // codes of key lane % 16, the lane group's words
  uint32_t kpa[2][NG];     // pairs of that key
  uint32_t kpc[2][NG];     // pairs of key 4 g + lane % 4
  uint32_t vw[2][2 * HN];  // codes of positions 4 g .. 4 g + 3
  uint32_t vp[2][4];       // pairs of group lane % NG, those positions
};

// Where a lane's words lie in a block, from the first of 16 positions on.
template <int D>
struct PaLane {
  static constexpr int NG = D / kKvGroup, HN = D / 64;
  uint32_t kc, kpa, kpc, vc, vp;
  __device__ __forceinline__ PaLane(int lane, int ps) {
    using P = KvParts<D>;
    const int g = lane >> 4, r = lane & 15;
    kc = P::kc() + r * (D / 2) + g * NG * 4;
    kpa = P::kp(ps) + r * NG * 4;
    kpc = P::kp(ps) + (4 * g + (lane & 3)) * NG * 4;
    vc = P::vc(ps) + (g * 16 + r) * (HN * 8);
    vp = P::vp(ps) + ((r & (NG - 1)) * ps + 4 * g) * 4;
  }
};

// Tile T of a step; blk: the block of its positions, in: the first one's place in the page (both the wave's).
template <int D, int T>
__device__ __forceinline__ void pa_load(const char* blk, int in, const PaLane<D>& o, PaStepData<D>& x) {
  constexpr int NG = D / kKvGroup, HN = D / 64;
  ld_words<NG>(blk + in * (D / 2) + o.kc, x.kw[T]);
  ld_words<NG>(blk + in * (NG * 4) + o.kpa, x.kpa[T]);
  ld_words<NG>(blk + in * (NG * 4) + o.kpc, x.kpc[T]);
  ld_words<2 * HN>(blk + in * (D / 2) + o.vc, x.vw[T]);
  ld_words<4>(blk + in * 4 + o.vp, x.vp[T]);
}

// Whether head h of row t is in the row's list; every lane of the wave takes part.
__device__ __forceinline__ bool pa_selected(const PaArgs& a, int64_t t, int h, int lane) {
  for (int j0 = 0; j0 < a.nsel; j0 += 64) {
    const bool hit = j0 + lane < a.nsel && a.heads[t * a.nsel + j0 + lane] == h;
    if (__ballot(hit)) return true;
  }
  return false;
}

template <int D, typename T>
__device__ __forceinline__ void pa_store4(T* y, bool vec, float a, float b, float c, float d) {
  if constexpr (sizeof(T) == 4) {
    if (vec) {
      *reinterpret_cast<float4*>(y) = make_float4(a, b, c, d);
      return;
    }
  } else {
    if (vec) {
      *reinterpret_cast<uint2*>(y) = make_uint2(cvt_bf16x2(a, b), cvt_bf16x2(c, d));
      return;
    }
  }
  store_f32(y, a);
  store_f32(y + 1, b);
  store_f32(y + 2, c);
  store_f32(y + 3, d);
}

// Which part of which sequence block blockIdx.x of a kv head takes where the parts are
// dealt out by length: a sequence gets one for every `per` steps of 32 positions, such
// that all of them are about `share`.  The sequence, or -1 for a block without one.
__device__ __forceinline__ int pa_share(const PaArgs& a, int lane, int waves, int* split, int* parts) {
  const int64_t cap = a.cols << a.ps_log2;
  uint32_t steps = 0, mine = 0;
  if (lane < a.batch) {
    const int64_t o0 = max(a.off[lane], (int64_t)0), o1 = min(a.off[lane + 1], a.rows), n = o1 - o0;
    const int64_t L = min(max(a.len[lane], (int64_t)0), cap);
    const int64_t from = a.window > 0 && L - n - a.window + 1 > 0 ? L - n - a.window + 1 : 0;
    if (n > 0) mine = 1, steps = (uint32_t)((L + kPaStep - 1) / kPaStep - from / kPaStep);
  }
  // halves of steps: 64 lanes' sum stays below 2^31
  const uint32_t all = __builtin_amdgcn_readlane(wave_incl_scan((int)((steps + 1) >> 1)), 63);
  uint32_t per = all / (uint32_t)a.share * 2 + 2;
  per = (per + waves - 1) / waves * waves;
  mine = mine ? min(max((steps + per - 1) / per, 1u), (uint32_t)a.nsplit) : 0u;
  const uint32_t upto = (uint32_t)wave_incl_scan((int)mine);
  const uint64_t past = __ballot(upto > blockIdx.x);
  if (!past) return -1;
  const int b = __builtin_ctzll(past);
  *parts = (int)__builtin_amdgcn_readlane(mine, b);
  *split = (int)(blockIdx.x - (__builtin_amdgcn_readlane(upto, b) - *parts));
  return b;
}

// Row tiles tile0, + tiles, ... of one (sequence, kv head): part `split` of `parts` of the
// positions that each sees.  pre: the first 64 of the sequence's pages, one a lane.
// NP: BF16 terms of the weights; each NP has the whole body to itself, from the queries to
// the join: one loop for either in a body that both share spills 276 registers.
template <int D, typename T, int NP>
__device__ __forceinline__ void pa_tiles(const PaArgs& a, float* s_o, const PaLane<D>& lo_, const int32_t* __restrict__ table,
                                         int pre, int h, int split, int parts, int tile0, int64_t o0, int n, int64_t L) {
  constexpr int NG = D / kKvGroup, HN = D / 64, NF = D / 16, NW = PaShape<D, T>::NW;
  constexpr int BIAS = sizeof(T) == 4 ? 0 : 16;
  constexpr int NQ = sizeof(T) == 4 ? 3 : 1;  // terms of q: all of its bits
  constexpr int OS = PaShape<D, T>::kOS;
  float* s_m = s_o + NW * 16 * OS;
  float* s_l = s_m + NW * 16;
  const int lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ps = 1 << a.ps_log2, nr = n * a.gs;  // rows x heads of a kv head: below 2^31
  for (int tile = tile0; tile < (nr + 15) >> 4; tile += a.tiles) {
    // the lane's row (column of the products)
    const int rr = tile * 16 + col;
    const bool inside = rr < nr;
    const int i = a.gs == 1 ? (inside ? rr : 0) : (int)((uint32_t)(inside ? rr : 0) / (uint32_t)a.gs);
    const int64_t t = o0 + i;
    const int head = h * a.gs + ((inside ? rr : 0) - i * a.gs);
    bool on = inside;
    if (a.heads) {
      uint32_t sel = 0;
      for (int c = 0; c < 16 && tile * 16 + c < nr; ++c) {
        const int cr = tile * 16 + c, ci = (int)((uint32_t)cr / (uint32_t)a.gs);
        if (pa_selected(a, o0 + ci, h * a.gs + (cr - ci * a.gs), lane)) sel |= 1u << c;
      }
      on = on && (sel >> col & 1);
    }
    int lo = 0, hi = 0;
    if (on) {
      const int64_t p = L - n + i;
      const int64_t e = a.causal ? (p + 1 < L ? p + 1 : L) : L;
      const int64_t s = a.window > 0 && p - a.window + 1 > 0 ? p - a.window + 1 : 0;
      if (e > s) lo = (int)s, hi = (int)e;
    }
    const bool some = hi > lo;
    // the tile's range, and the part of it that every row sees (the rows that see anything)
    const int tlo = (int)wave_min_u32(some ? (uint32_t)lo : 0x7fffffffu);
    const int thi = (int)wave_max_u32(some ? (uint32_t)hi : 0u);
    const int all_lo = (int)wave_max_u32(some ? (uint32_t)lo : 0u);
    const int all_hi = (int)wave_min_u32(some ? (uint32_t)hi : 0x7fffffffu);

    float m = -INFINITY, l = 0.0f;
    kh_f32x4 o[NF], om;
    float os[NG];  // sums of R of the lane's positions, where there is a bias
#pragma unroll
    for (int f = 0; f < NF; ++f) o[f] = kh_f32x4{0, 0, 0, 0};
    om = kh_f32x4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < NG; ++j) os[j] = 0.0f;

    const int first = tlo / kPaStep, steps = thi > tlo ? (thi + kPaStep - 1) / kPaStep - first : 0;
    const int per = (steps + parts - 1) / parts;
    const int sb = first + split * per, se = min(first + steps, sb + per);
    if (sb < se) {
      // The wave's steps sb + wave, + NW, ...: lane k holds the pages of the k-th of
      // the next 64, and a step's words are loaded while the one before it is worked on.
      const int mine = (se - sb - wave + NW - 1) / NW;
      const bool known = ((thi - 1) >> a.ps_log2) < 64;  // every page is among the first 64
      int pg0 = 0, pg1 = 0;
      const auto pages = [&](int k0) {
        const int k = k0 + lane, tok = (sb + wave + min(k, mine - 1) * NW) * kPaStep;
        // a half of the step that no row of the tile sees takes the other half's page:
        // the table need not name one there
        const int c0 = (tok + 16 <= tlo ? tok + 16 : tok) >> a.ps_log2;
        const int c1 = (tok + 16 >= thi ? tok : tok + 16) >> a.ps_log2;
        pg0 = known ? __shfl(pre, c0) : table[c0];
        pg1 = known ? __shfl(pre, c1) : table[c1];
        if (pg0 < 0 || pg0 >= a.pages) pg0 = -1;
        if (pg1 < 0 || pg1 >= a.pages) pg1 = -1;
        if ((pg0 | pg1) < 0) atomicOr(a.err, 2);
      };
      const auto load = [&](int k, PaStepData<D>& x) {
        const int tok = (sb + wave + k * NW) * kPaStep;
        const int p0 = max(__builtin_amdgcn_readlane(pg0, k & 63), 0), p1 = max(__builtin_amdgcn_readlane(pg1, k & 63), 0);
        pa_load<D, 0>(a.pool + ((int64_t)p0 * a.nkv + h) * a.block, tok & (ps - 1), lo_, x);
        pa_load<D, 1>(a.pool + ((int64_t)p1 * a.nkv + h) * a.block, (tok + 16) & (ps - 1), lo_, x);
      };
      constexpr bool ahead = PaShape<D, T>::kAhead > 0;
      PaStepData<D> x[ahead ? 2 : 1];
      Raw8<T> qr[NG];
      const T* q = static_cast<const T*>(a.q) + t * a.qs + head * a.qh;
#pragma unroll
      for (int j = 0; j < NG; ++j) qr[j].load(q + 32 * j + 8 * g, a.qvec);
      if (mine > 0) {
        pages(0);
        load(0, x[0]);
      }
      // q as the second operand: slots (0,4,1,5,2,6,3,7) of eight neighbouring
      // elements, the order in which codes2 takes the nibbles of a word
      uint4 qf[NG][NQ];
      uint4 qm[(NG + 3) / 4];
      {
        float qsum[NG];
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          float f[8];
          qr[j].get(f);
          const float e[8] = {f[0], f[4], f[1], f[5], f[2], f[6], f[3], f[7]};
          terms8<NQ>(e, qf[j]);
          qsum[j] = across_groups_sum(((f[0] + f[1]) + (f[2] + f[3])) + ((f[4] + f[5]) + (f[6] + f[7])));
        }
#pragma unroll
        for (int k = 0; k < (NG + 3) / 4; ++k) {
          float e[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float s = 4 * k + j < NG ? qsum[4 * k + j < NG ? 4 * k + j : 0] : 0.0f;
            e[2 * j] = s;
            e[2 * j + 1] = -(float)BIAS * s;
          }
          uint4 tm[3];
          terms8<3>(e, tm);
          const auto pick = [g](uint32_t x, uint32_t y, uint32_t z) { return g == 0 ? x : g == 1 ? y : g == 2 ? z : 0u; };
          qm[k] = make_uint4(pick(tm[0].x, tm[1].x, tm[2].x), pick(tm[0].y, tm[1].y, tm[2].y),
                             pick(tm[0].z, tm[1].z, tm[2].z), pick(tm[0].w, tm[1].w, tm[2].w));
        }
      }

      const auto step = [&](PaStepData<D>& x, int tok, bool ok0, bool ok1) {
        const bool whole = tok >= all_lo && tok + kPaStep <= all_hi && ok0 && ok1;
        // scores: positions 16 t + 4 g + r along registers, rows along lanes
        float s[2][4];
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
          kh_f32x4 base = {0, 0, 0, 0};
#pragma unroll
          for (int k = 0; k < (NG + 3) / 4; ++k) {
            uint4 av;
            if constexpr (NG == 2) av = make_uint4(x.kpa[tt][0], x.kpa[tt][1], 0, 0);
            else av = make_uint4(x.kpa[tt][4 * k], x.kpa[tt][4 * k + 1], x.kpa[tt][4 * k + 2], x.kpa[tt][4 * k + 3]);
            base = mfma16(av, qm[k], base);
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) s[tt][r] = base[r];
#pragma unroll
          for (int j = 0; j < NG; ++j) {
            const uint32_t w = x.kw[tt][j];
            const uint4 kf = make_uint4(codes2<BIAS>(w, 0), codes2<BIAS>(w, 1), codes2<BIAS>(w, 2), codes2<BIAS>(w, 3));
            kh_f32x4 c = {0, 0, 0, 0};
#pragma unroll
            for (int k = NQ - 1; k >= 0; --k) c = mfma16(kf, qf[j][k], c);
            const uint32_t ks = x.kpc[tt][j] & 0xffff0000u;
            s[tt][0] = fma_quad<0>(c[0], ks, s[tt][0]);
            s[tt][1] = fma_quad<1>(c[1], ks, s[tt][1]);
            s[tt][2] = fma_quad<2>(c[2], ks, s[tt][2]);
            s[tt][3] = fma_quad<3>(c[3], ks, s[tt][3]);
          }
        }
        bool see[2][4];
        float mx = -INFINITY;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (!whole) {
              const int j = tok + 16 * tt + 4 * g + r;
              see[tt][r] = j >= lo && j < hi && (tt ? ok1 : ok0);
              if (!see[tt][r]) s[tt][r] = -INFINITY;
            }
            mx = fmaxf(mx, s[tt][r]);
          }
        // a new maximum is looked for across the lanes only where one passes the old
        if (__ballot(mx > m)) {
          const float mn = fmaxf(m, across_groups_max(mx));
          const float alpha = mn == m ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * a.c1);
          l *= alpha;
          om *= alpha;
          if constexpr (BIAS != 0) {
#pragma unroll
            for (int j = 0; j < NG; ++j) os[j] *= alpha;
          }
#pragma unroll
          for (int f = 0; f < NF; ++f) o[f] *= alpha;
          m = mn;
        }
        const float mc = m == -INFINITY ? 0.0f : m * a.c1;
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(s[e >> 2][e & 3], a.c1, -mc));
        l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));

        uint4 pt[NP];
        terms8<NP>(p, pt);
        // rows m_g, then the scales alone
        const uint4 vm = make_uint4(__builtin_amdgcn_perm(x.vp[0][1], x.vp[0][0], 0x05040100u),
                                    __builtin_amdgcn_perm(x.vp[0][3], x.vp[0][2], 0x05040100u),
                                    __builtin_amdgcn_perm(x.vp[1][1], x.vp[1][0], 0x05040100u),
                                    __builtin_amdgcn_perm(x.vp[1][3], x.vp[1][2], 0x05040100u));
#pragma unroll
        for (int k = NP - 1; k >= 0; --k) om = mfma16(vm, pt[k], om);
#pragma unroll
        for (int e = 0; e < 8; ++e) x.vp[e >> 2][e & 3] &= 0xffff0000u;

        const auto group = [&](auto G) {
          constexpr int gi = decltype(G)::value;
          float ps8[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) ps8[e] = mul_row<gi>(p[e], x.vp[e >> 2][e & 3]);
          if (!whole) {
#pragma unroll
            for (int e = 0; e < 8; ++e) ps8[e] = see[e >> 2][e & 3] ? ps8[e] : 0.0f;
          }
          uint4 pg[NP];
          terms8<NP>(ps8, pg);
          if constexpr (BIAS != 0) {
#pragma unroll
            for (int k = NP - 1; k >= 0; --k)
              os[gi] = add2(pg[k].w, add2(pg[k].z, add2(pg[k].y, add2(pg[k].x, os[gi]))));
          }
#pragma unroll
          for (int ff = 0; ff < 2; ++ff) {
            const int f = 2 * gi + ff, hf = f >> 2, nb = f & 3;
            const uint4 vf = make_uint4(codes2<BIAS>(x.vw[0][hf], nb), codes2<BIAS>(x.vw[0][HN + hf], nb),
                                        codes2<BIAS>(x.vw[1][hf], nb), codes2<BIAS>(x.vw[1][HN + hf], nb));
#pragma unroll
            for (int k = NP - 1; k >= 0; --k) o[f] = mfma16(vf, pg[k], o[f]);
          }
        };
        group(std::integral_constant<int, 0>{});
        group(std::integral_constant<int, 1>{});
        if constexpr (NG >= 4) {
          group(std::integral_constant<int, 2>{});
          group(std::integral_constant<int, 3>{});
        }
        if constexpr (NG >= 8) {
          group(std::integral_constant<int, 4>{});
          group(std::integral_constant<int, 5>{});
          group(std::integral_constant<int, 6>{});
          group(std::integral_constant<int, 7>{});
        }
      };

      const auto work = [&](int k, int q0, int q1, PaStepData<D>& x) {
        step(x, (sb + wave + k * NW) * kPaStep, q0 >= 0, q1 >= 0);
      };
      if constexpr (ahead) {
        for (int k = 0; k < mine; k += 2) {
          int q0 = __builtin_amdgcn_readlane(pg0, k & 63), q1 = __builtin_amdgcn_readlane(pg1, k & 63);
          if (k + 1 < mine) load(k + 1, x[1]);  // 64 is even: of the same pages
          work(k, q0, q1, x[0]);
          if (k + 1 >= mine) break;
          q0 = __builtin_amdgcn_readlane(pg0, (k + 1) & 63);
          q1 = __builtin_amdgcn_readlane(pg1, (k + 1) & 63);
          if (k + 2 < mine) {
            if (((k + 2) & 63) == 0) pages(k + 2);
            load(k + 2, x[0]);
          }
          work(k + 1, q0, q1, x[1]);
        }
      } else {
        for (int k = 0; k < mine; ++k) {
          work(k, __builtin_amdgcn_readlane(pg0, k & 63), __builtin_amdgcn_readlane(pg1, k & 63), x[0]);
          if (k + 1 < mine) {
            if (((k + 1) & 63) == 0) pages(k + 1);
            load(k + 1, x[0]);
          }
        }
      }
    }

    // -B sum R + sum p m: row j of om lies with lane group j / 4
    l = across_groups_sum(l);
    {
#pragma unroll
      for (int gi = 0; gi < NG; ++gi) {
        float c = __shfl(om[gi & 3], (gi >> 2) * 16 + col);
        if constexpr (BIAS != 0) c -= (float)BIAS * across_groups_sum(os[gi]);
#pragma unroll
        for (int ff = 0; ff < 2; ++ff)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[2 * gi + ff][r] += c;
      }
    }
    // The waves' parts go to LDS as they are, and behind one barrier every thread
    // joins four elements of a row, in the order of the waves; maxima in powers of two.
    if (g == 0) s_m[wave * 16 + col] = some ? m * a.c1 : -INFINITY, s_l[wave * 16 + col] = some ? l : 0.0f;
#pragma unroll
    for (int f = 0; f < NF; ++f)
      *reinterpret_cast<kh_f32x4*>(s_o + (wave * 16 + col) * OS + 16 * f + 4 * g) = o[f];
    __syncthreads();
#pragma unroll
    for (int it = 0; it < (4 * D + 64 * NW - 1) / (64 * NW); ++it) {
      const int e = it * 64 * NW + (int)threadIdx.x, r = e / (D / 4), d = (e - r * (D / 4)) * 4;
      const int row16 = tile * 16 + r;
      if (r >= 16 || row16 >= nr) break;
      float M = -INFINITY, tot = 0.0f;
#pragma unroll
      for (int w = 0; w < NW; ++w) M = fmaxf(M, s_m[w * 16 + r]);
      const float Mu = M == -INFINITY ? 0.0f : M;
      kh_f32x4 v = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float fac = __builtin_amdgcn_exp2f(s_m[w * 16 + r] - Mu);
        tot = fmaf(s_l[w * 16 + r], fac, tot);
        const kh_f32x4 x = *reinterpret_cast<const kh_f32x4*>(s_o + (w * 16 + r) * OS + d);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = fmaf(x[k], fac, v[k]);
      }
      const int ri = a.gs == 1 ? row16 : (int)((uint32_t)row16 / (uint32_t)a.gs);
      const int64_t rt = o0 + ri;
      const int rh = h * a.gs + (row16 - ri * a.gs);
      const int64_t row = rt * a.nh + rh;
      // a row that sees nothing (here): no maximum and no sum; NaN scores leave the maximum behind
      const bool any = M != -INFINITY || tot != 0.0f;
      if (a.nsplit > 1) {
        const int64_t at = row * a.nsplit + split;
        if (d == 0) {
          a.part_ml[at] = make_float2(M, tot);
          for (int s = split + parts; s < a.nsplit; s += parts) a.part_ml[row * a.nsplit + s] = make_float2(-INFINITY, 0.0f);
        }
        if (any) *reinterpret_cast<float4*>(a.part_o + at * D + d) = make_float4(v[0], v[1], v[2], v[3]);
      } else {
        const float inv = any ? 1.0f / tot : 0.0f;
        pa_store4<D, T>(static_cast<T*>(a.out) + rt * a.os + rh * a.oh + d, a.ovec, any ? v[0] * inv : 0.0f,
                        any ? v[1] * inv : 0.0f, any ? v[2] * inv : 0.0f, any ? v[3] * inv : 0.0f);
        if (a.lse && d == 0) a.lse[row] = any ? kLn2 * (M + __builtin_amdgcn_logf(tot)) : -INFINITY;
      }
    }
    __syncthreads();
  }
}

// Block: one row tile of one (sequence, kv head), one of nsplit parts of the
// positions that the tile sees; its waves take every NW-th step of 32, the next step's
// codes under way.  As many blocks as the registers let the chip hold at once: twice as
// many parts were slower (64 sequences: 26.9 us instead of 25), each begins with the chain.
//
// BF16 terms of the weights P: f32 rows take three, all of their bits.  BF16 rows
// take one, as their output has, where the roundings of many positions cancel, and two
// where the sequence's length, or the window, lets them see 1024 or fewer: with one the
// error against 64 bits was 1.9 times that of rounding the output alone for 20 positions,
// 1.4 for 180 and 1.5 for lengths up to 650 mixed (two terms: 1.00).  Eight sequences of
// 1024 take 16.2 us with one, 18.3 with two, of 2048 25 and 30.
template <int D, typename T>
__global__ __launch_bounds__((64 * PaShape<D, T>::NW), (PaShape<D, T>::kPerSimd)) void paged_rows_kernel(PaArgs a) {
  constexpr int NW = PaShape<D, T>::NW;
  extern __shared__ __align__(16) float s_o[];  // [NW][16][OS], then the maxima and sums
  const int lane = threadIdx.x & 63;
  const int h = blockIdx.y;
  const int64_t cap = a.cols << a.ps_log2;
  const PaLane<D> lo_(lane, 1 << a.ps_log2);
  int split = blockIdx.x, parts = a.nsplit;
  int64_t z0 = blockIdx.z;
  if (a.share) {
    const int s = pa_share(a, lane, NW, &split, &parts);
    if (s < 0) return;
    z0 = s;
  }
  for (int64_t bt = z0; bt < a.batch * a.tiles; bt += a.share ? a.batch : gridDim.z) {
  const int64_t b = a.tiles == 1 ? bt : bt / a.tiles;
  const int tile0 = a.tiles == 1 ? 0 : (int)(bt - b * a.tiles);
  // the first of the chain's loads together: rows, length, the first 64 pages
  const int32_t* __restrict__ table = a.table + b * a.table_stride;
  const int pre = lane < a.cols ? table[lane] : -1;
  int64_t o0 = a.off[b], o1 = a.off[b + 1], L = a.len[b];
  o0 = o0 < 0 ? 0 : o0;
  o1 = o1 > a.rows ? a.rows : o1;
  if (o1 <= o0) continue;
  const int n = (int)(o1 - o0);
  if (L < 0 || L > cap) {
    if (threadIdx.x == 0) atomicOr(a.err, 1);
    L = L < 0 ? 0 : cap;
  }

  const auto run = [&](auto terms) {
    pa_tiles<D, T, decltype(terms)::value>(a, s_o, lo_, table, pre, h, split, parts, tile0, o0, n, L);
  };
  if constexpr (sizeof(T) == 4) run(std::integral_constant<int, 3>{});
  else if ((a.window > 0 && a.window < L ? a.window : L) <= kPaFine) run(std::integral_constant<int, 2>{});
  else run(std::integral_constant<int, 1>{});
  }
}

// ---------------------------------------------------------------- many rows
// Tiles of many rows (prompts and chunks, BF16): a step's 64 positions lie in LDS as
// BF16 numbers s c + m, in the order of the matrix core's first operand, and every wave
// runs its own rows (16 CT columns) over them, so the work of unpacking is shared by all
// rows of the block.  Rounding a key or a value to BF16 is off by at most 2^-8 of it, as
// in a BF16 cache, and queries and weights are BF16 themselves.  The next step's codes are
// loaded and unpacked while this one is worked on: two LDS buffers, one barrier a step.
//
// Where three row tiles or more see the same positions, a kernel unpacks them once into
// the workspace and the tiles copy them to LDS as they are: 4096 causal rows of 32 heads
// of 128 take 13 + 161 us so, 210 us where each tile unpacks them (at 137 GFLOP 0.85
// PFLOP/s; a call in a stream of them 149 us).  The copies go through registers: for a
// load straight to LDS the compiler waits before the next read of any LDS (178 us).
//
// A value's group that stands for NaN is unpacked as 0 and marked in a mask of its
// positions: rows that see one of them get their NaN from the mask.
//
// Bound by its own latency: two waves a SIMD (registers), each with its products (41% of
// the time), other vector instructions (39%) and waits (29% of its cycles) one after the other;
// at D = 256 by reading LDS, where a fragment feeds one product a wave (four chunks of 41 to
// 331 rows of 16 heads over 2, window 1024: 11 + 42 us and 8 of join).  Half of the
// waves a phase later (177 us), exponentials between the products of the step before
// (spills), blocks of four waves (187 us) and raised priority for products (no change)
// did not help.
constexpr int kOnlyAlu = 0x6;  // what a scheduling barrier lets pass: vector and scalar arithmetic
constexpr float kPtSlack = 6.0f;  // a maximum that is passed by less (in powers of two) is kept

// KT: BF16 terms that a key is held in.  One gives outputs as exact as their type
// holds; two (to 2^-16) and sums of weights that are not rounded are for callers who
// want the log-sum-exp, which is f32.
template <int D, int KT>
struct PtShape {
  static constexpr int NW = 8;
  static constexpr int NG = D / kKvGroup, HN = D / 64, NF = D / 16;
  static constexpr int CT = D == 256 ? 1 : 2;  // column tiles of 16 rows a wave holds
  static constexpr int RW = 16 * CT, RB = RW * NW;
  static constexpr int KEYS = D == 256 && KT == 2 ? 32 : 64;  // positions of a step: two steps' fit in LDS
  static constexpr int TK = KEYS / 16, TV = KEYS / 32;        // tiles of 16, halves of 32
  static constexpr int kKeyPart = KEYS * D * 2, kKeys = KT * kKeyPart, kValues = KEYS * D * 2;
  static constexpr int kStep = kKeys + kValues;               // bytes of a step
  static constexpr int kLds = 2 * kStep;
  static constexpr int KF = TK * NG / NW, VF = TV * NF / NW;  // fragments a wave unpacks
  static constexpr int VG = VF < 2 ? 1 : VF / 2, VH = VF <= 4 ? 1 : VF / 4;
};

typedef int kh_i32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 kh_f16x2 __attribute__((ext_vector_type(2)));

// Nibble n of each half of w as 16 + c, a pair of f16: six bits up it counts ones
// behind the bits of 16.
__device__ __forceinline__ kh_f16x2 codes_f16(uint32_t w, int n) {
  const uint32_t x = n == 0 ? w << 6 : n == 1 ? w << 2 : n == 2 ? w >> 2 : w >> 6;
  return __builtin_bit_cast(kh_f16x2, (x & 0x03c003c0u) | 0x4c004c00u);
}

template <int D, int KT>
struct PtCodes {
  using S = PtShape<D, KT>;
  uint32_t kw[S::KF], kp[S::KF];
  uint32_t vw[S::VH][4], vp[S::VG][8];
};

template <int N>
__device__ __forceinline__ void ld_n(const char* p, uint32_t* w) {
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

// What wave `wave` of NW does to a step's positions: KF fragments of keys of one of
// their tiles of 16, VF of values of one half of 32.  A fragment is what the 64 lanes of
// a wave hold of a matrix-core operand, 16 bytes each: of keys, tile by tile, NG; of
// values, half by half, D / 16.
template <int D, int KT>
struct PtUnpack {
  using S = PtShape<D, KT>;
  using C = PtCodes<D, KT>;
  using P = KvParts<D>;
  static constexpr int NG = S::NG, HN = S::HN, NF = S::NF, KF = S::KF, VF = S::VF, NW = S::NW;
  int ps, g, ktile, kj0, vtb, vf0;
  uint32_t koff, kpoff, voff, vpoff;  // the lane's words in a block
  __device__ __forceinline__ PtUnpack(int lane, int wave, int page_size) : ps(page_size), g(lane >> 4) {
    const int col = lane & 15;
    ktile = wave / (NW / S::TK);
    kj0 = (wave % (NW / S::TK)) * KF;
    vtb = wave / (NW / S::TV);
    vf0 = (wave % (NW / S::TV)) * VF;
    koff = P::kc() + col * (D / 2) + (g * NG + kj0) * 4;
    kpoff = P::kp(ps) + (col * NG + kj0) * 4;
    voff = P::vc(ps) + (g * 16 + col) * (HN * 8) + (vf0 >> 2) * 4;
    vpoff = P::vp(ps) + ((vf0 >> 1) * ps + 4 * g) * 4;
  }
  // tok: the first of the step's positions; blk(k): the block of their k-th tile of 16.
  template <typename B>
  __device__ __forceinline__ void load(int tok, B blk, C& x) const {
    const int in = (tok + ktile * 16) & (ps - 1);
    const char* kb = blk(ktile);
    ld_n<KF>(kb + in * (D / 2) + koff, x.kw);
    ld_n<KF>(kb + in * (NG * 4) + kpoff, x.kp);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int iv = (tok + vtb * 32 + q * 16) & (ps - 1);
      const char* vb = blk(2 * vtb + q);
      const char* vw = vb + iv * (D / 2) + voff;
#pragma unroll
      for (int hh = 0; hh < S::VH; ++hh) {
        x.vw[hh][2 * q] = *reinterpret_cast<const uint32_t*>(vw + hh * 4);
        x.vw[hh][2 * q + 1] = *reinterpret_cast<const uint32_t*>(vw + HN * 4 + hh * 4);
      }
#pragma unroll
      for (int gi = 0; gi < S::VG; ++gi) ld_n<4>(vb + iv * 4 + gi * ps * 4 + vpoff, &x.vp[gi][4 * q]);
    }
  }
  // put(term, fragment, the lane's 16 bytes)
  template <typename F>
  __device__ __forceinline__ void keys(const C& x, F put) const {
#pragma unroll
    for (int f = 0; f < KF; ++f) {
      const float s = __uint_as_float(x.kp[f] & 0xffff0000u);
      const float t = fmaf(-16.0f, s, __uint_as_float(x.kp[f] << 16));
      float v[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const kh_f16x2 c = codes_f16(x.kw[f], i);
        v[i] = fmaf((float)c.x, s, t);
        v[i + 4] = fmaf((float)c.y, s, t);
      }
      uint4 w[KT];
      terms8<KT>(v, w);
#pragma unroll
      for (int k = 0; k < KT; ++k) put(k, ktile * NG + kj0 + f, w[k]);
    }
  }
  // A group that stands for NaN counts as 0 from here on: mask(group, half, its
  // positions among the half's 32).
  template <typename F>
  __device__ __forceinline__ void nan(C& x, F mask) const {
#pragma unroll
    for (int gi = 0; gi < S::VG; ++gi) {
      uint32_t top = x.vp[gi][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) top = max(top, x.vp[gi][e]);
      uint32_t nan = 0;
      if (__ballot(top >= 0x7fc00000u)) {
        uint32_t from = 0x7fc00000u;
        asm volatile("" : "+s"(from));  // keeps this behind its branch
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t is = x.vp[gi][e] >= from ? 1u : 0u;
          nan |= is << ((e < 4 ? 0 : 16) + 4 * g + (e & 3));
          x.vp[gi][e] &= is - 1u;
        }
        nan = across_groups_or(nan);
      }
      if (VF > 1 || (vf0 & 1) == 0) mask((vf0 >> 1) + gi, vtb, nan);
    }
  }
  template <typename F>
  __device__ __forceinline__ void values(const C& x, F put) const {
#pragma unroll
    for (int gi = 0; gi < S::VG; ++gi) {
      float s[8], t[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s[e] = __uint_as_float(x.vp[gi][e] & 0xffff0000u);
        t[e] = fmaf(-16.0f, s[e], __uint_as_float(x.vp[gi][e] << 16));
      }
#pragma unroll
      for (int ff = 0; ff < (VF < 2 ? 1 : 2); ++ff) {
        const int fi = 2 * gi + ff;  // of the wave's
        float v[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const kh_f16x2 c = codes_f16(x.vw[VF <= 4 ? 0 : fi >> 2][e], (vf0 + fi) & 3);
          v[2 * e] = fmaf((float)c.x, s[2 * e], t[2 * e]);
          v[2 * e + 1] = fmaf((float)c.y, s[2 * e + 1], t[2 * e + 1]);
        }
        uint4 w[1];
        terms8<1>(v, w);
        put(vtb * NF + vf0 + fi, w[0]);
      }
    }
  }
};

// Where a step's positions of one (sequence, kv head) lie in the workspace once they
// are unpacked for all tiles, kStep bytes each: their keys' fragments, term by term,
// then their values'.  Behind all steps: the masks [NG][TV] of value groups that
// stand for NaN, one bit for each of 32 positions.
__device__ __forceinline__ int64_t pt_step(const PaArgs& a, int64_t b, int h, int st) {
  return (b * a.nkv + h) * a.un_steps + st;
}

// The positions that some row of the call sees, unpacked once for all of its row
// tiles: a block a step of a (sequence, kv head).
template <int D, int KT>
__global__ __launch_bounds__((64 * PtShape<D, KT>::NW)) void paged_unpack_kernel(PaArgs a) {
  using S = PtShape<D, KT>;
  using U = PtUnpack<D, KT>;
  constexpr int NG = S::NG, KEYS = S::KEYS;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int st = blockIdx.x, h = blockIdx.y;
  const U u(lane, wave, 1 << a.ps_log2);
  for (int64_t b = blockIdx.z; b < a.batch; b += gridDim.z) {
    const int32_t* __restrict__ table = a.table + b * a.table_stride;
    const int64_t n = min(a.off[b + 1], a.rows) - max(a.off[b], (int64_t)0), L = a.len[b];
    if (n <= 0 || L > (a.cols << a.ps_log2) || L > (int64_t)a.un_steps * KEYS) continue;
    const int64_t first = a.window > 0 && L - n - a.window + 1 > 0 ? L - n - a.window + 1 : 0;
    if ((int64_t)(st + 1) * KEYS <= first || (int64_t)st * KEYS >= L) continue;
    const auto blk = [&](int k) -> const char* {
      const int tok = min(max(st * KEYS + k * 16, (int)first), (int)L - 1);
      int pg = __builtin_amdgcn_readfirstlane(table[tok >> a.ps_log2]);
      if (pg < 0 || pg >= a.pages) pg = 0;  // the tiles' rows know that it is not there
      return a.pool + ((int64_t)pg * a.nkv + h) * a.block;
    };
    typename U::C x;
    u.load(st * KEYS, blk, x);
    const int64_t at = pt_step(a, b, h, st);
    char* to = a.un + at * S::kStep + lane * 16;
    u.keys(x, [&](int k, int f, const uint4& w) { *reinterpret_cast<uint4*>(to + k * S::kKeyPart + f * 1024) = w; });
    u.nan(x, [&](int gi, int half, uint32_t m) {
      if (lane == 0) a.un_nan[(at * NG + gi) * S::TV + half] = m;
    });
    u.values(x, [&](int f, const uint4& w) { *reinterpret_cast<uint4*>(to + S::kKeys + f * 1024) = w; });
  }
}

// UN: the positions lie unpacked in the workspace, and go from there to LDS as they
// are.
template <int D, int KT, bool UN>
__device__ __forceinline__ void pt_tiles(const PaArgs& a, char* s_buf, int* s_lo, int* s_hi,
                                         uint32_t (*s_nan)[D / kKvGroup][PtShape<D, KT>::TV], int64_t b, int h, int split, int tile0,
                                         int every, int64_t o0, int64_t o1, int64_t L) {
  using S = PtShape<D, KT>;
  constexpr int NG = S::NG, NF = S::NF, CT = S::CT, RW = S::RW, RB = S::RB, NW = S::NW;
  constexpr int KEYS = S::KEYS, TK = S::TK, TV = S::TV;
  constexpr int kRound = 64 / TK;  // steps whose tiles' pages the lanes hold
  const int lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = (int)(o1 - o0), nr = n * a.gs;
  const int32_t* __restrict__ table = a.table + b * a.table_stride;
  const PtUnpack<D, KT> un(lane, wave, 1 << a.ps_log2);

  for (int64_t tl = tile0; tl < (nr + RB - 1) / RB; tl += every) {
    const int tile = (int)tl;
    int lo[CT], hi[CT];
    uint32_t row[CT];  // t * nh + head, below 2^31
    bool inside[CT];
    uint32_t wlo = 0x7fffffffu, whi = 0, all_lo = 0, all_hi = 0x7fffffffu;
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const int r0 = tile * RB + wave * RW + c * 16, rr = r0 + col;
      inside[c] = rr < nr;
      const int i = (int)((uint32_t)(inside[c] ? rr : 0) / (uint32_t)a.gs);
      const int head = h * a.gs + ((inside[c] ? rr : 0) - i * a.gs);
      row[c] = (uint32_t)((o0 + i) * a.nh + head);
      bool on = inside[c];
      if (a.heads) {
        uint32_t sel = 0;
        for (int k = 0; k < 16 && r0 + k < nr; ++k) {
          const int ci = (int)((uint32_t)(r0 + k) / (uint32_t)a.gs);
          if (pa_selected(a, o0 + ci, h * a.gs + (r0 + k - ci * a.gs), lane)) sel |= 1u << k;
        }
        on = on && (sel >> col & 1);
      }
      lo[c] = hi[c] = 0;
      if (on) {
        const int64_t p = L - n + i;
        const int64_t e = a.causal ? (p + 1 < L ? p + 1 : L) : L;
        const int64_t s = a.window > 0 && p - a.window + 1 > 0 ? p - a.window + 1 : 0;
        if (e > s) lo[c] = (int)s, hi[c] = (int)e;
      }
      const bool some = hi[c] > lo[c];
      wlo = min(wlo, wave_min_u32(some ? (uint32_t)lo[c] : 0x7fffffffu));
      whi = max(whi, wave_max_u32(some ? (uint32_t)hi[c] : 0u));
      all_lo = max(all_lo, wave_max_u32(some ? (uint32_t)lo[c] : 0u));
      all_hi = min(all_hi, wave_min_u32(some ? (uint32_t)hi[c] : 0x7fffffffu));
    }
    __syncthreads();  // the last tile's readers of s_lo, s_hi and the buffers
    if (lane == 0) s_lo[wave] = (int)wlo, s_hi[wave] = (int)whi;
    __syncthreads();
    int tlo = 0x7fffffff, thi = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) tlo = min(tlo, s_lo[w]), thi = max(thi, s_hi[w]);
    tlo = __builtin_amdgcn_readfirstlane(tlo);
    thi = __builtin_amdgcn_readfirstlane(thi);

    float m[CT];
    kh_f32x4 l[CT], o[CT][NF];  // l: a product with ones, all four alike; KT > 1: [0] of the lane's own weights
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      m[c] = -INFINITY;
      l[c] = kh_f32x4{0, 0, 0, 0};
#pragma unroll
      for (int f = 0; f < NF; ++f) o[c][f] = kh_f32x4{0, 0, 0, 0};
    }
    const int first = tlo / KEYS, steps = thi > tlo ? (thi + KEYS - 1) / KEYS - first : 0;
    const int per = (steps + a.nsplit - 1) / a.nsplit;
    const int sb = first + split * per, se = min(first + steps, sb + per);
    if (sb < se) {
      uint4 qf[CT][NG];
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        const uint16_t* q = static_cast<const uint16_t*>(a.q) + (int64_t)(row[c] / (uint32_t)a.nh) * a.qs +
                            (int64_t)(row[c] % (uint32_t)a.nh) * a.qh + 8 * g;
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          if (a.qvec) {
            qf[c][j] = *reinterpret_cast<const uint4*>(q + 32 * j);
          } else {
            uint32_t e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = q[32 * j + i];
            qf[c][j] = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
          }
        }
      }
      // Lane i holds the offset of the block of the i-th of 64 tiles of 16 positions, the next
      // kRound steps'.  Bits of okn say which pages there are, those of okm the round before.
      uint32_t blk_lo = 0, blk_hi = 0;
      uint64_t okm = 0, okn = 0;
      const auto pages = [&](int st) {
        const int tok = min(max(st * KEYS + lane * 16, tlo & ~15), (thi - 1) & ~15);
        const int pg = table[max(tok, tlo) >> a.ps_log2];
        const bool there = pg >= 0 && pg < a.pages;
        if (!there) atomicOr(a.err, 2);
        const uint64_t p = ((int64_t)(there ? pg : 0) * a.nkv + h) * a.block;
        blk_lo = (uint32_t)p;
        blk_hi = (uint32_t)(p >> 32);
        okn = __ballot(there);
      };
      const auto blk = [&](int st, int k) {
        const int l = ((st - sb) & (kRound - 1)) * TK + k;
        const uint32_t x = __builtin_amdgcn_readlane(blk_lo, l), y = __builtin_amdgcn_readlane(blk_hi, l);
        return a.pool + ((uint64_t)y << 32 | x);
      };
      PtCodes<D, KT> x;
      const auto load = [&](int st) { un.load(st * KEYS, [&](int k) { return blk(st, k); }, x); };
      const auto unpack = [&](int st) {
        char* buf = s_buf + (st & 1) * S::kStep + lane * 16;
        un.keys(x, [&](int k, int f, const uint4& w) { *reinterpret_cast<uint4*>(buf + k * S::kKeyPart + f * 1024) = w; });
        un.nan(x, [&](int gi, int half, uint32_t m) {
          if (lane == 0) s_nan[st & 1][gi][half] = m;
        });
        un.values(x, [&](int f, const uint4& w) { *reinterpret_cast<uint4*>(buf + S::kKeys + f * 1024) = w; });
      };
      // UN: a wave's share of the step's bytes, and the masks
      constexpr int SHARE = S::kStep / 1024 / NW;
      kh_i32x4 raw[SHARE];
      uint32_t nan0 = 0, nan1 = 0, nan2 = 0;  // of the step that is worked on, and the next two
      const auto fetch = [&](int st) {
        const int64_t at = pt_step(a, b, h, st);
        const char* from = a.un + at * S::kStep + wave * SHARE * 1024 + lane * 16;
#pragma unroll
        for (int i = 0; i < SHARE; ++i) raw[i] = *reinterpret_cast<const kh_i32x4*>(from + i * 1024);
        nan2 = a.un_nan[at * (TV * NG) + (lane & (TV * NG - 1))];
      };
      const auto place = [&](int st) {
        char* to = s_buf + (st & 1) * S::kStep + wave * SHARE * 1024 + lane * 16;
#pragma unroll
        for (int i = 0; i < SHARE; ++i) *reinterpret_cast<kh_i32x4*>(to + i * 1024) = raw[i];
      };
      kh_f32x4 sc[CT][TK];
      uint4 pf[CT][TV];
      float mc[CT];
      // Fragments are read one group ahead of the products that take them.
      const auto scores = [&](int st) {
        const char* kbuf = s_buf + (st & 1) * S::kStep + lane * 16;
        constexpr int R = TK * KT;  // groups of NG fragments: a tile's last term first
        uint4 kf[2][NG];
        const auto at = [&](int r, int j) { return kbuf + (KT - 1 - r % KT) * S::kKeyPart + (r / KT * NG + j) * 1024; };
#pragma unroll
        for (int j = 0; j < NG; ++j) kf[0][j] = *reinterpret_cast<const uint4*>(at(0, j));
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (r + 1 < R) {
#pragma unroll
            for (int j = 0; j < NG; ++j) kf[(r + 1) & 1][j] = *reinterpret_cast<const uint4*>(at(r + 1, j));
          }
          __builtin_amdgcn_sched_barrier(kOnlyAlu);
          const int kt = r / KT;
          if (r % KT == 0) {
#pragma unroll
            for (int c = 0; c < CT; ++c) sc[c][kt] = kh_f32x4{0, 0, 0, 0};
          }
#pragma unroll
          for (int j = 0; j < NG; ++j)
#pragma unroll
            for (int c = 0; c < CT; ++c) sc[c][kt] = mfma16(kf[r & 1][j], qf[c][j], sc[c][kt]);
          __builtin_amdgcn_sched_barrier(kOnlyAlu);
        }
      };
      const auto whole = [&](int st, int ok) {
        return st * KEYS >= (int)all_lo && (st + 1) * KEYS <= (int)all_hi && ok == (1 << TK) - 1;
      };
      const auto hide = [&](int st, int ok) {
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          int from = lo[c] - st * KEYS - 4 * g;
          asm volatile("" : "+v"(from));  // keeps this behind its branch: 32 selects of every step otherwise
          const uint32_t span = (uint32_t)(hi[c] - lo[c]);
#pragma unroll
          for (int kt = 0; kt < TK; ++kt) {
            const uint32_t n = ok >> kt & 1 ? span : 0u;
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if ((uint32_t)(16 * kt + r - from) >= n) sc[c][kt][r] = -INFINITY;
          }
        }
      };
      float mx[CT];
      const auto top = [&]() {
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          mx[c] = sc[c][0][0];
#pragma unroll
          for (int e = 1; e < 4 * TK; ++e) mx[c] = fmaxf(mx[c], sc[c][e >> 2][e & 3]);
        }
      };
      const auto rescale = [&]() {
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          if (__ballot((mx[c] - m[c]) * a.c1 > kPtSlack)) {
            const float mn = fmaxf(m[c], across_groups_max(mx[c]));
            const float alpha = mn == m[c] ? 1.0f : __builtin_amdgcn_exp2f((m[c] - mn) * a.c1);
            l[c] *= alpha;
#pragma unroll
            for (int f = 0; f < NF; ++f) o[c][f] *= alpha;
            m[c] = mn;
            mc[c] = mn == -INFINITY ? 0.0f : mn * a.c1;
          }
        }
      };
      const auto weights = [&](int tb) {
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          float p[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(sc[c][2 * tb + (e >> 2)][e & 3], a.c1, -mc[c]));
          uint4 w[1];
          terms8<1>(p, w);
          pf[c][tb] = w[0];
          if (KT > 1) l[c][0] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
        }
      };
      constexpr int VQ = 4;  // value fragments of a group
      uint4 vf[2][VQ];
      const auto values = [&](int st, int k) {  // group k of step st's
        const char* vbuf = s_buf + (st & 1) * S::kStep + S::kKeys + lane * 16;
#pragma unroll
        for (int i = 0; i < VQ; ++i) vf[k & 1][i] = *reinterpret_cast<const uint4*>(vbuf + (k * VQ + i) * 1024);
      };
      const auto sum_values = [&](int st) {  // values(st, 0) is under way
        const uint4 ones = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
#pragma unroll
        for (int k = 0; k < TV * NF / VQ; ++k) {
          const int tb = k * VQ / NF;
          if (k + 1 < TV * NF / VQ) values(st, k + 1);
          __builtin_amdgcn_sched_barrier(kOnlyAlu);
          if (KT == 1 && k * VQ % NF == 0) {
#pragma unroll
            for (int c = 0; c < CT; ++c) l[c] = mfma16(ones, pf[c][tb], l[c]);
          }
#pragma unroll
          for (int i = 0; i < VQ; ++i)
#pragma unroll
            for (int c = 0; c < CT; ++c) {
              const int f = (k * VQ + i) % NF;
              o[c][f] = mfma16(vf[k & 1][i], pf[c][tb], o[c][f]);
            }
          __builtin_amdgcn_sched_barrier(kOnlyAlu);
        }
      };
      const auto spread_nan = [&](int st, int ok) {
        uint32_t any = 0;
        if constexpr (UN) {
          any = __ballot(nan0 != 0) != 0;
        } else {
#pragma unroll
          for (int gi = 0; gi < NG; ++gi)
#pragma unroll
            for (int tb = 0; tb < TV; ++tb) any |= s_nan[st & 1][gi][tb];
        }
        if (!__builtin_amdgcn_readfirstlane(any)) return;
        int tok = st * KEYS;
        asm volatile("" : "+s"(tok));  // keeps this behind its branch
#pragma unroll
        for (int gi = 0; gi < NG; ++gi) {
          uint64_t mask = 0;
#pragma unroll
          for (int tb = 0; tb < TV; ++tb) {
            if constexpr (UN) mask |= (uint64_t)(uint32_t)__builtin_amdgcn_readlane(nan0, TV * gi + tb) << (32 * tb);
            else mask |= (uint64_t)s_nan[st & 1][gi][tb] << (32 * tb);
          }
#pragma unroll
          for (int c = 0; c < CT; ++c) {
            const int from = max(lo[c] - tok, 0), to = min(hi[c] - tok, KEYS);  // of the step's positions
            uint64_t see = to > from ? (~0ull >> (64 - (to - from))) << from : 0;
            for (int k = 0; k < TK; ++k)
              if (!(ok >> k & 1)) see &= ~(0xffffull << (16 * k));
            if (mask & see) {
              const float x = __uint_as_float(0x7fc00000u);
              o[c][2 * gi] = o[c][2 * gi + 1] = kh_f32x4{x, x, x, x};
            }
          }
        }
      };

#pragma unroll
      for (int c = 0; c < CT; ++c) mc[c] = 0.0f;
      const bool busy = whi > wlo;  // some row of the wave sees something
      pages(sb);
      if constexpr (UN) {
        fetch(sb);
        place(sb);
        nan1 = nan2;
        if (sb + 1 < se) fetch(sb + 1);
      } else {
        load(sb);
        unpack(sb);
        if (sb + 1 < se) load(sb + 1);
      }
      for (int st = sb; st < se; ++st) {
        // pages() for the next round comes two steps before it
        const int i = (st - sb) & (kRound - 1);
        __syncthreads();
        nan0 = nan1;
        nan1 = nan2;
        if (st + 1 < se) {
          if constexpr (UN) place(st + 1);
          else unpack(st + 1);
        }
        if (i == kRound - 2) okm = okn;
        if (st + 2 < se) {
          if (i == kRound - 2) pages(st + 2);
          if constexpr (UN) fetch(st + 2);
          else load(st + 2);
        }
        const int ok = (int)((i >= kRound - 2 ? okm : okn) >> (TK * i)) & ((1 << TK) - 1);
        if (busy) {
          scores(st);
          values(st, 0);
          if (!whole(st, ok)) hide(st, ok);
          top();
          rescale();
#pragma unroll
          for (int tb = 0; tb < TV; ++tb) weights(tb);
          sum_values(st);
          spread_nan(st, ok);
        }
      }
    }

#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const float tot = KT > 1 ? across_groups_sum(l[c][0]) : l[c][0];
      const float M = m[c] * a.c1;
      const bool some = hi[c] > lo[c];
      if (!inside[c]) continue;
      const int64_t t = row[c] / (uint32_t)a.nh;
      const int head = (int)(row[c] - t * a.nh);
      if (a.nsplit > 1) {
        const int64_t at = (int64_t)row[c] * a.nsplit + split;
        if (g == 0) a.part_ml[at] = make_float2(some ? M : -INFINITY, some ? tot : 0.0f);
        if (some && sb < se) {
#pragma unroll
          for (int f = 0; f < NF; ++f)
            *reinterpret_cast<float4*>(a.part_o + at * D + 16 * f + 4 * g) =
                make_float4(o[c][f][0], o[c][f][1], o[c][f][2], o[c][f][3]);
        }
      } else {
        const bool any = some && (M != -INFINITY || tot != 0.0f);
        const float inv = any ? 1.0f / tot : 0.0f;
        uint16_t* y = static_cast<uint16_t*>(a.out) + t * a.os + head * a.oh + 4 * g;
#pragma unroll
        for (int f = 0; f < NF; ++f)
          pa_store4<D, uint16_t>(y + 16 * f, a.ovec, any ? o[c][f][0] * inv : 0.0f, any ? o[c][f][1] * inv : 0.0f,
                                 any ? o[c][f][2] * inv : 0.0f, any ? o[c][f][3] * inv : 0.0f);
        if (a.lse && g == 0) a.lse[row[c]] = any ? kLn2 * (M + __builtin_amdgcn_logf(tot)) : -INFINITY;
      }
    }
  }
}

// The u-th row tile of up to 64 sequences, the last tiles (which see the most) of all of
// them first: false where there are no more.  Grids of every sequence's most tiles left
// compute units empty behind blocks without rows (chunks of 331, 255, 41 and 286 rows:
// 232 blocks with rows among 336 began in two rounds, 71 us instead of 42).
__device__ __forceinline__ bool pt_tile(const PaArgs& a, int lane, int rb, uint32_t u, int* b, int* tile) {
  uint32_t n = 0;
  if (lane < a.batch) {
    const int64_t rows = min(a.off[lane + 1], a.rows) - max(a.off[lane], (int64_t)0);
    if (rows > 0) n = (uint32_t)((rows * a.gs + rb - 1) / rb);
  }
  const auto from = [&](uint32_t t) {  // tiles t and later of all sequences
    return (uint32_t)__builtin_amdgcn_readlane(wave_incl_scan((int)(n > t ? n - t : 0u)), 63);
  };
  if (u >= from(0)) return false;
  uint32_t lo = 0, hi = wave_max_u32(n);  // from(lo) > u >= from(hi)
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) >> 1;
    if (from(mid) > u) lo = mid;
    else hi = mid;
  }
  const uint64_t level = __ballot(n > lo);
  const uint32_t k = u - from(hi), rank = __builtin_popcountll(level & ((1ull << lane) - 1));
  *b = __builtin_ctzll(__ballot(n > lo && rank == k));
  *tile = (int)lo;
  return true;
}

// Blocks of the same kv head lie on the same XCD (h is what varies fastest, and
// there are eight XCDs).
template <int D, int KT, bool UN>
__global__ __launch_bounds__((64 * PtShape<D, KT>::NW), 2) void paged_tile_kernel(PaArgs a) {
  extern __shared__ __align__(16) char s_buf[];
  __shared__ int s_lo[PtShape<D, KT>::NW], s_hi[PtShape<D, KT>::NW];
  __shared__ uint32_t s_nan[2][D / kKvGroup][PtShape<D, KT>::TV];  // positions whose value group stands for NaN
  uint32_t id = blockIdx.x;
  const int h = (int)(id % (uint32_t)a.nkv);
  id /= (uint32_t)a.nkv;
  const int split = (int)(id % (uint32_t)a.nsplit);
  id /= (uint32_t)a.nsplit;
  int tile0, every = a.tiles;
  int64_t b;
  if (a.batch <= 64) {
    int s;
    if (!pt_tile(a, threadIdx.x & 63, PtShape<D, KT>::RB, id, &s, &tile0)) return;
    b = s;
    every = INT32_MAX;
  } else {
    b = id % (uint32_t)a.batch;
    tile0 = a.tiles - 1 - (int)(id / (uint32_t)a.batch);
  }
  int64_t o0 = a.off[b], o1 = a.off[b + 1], L = a.len[b];
  o0 = o0 < 0 ? 0 : o0;
  o1 = o1 > a.rows ? a.rows : o1;
  if (o1 <= o0) return;
  const int64_t cap = a.cols << a.ps_log2;
  if (L < 0 || L > cap) {
    if (threadIdx.x == 0) atomicOr(a.err, 1);
    L = L < 0 ? 0 : cap;
  }
  // a sequence that is longer than the caller said was not unpacked
  if (UN && a.len[b] <= (int64_t)a.un_steps * PtShape<D, KT>::KEYS && a.len[b] <= cap)
    pt_tiles<D, KT, true>(a, s_buf, s_lo, s_hi, s_nan, b, h, split, tile0, every, o0, o1, L);
  else
    pt_tiles<D, KT, false>(a, s_buf, s_lo, s_hi, s_nan, b, h, split, tile0, every, o0, o1, L);
}

// Joins the parts of each row from first_row on: W waves a (row, head), four elements a lane, so
// that 256 / D parts of a wave are in flight at once.  4 us, latency: the parts come
// from other XCDs' caches.
template <int D, typename T, int W>
__global__ __launch_bounds__(256) void paged_join_kernel(PaArgs a, int64_t first_row) {
  constexpr int C = D / 4, NS = 64 / C;
  __shared__ __align__(16) float s_acc[W > 1 ? W : 1][D];
  const int lane = threadIdx.x & 63, c = lane % C, sub = lane / C;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = first_row + (W > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave);
  const uint32_t t = (uint32_t)(row / a.nh);
  if (t >= a.rows) return;
  const int head = (int)(row - (int64_t)t * a.nh);
  const float2* __restrict__ ml = a.part_ml + row * a.nsplit;
  const float* __restrict__ po = a.part_o + row * a.nsplit * D + 4 * c;
  // every load that the first parts need at once, whether the row is one of a sequence or not
  const int s0 = (W > 1 ? wave : 0) * NS + sub;
  constexpr int ST = (W > 1 ? W : 1) * NS, U = 4;
  const int64_t first = a.off[0], last = a.off[a.batch];
  float4 v[U];
  float ms[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int s = min(s0 + u * ST, a.nsplit - 1);
    ms[u] = ml[s].x;
    v[u] = *reinterpret_cast<const float4*>(po + (int64_t)s * D);
  }
  float2 x[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) x[k] = lane + 64 * k < a.nsplit ? ml[lane + 64 * k] : make_float2(-INFINITY, 0.0f);
  if (t < first || t >= last) return;
  const float M = wave_max(fmaxf(x[0].x, x[1].x)), Mu = M == -INFINITY ? 0.0f : M;
  const float tot = wave_sum(__builtin_amdgcn_exp2f(x[0].x - Mu) * x[0].y + __builtin_amdgcn_exp2f(x[1].x - Mu) * x[1].y);
  float4 acc = make_float4(0, 0, 0, 0);
  const auto add = [&](float m, const float4& y, bool there) {
    // a part without a key was not written; where NaN scores left no maximum, tot is NaN
    const bool none = !there || m == -INFINITY;
    const float w = none ? 0.0f : __builtin_amdgcn_exp2f(m - Mu);
    acc.x = fmaf(w, none ? 0.0f : y.x, acc.x);
    acc.y = fmaf(w, none ? 0.0f : y.y, acc.y);
    acc.z = fmaf(w, none ? 0.0f : y.z, acc.z);
    acc.w = fmaf(w, none ? 0.0f : y.w, acc.w);
  };
#pragma unroll
  for (int u = 0; u < U; ++u) add(ms[u], v[u], s0 + u * ST < a.nsplit);
#pragma unroll 4
  for (int s = s0 + U * ST; s < a.nsplit; s += ST) add(ml[s].x, *reinterpret_cast<const float4*>(po + (int64_t)s * D), true);
#pragma unroll
  for (int m = C; m < 64; m <<= 1) {
    acc.x += __shfl_xor(acc.x, m);
    acc.y += __shfl_xor(acc.y, m);
    acc.z += __shfl_xor(acc.z, m);
    acc.w += __shfl_xor(acc.w, m);
  }
  if (W > 1) {
    if (sub == 0) *reinterpret_cast<float4*>(&s_acc[wave][4 * c]) = acc;
    __syncthreads();
    if (wave > 0) return;
    acc = *reinterpret_cast<const float4*>(&s_acc[0][4 * c]);
#pragma unroll
    for (int w = 1; w < W; ++w) {
      const float4 v = *reinterpret_cast<const float4*>(&s_acc[w][4 * c]);
      acc.x += v.x;
      acc.y += v.y;
      acc.z += v.z;
      acc.w += v.w;
    }
  }
  const bool any = M != -INFINITY || tot != 0.0f;
  if (sub == 0) {
    T* y = static_cast<T*>(a.out) + t * a.os + head * a.oh + 4 * c;
    pa_store4<D, T>(y, a.ovec, any ? acc.x / tot : 0.0f, any ? acc.y / tot : 0.0f, any ? acc.z / tot : 0.0f,
                    any ? acc.w / tot : 0.0f);
  }
  if (a.lse && lane == 0) a.lse[row] = any ? kLn2 * (M + __builtin_amdgcn_logf(tot)) : -INFINITY;
}

// How a call is cut: row tiles per (sequence, kv head) as the caller expects
// them, and parts along the positions when the tiles alone do not fill the chip.
//
// Tiles of many rows pay where the tiles of 16 rows do not fit on the chip at once, or
// have far to go: below, each goes over its positions from the start (12 against 30 us for
// 64 rows of 32 heads of 128 over 564 positions, 25 against 33 for 128 over 2176, 38
// against 50 for 256 over 2304, where the 16-row tiles need two rounds; 46 against 36 for
// 64 over 8064).  Sizes are in rows times positions.
constexpr int kPtMinRows = 64;
constexpr int64_t kPtMinWork = 3000;  // positions of a full chip of 16-row tiles
// Positions are unpacked ahead where three row tiles or more see them and there are
// enough: it takes 10 us (8 sequences of 256 rows: 42 against 37 us over 556 positions,
// 101 against 110 over 2304).
constexpr int kPtUnpackTiles = 3;
constexpr int64_t kPtUnpackWork = 1 << 18;           // row tiles times positions
constexpr int64_t kPtUnpackMost = (int64_t)1 << 30;  // bytes of them
constexpr int64_t kPtMostBlocks = (int64_t)1 << 20;  // tiles of more than 64 sequences, as guessed
template <typename T>
static int pa_fill_t(int d) {
  return d == 64 ? PaShape<64, T>::kFill : d == 128 ? PaShape<128, T>::kFill : PaShape<256, T>::kFill;
}
static int pa_waves(int d, int dtype) {
  return d == 64 ? (dtype == KH_DT_F32 ? PaShape<64, float>::NW : PaShape<64, uint16_t>::NW)
       : d == 128 ? (dtype == KH_DT_F32 ? PaShape<128, float>::NW : PaShape<128, uint16_t>::NW)
                  : PaShape<256, uint16_t>::NW;
}
static int pa_fill(int d, int dtype) { return dtype == KH_DT_F32 ? pa_fill_t<float>(d) : pa_fill_t<uint16_t>(d); }
struct PtSize {
  int keys, step, masks, rows, fill;  // positions of a step, their bytes and their masks', rows of a block, blocks that the chip holds
};
template <int D, int KT>
static PtSize pt_size_dk() {
  using S = PtShape<D, KT>;
  return {S::KEYS, S::kStep, S::NG * S::TV * 4, S::RB, 256 * 8 / S::NW};
}
template <int D>
static PtSize pt_size_d(bool lse) {
  return lse ? pt_size_dk<D, 2>() : pt_size_dk<D, 1>();
}
static PtSize pt_size(int d, bool lse) {
  return d == 64 ? pt_size_d<64>(lse) : d == 128 ? pt_size_d<128>(lse) : pt_size_d<256>(lse);
}
struct PaPlan {
  bool many;  // paged_tile_kernel
  int64_t tiles, base;
  int nsplit, share;
  int64_t un_steps;  // steps of each sequence that are unpacked ahead, or 0
};
static PaPlan pa_plan(const kh_paged_kv* c, int dtype, int nh, int64_t rows, int64_t batch, int64_t max_rows,
                      int64_t max_len, bool lse) {
  PaPlan p;
  const int64_t gs = nh / c->nkv;
  if (max_rows > rows) max_rows = rows;
  if (max_len > INT32_MAX) max_len = INT32_MAX;  // more than a table holds
  const int64_t tiles16 = std::min<int64_t>((max_rows * gs + 15) / 16, 65536) * batch * c->nkv, held = pa_fill(c->d, dtype);
  p.many = dtype == KH_DT_BF16 && max_rows * gs >= kPtMinRows &&
           (tiles16 > held || (max_len > 0 && tiles16 > kPtMinWork * held / max_len));
  const PtSize z = pt_size(c->d, lse);
  // a block of its own for each tile that the guess allows, as far as a grid goes: past
  // that a block takes every tiles-th
  const int64_t most_tiles = p.many && batch > 64 ? kPtMostBlocks / (batch * c->nkv) : 65535 / batch;
  if (p.many && most_tiles < 1) p.many = false;
  const int64_t rb = p.many ? z.rows : 16;
  p.tiles = std::max<int64_t>(std::min<int64_t>((max_rows * gs + rb - 1) / rb, most_tiles), 1);
  p.base = batch * c->nkv * p.tiles;
  const int64_t fill = p.many ? z.fill : pa_fill(c->d, dtype);
  if (p.many && batch <= 64) p.base = c->nkv * ((rows * gs + batch * (rb - 1)) / rb);  // as pt_tile counts them
  int64_t want = fill / p.base;  // one round of blocks: a second would begin with its own latency
  // parts of fewer than four steps a wave do not pay for the join
  const int64_t step = p.many ? 512 : 32 * pa_waves(c->d, dtype);
  const int64_t most = max_len < 4 * step ? 1 : (max_len + step - 1) / step;
  if (want > most) want = most;
  if (want > kPaMaxSplit) want = kPaMaxSplit;
  p.nsplit = want < 1 ? 1 : (int)want;
  p.share = 0;
  // Single rows of several sequences: parts by length, which every block works out from
  // the lengths for itself (64 sequences of 1 to 4096 positions: 25 us with three parts
  // for each, 21 with eight at most; where all have 4096, 33 and 34).
  if (!p.many && p.nsplit > 1 && p.tiles == 1 && batch > 1 && batch <= 64) {
    p.share = (int)(fill / c->nkv - batch / 2);
    p.nsplit = (int)std::min<int64_t>(std::min(2 * p.nsplit + 2, kPaMaxSplit), most);
  }
  p.un_steps = 0;
  if (p.many && p.tiles >= kPtUnpackTiles && max_len >= kPtUnpackWork / p.base) {
    const int64_t steps = (max_len + z.keys - 1) / z.keys;
    if (steps <= kPtUnpackMost / z.step / (batch * c->nkv)) p.un_steps = steps;
  }
  return p;
}
// The workspace: parts of rows, their maxima and sums, unpacked positions, their masks.
struct PaSpace {
  int64_t ml, un, nan, bytes;
};
static PaSpace pa_space(const PaPlan& p, int64_t rows, int64_t batch, int nkv, int nh, int d, bool lse) {
  const int64_t parts = p.nsplit > 1 ? rows * nh * p.nsplit : 0, steps = batch * nkv * p.un_steps;
  PaSpace s;
  s.ml = parts * 4 * d;
  s.un = (s.ml + parts * 8 + 15) / 16 * 16;
  s.nan = s.un + steps * pt_size(d, lse).step;
  s.bytes = s.nan + steps * pt_size(d, lse).masks;
  return s;
}

template <int D, int KT>
static int pt_launch(const PaArgs& a, int64_t blocks, hipStream_t st) {
  constexpr int lds = PtShape<D, KT>::kLds;
  const dim3 g((unsigned)blocks), blk(64 * PtShape<D, KT>::NW);
  if (a.un_steps) {
    hipLaunchKernelGGL((paged_unpack_kernel<D, KT>),
                       dim3((unsigned)a.un_steps, (unsigned)a.nkv, (unsigned)(a.batch < 65535 ? a.batch : 65535)), blk,
                       0, st, a);
    hipLaunchKernelGGL((paged_tile_kernel<D, KT, true>), g, blk, lds, st, a);
  } else {
    hipLaunchKernelGGL((paged_tile_kernel<D, KT, false>), g, blk, lds, st, a);
  }
  KH_LAUNCHED();
  return KH_OK;
}

template <int D, typename T>
static int pa_launch(const PaArgs& a, bool many, int64_t blocks, hipStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (many) {
      const int rc = a.lse ? pt_launch<D, 2>(a, blocks, st) : pt_launch<D, 1>(a, blocks, st);
      if (rc != KH_OK) return rc;
    }
  }
  if (!many) {
    const dim3 g((unsigned)(a.share ? a.share + a.batch : a.nsplit), (unsigned)a.nkv,
                 (unsigned)(a.share ? 1 : a.batch * a.tiles < 65535 ? a.batch * a.tiles : 65535));
    const dim3 blk((64 * PaShape<D, T>::NW));
    constexpr int lds = PaShape<D, T>::kLds;
    hipLaunchKernelGGL((paged_rows_kernel<D, T>), g, blk, lds, st, a);
  }
  if (a.nsplit > 1) {
    const int64_t all = a.rows * a.nh, each = a.nsplit > 16 ? 1 : 4, most = kGridThreads / 256 * each;
    for (int64_t row = 0; row < all; row += most) {
      const dim3 g((unsigned)((std::min(all - row, most) + each - 1) / each));
      if (each == 1) hipLaunchKernelGGL((paged_join_kernel<D, T, 4>), g, dim3(256), 0, st, a, row);
      else hipLaunchKernelGGL((paged_join_kernel<D, T, 1>), g, dim3(256), 0, st, a, row);
    }
  }
  KH_LAUNCHED();
  return KH_OK;
}
template <typename T>
static int pa_launch_d(int d, const PaArgs& a, bool many, int64_t blocks, hipStream_t st) {
  if (d == 64) return pa_launch<64, T>(a, many, blocks, st);
  if (d == 128) return pa_launch<128, T>(a, many, blocks, st);
  return pa_launch<256, T>(a, many, blocks, st);
}

// Dynamic LDS of more than 64 KB has to be asked for, a kernel and device: when a cache
// is made, so that no call does it inside a capture.
template <typename K>
static int allow_lds(K* kernel, int bytes) {
  KH_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
  return KH_OK;
}
template <int D>
static int allow_lds_d() {
  int rc = allow_lds(&paged_rows_kernel<D, float>, PaShape<D, float>::kLds);
  if (rc == KH_OK) rc = allow_lds(&paged_rows_kernel<D, uint16_t>, PaShape<D, uint16_t>::kLds);
  if (rc == KH_OK) rc = allow_lds(&paged_tile_kernel<D, 1, false>, PtShape<D, 1>::kLds);
  if (rc == KH_OK) rc = allow_lds(&paged_tile_kernel<D, 1, true>, PtShape<D, 1>::kLds);
  if (rc == KH_OK) rc = allow_lds(&paged_tile_kernel<D, 2, false>, PtShape<D, 2>::kLds);
  if (rc == KH_OK) rc = allow_lds(&paged_tile_kernel<D, 2, true>, PtShape<D, 2>::kLds);
  return rc;
}
int paged_attn_prepare(int d) { return d == 64 ? allow_lds_d<64>() : d == 128 ? allow_lds_d<128>() : allow_lds_d<256>(); }

static int pa_shape(const kh_paged_kv* c, int dtype, int64_t rows, int64_t batch, int num_heads, int64_t max_rows,
                    int64_t max_len) {
  KH_CHECK_ARG(c != nullptr, "null handle");
  KH_CHECK_ARG(dtype == KH_DT_F32 || dtype == KH_DT_BF16, "dtype %d: f32 and BF16 are supported", dtype);
  KH_CHECK_ARG(rows >= 0 && rows < (int64_t)1 << 31 && batch >= 0 && batch < (int64_t)1 << 31,
               "rows %lld, batch %lld not in [0,2^31)", (long long)rows, (long long)batch);
  KH_CHECK_ARG(num_heads >= c->nkv && num_heads % c->nkv == 0 && num_heads <= 65536,
               "num_heads %d is no multiple of the cache's %d", num_heads, c->nkv);
  KH_CHECK_ARG(rows * (num_heads / c->nkv) < (int64_t)1 << 31, "%lld rows of %d heads: too many for one call",
               (long long)rows, num_heads);
  KH_CHECK_ARG(max_rows >= 0 && max_len >= 0, "max_rows %lld, max_len %lld", (long long)max_rows, (long long)max_len);
  return KH_OK;
}

}  // namespace kh

using namespace kh;

extern "C" int kh_paged_kv_attention_workspace(const kh_paged_kv* c, int dtype, int64_t rows, int64_t batch,
                                               int num_heads, int64_t max_rows, int64_t max_len, int with_lse,
                                               int64_t* bytes) {
  KH_CHECK_ARG(bytes != nullptr, "null output");
  const int rc = pa_shape(c, dtype, rows, batch, num_heads, max_rows, max_len);
  if (rc != KH_OK) return rc;
  *bytes = 0;
  if (rows && batch)
    *bytes = pa_space(pa_plan(c, dtype, num_heads, rows, batch, max_rows, max_len, with_lse != 0), rows, batch, c->nkv,
                      num_heads, c->d, with_lse != 0).bytes;
  return KH_OK;
}

extern "C" int kh_paged_kv_attention(const kh_paged_kv* c, int dtype, const void* q_dev, int64_t q_row_stride,
                                     int64_t q_head_stride, int num_heads, int64_t rows, const int64_t* off_dev,
                                     int64_t batch, const int64_t* len_dev, const int32_t* table_dev,
                                     int64_t table_cols, int64_t table_stride, int64_t max_rows, int64_t max_len,
                                     float scale, int causal, int64_t window, const int32_t* heads_dev, int n_heads,
                                     void* out_dev, int64_t out_row_stride, int64_t out_head_stride, float* lse_dev,
                                     void* ws_dev, int64_t ws_bytes, void* stream) {
  int rc = pa_shape(c, dtype, rows, batch, num_heads, max_rows, max_len);
  if (rc != KH_OK) return rc;
  KH_CHECK_ARG(table_cols >= 1 && table_stride >= table_cols, "page table of %lld columns, %lld apart",
               (long long)table_cols, (long long)table_stride);
  KH_CHECK_ARG(table_cols <= (INT32_MAX - 64) >> c->ps_log2, "a page table of %lld columns holds 2^31 positions",
               (long long)table_cols);
  KH_CHECK_ARG(std::isfinite(scale * kLog2e) && scale > 0, "scale must be positive and finite");
  KH_CHECK_ARG(window >= 0 && (window == 0 || causal), "a window (%lld) needs causal attention", (long long)window);
  KH_CHECK_ARG(q_row_stride >= 0 && q_head_stride >= 0, "negative stride");
  KH_CHECK_ARG(n_heads >= 0 && n_heads <= 4 * num_heads, "n_heads %d not in [0,%d]", n_heads, 4 * num_heads);
  KH_CHECK_ARG(strides_disjoint(rows, out_row_stride, num_heads, out_head_stride, c->d),
               "output strides (%lld, %lld) let heads overlap", (long long)out_row_stride,
               (long long)out_head_stride);
  if (rows == 0 || batch == 0) return KH_OK;
  KH_CHECK_ARG(q_dev && off_dev && len_dev && table_dev && out_dev, "null argument");
  KH_CHECK_ARG(heads_dev || n_heads == 0, "null head list");
  const PaPlan p = pa_plan(c, dtype, num_heads, rows, batch, max_rows, max_len, lse_dev != nullptr);
  const PaSpace sp = pa_space(p, rows, batch, c->nkv, num_heads, c->d, lse_dev != nullptr);
  const int64_t need = sp.bytes;
  if (need > 0 && (!ws_dev || ws_bytes < need)) {
    set_error("the workspace holds %lld bytes, %lld are needed", (long long)(ws_dev ? ws_bytes : 0),
              (long long)need);
    return KH_ERR_CAPACITY;
  }
  KH_CHECK_ARG((reinterpret_cast<uintptr_t>(ws_dev) & 15) == 0, "the workspace must be 16-byte aligned");
  const int64_t blocks = p.base * p.nsplit;  // of many rows' tiles
  KH_CHECK_ARG((!p.many || blocks <= kGridThreads / 512) && rows * num_heads < (int64_t)1 << 31,
               "too many rows for one call");
  KH_ON_DEVICE(c->device, "the cache");
  PaArgs a;
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
  a.heads = heads_dev;
  a.nsel = n_heads;
  a.nh = num_heads;
  a.gs = num_heads / c->nkv;
  a.c1 = scale * kLog2e;
  a.causal = causal ? 1 : 0;
  a.window = window <= INT32_MAX ? window : 0;  // wider than a table hides nothing; differences from it stay in 64 bits
  a.out = out_dev;
  a.os = out_row_stride;
  a.oh = out_head_stride;
  a.lse = lse_dev;
  a.nsplit = p.nsplit;
  a.share = p.share;
  a.tiles = (int)p.tiles;
  char* ws = static_cast<char*>(ws_dev);
  a.part_o = reinterpret_cast<float*>(ws);
  a.part_ml = reinterpret_cast<float2*>(ws + sp.ml);
  a.un = ws + sp.un;
  a.un_nan = reinterpret_cast<uint32_t*>(ws + sp.nan);
  a.un_steps = (int)p.un_steps;
  a.qvec = aligned16(q_dev, dtype, q_row_stride, q_head_stride) ? 1 : 0;
  a.ovec = aligned16(out_dev, dtype, out_row_stride, out_head_stride) ? 1 : 0;
  return dtype == KH_DT_F32 ? pa_launch_d<float>(c->d, a, p.many, blocks, as_stream(stream))
                            : pa_launch_d<uint16_t>(c->d, a, p.many, blocks, as_stream(stream));
}
