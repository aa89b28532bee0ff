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
__device__ __forceinline__ uint32_t kv_code(float x, float m, float s) {
  if (!(s > 0.0f)) return 0;
  const float q = rintf(__fdiv_rn(__fsub_rn(x, m), s));
  return (uint32_t)fminf(fmaxf(q, 0.0f), 15.0f);
}
// The codes of eight values, four bits each.  The quotient without a division
// (Markstein): with y the correctly rounded reciprocal of s and q = d y within an
// ulp of d / s, q + (d - q s) y rounds to the correctly rounded d / s.  One step
// from the hardware's reciprocal gives y (for significands that are not all ones; s
// has eight bits), where nothing underflows: scales below 2^-90 are divided.
__device__ __forceinline__ uint32_t kv_codes8(const float (&f)[8], uint32_t pair) {
  const float s = __uint_as_float(pair & 0xffff0000u), m = __uint_as_float(pair << 16);
  uint32_t w = 0;
  if (s > 0.0f && s < 0x1p-90f) {
#pragma unroll
    for (int i = 7; i >= 0; --i) w = w << 4 | kv_code(f[i], m, s);
    return w;
  }
  const float y0 = __builtin_amdgcn_rcpf(s), y = fmaf(fmaf(-s, y0, 1.0f), y0, y0);
#pragma unroll
  for (int i = 7; i >= 0; --i) {
    const float d = f[i] - m, q = d * y;
    w = w << 4 | (uint32_t)(int)rintf(fmaf(fmaf(-q, s, d), y, q));
  }
  return s > 0.0f ? w : 0;
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

struct AppendArgs {
  KvRows r;
  const void *k, *v;
  int64_t ks, kh, vs, vh;
  const int64_t* pos;  // rotary positions of the rows, or nullptr: their places in the cache
  const float2* table;
  int64_t max_pos;
  int rot, half_layout, mode;
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

// The quads (four positions that share bytes) that the rows of sequences c0 ..
// c0 + nb - 1 touch: s_q[i] of them lie before sequence c0 + i.  The whole block
// takes part; returns their number.
constexpr int kSeqChunk = 1024;
__device__ __forceinline__ int quads_of(int64_t n, int64_t start) {
  if (n <= 0) return 0;
  // a start past 2^40 is out of every table: one quad reports it
  if (start <= -((int64_t)1 << 40) || start >= (int64_t)1 << 40) return 1;
  return (int)(((start + n - 1) >> 2) - (start >> 2) + 1);
}
__device__ __forceinline__ int stage_quads(const KvRows& a, int64_t c0, int nb, int* s_q, int* wsum, int* s_tot) {
  constexpr int E = kSeqChunk / kKvThreads;
  int n[E], sum = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = threadIdx.x * E + e;
    n[e] = 0;
    if (i < nb) {
      n[e] = quads_of(min(a.off[c0 + i + 1], a.rows) - max(a.off[c0 + i], (int64_t)0), a.start[c0 + i]);
    }
    sum += n[e];
  }
  int at = block_excl_scan(sum, wsum, s_tot);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    s_q[threadIdx.x * E + e] = at;
    at += n[e];
  }
  __syncthreads();
  return *s_tot;
}

// How the rows' keys are rotated: not at all, pieces of eight elements by their
// pairs, or element by element (any rot).
constexpr int kRotNone = 0, kRotHalf = 1, kRotInterleaved = 2, kRotAny = 3;

// Up to 64 sequences: lane i holds sequence i's quads and those before it.
struct WaveSeqs {
  int before = 0, n = 0, o0 = 0, o1 = 0;
  int64_t start = 0;
};
__device__ __forceinline__ int64_t readlane64(int64_t v, int l) {
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)v, l), hi = __builtin_amdgcn_readlane((uint32_t)(v >> 32), l);
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// Gives the waves of the grid their quads, one unit (hpu heads) at a time:
// f(p0, t0, o0, o1, pg, h0, nh), with the quad's first position and its row, the
// sequence's rows, the page, and the unit's heads.  Rows t0 .. t0 + 3 that lie in
// [o0, o1) are the quad's.  Places that are not there are recorded and skipped.
template <typename F>
__device__ __forceinline__ void walk_quads(const KvRows& r, int units, int hpu, int* s_q, int* s_wsum, int* s_tot, F f) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool few = r.batch <= 64;
  for (int64_t c0 = 0; c0 < r.batch; c0 += kSeqChunk) {
    const int nb = (int)min((int64_t)kSeqChunk, r.batch - c0);
    WaveSeqs ws;
    int quads;
    if (few) {
      if (lane < nb) {
        ws.o0 = (int)min(max(r.off[lane], (int64_t)0), r.rows);
        ws.o1 = (int)min(max(r.off[lane + 1], (int64_t)0), r.rows);
        ws.start = r.start[lane];
        ws.n = quads_of(ws.o1 - ws.o0, ws.start);
      }
      const int incl = wave_incl_scan(ws.n);
      ws.before = incl - ws.n;
      quads = __builtin_amdgcn_readlane(incl, 63);
    } else {
      if (c0) __syncthreads();
      quads = stage_quads(r, c0, nb, s_q, s_wsum, s_tot);
    }
    const uint32_t end = (uint32_t)quads * (uint32_t)units;  // below 2^31 (checked on the host)
    for (uint32_t u = blockIdx.x * (kKvThreads / 64) + wave; u < end; u += gridDim.x * (kKvThreads / 64)) {
      const int qi = (int)(u / (uint32_t)units), h0 = (int)(u - (uint32_t)qi * (uint32_t)units) * hpu;
      int lo = 0;  // the sequence: the last one with no more than qi quads before it, and some of its own
      int o0, o1, first;
      int64_t start;
      if (few) {
        lo = 63 - __builtin_clzll(__ballot(ws.n > 0 && ws.before <= qi));
        o0 = __builtin_amdgcn_readlane(ws.o0, lo);
        o1 = __builtin_amdgcn_readlane(ws.o1, lo);
        start = readlane64(ws.start, lo);
        first = __builtin_amdgcn_readlane(ws.before, lo);
      } else {
        int hi = nb;
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (s_q[mid] <= qi) lo = mid;
          else hi = mid;
        }
        lo = __builtin_amdgcn_readfirstlane(lo);
        o0 = (int)max(r.off[c0 + lo], (int64_t)0);
        o1 = (int)min(r.off[c0 + lo + 1], r.rows);
        start = r.start[c0 + lo];
        first = __builtin_amdgcn_readfirstlane(s_q[lo]);
      }
      const int64_t p0 = ((start >> 2) + (qi - first)) * 4;
      const int64_t colm = p0 >> r.ps_log2;
      if (p0 < 0 || colm >= r.cols) {
        if (lane == 0) atomicOr(r.err, 1);
        continue;
      }
      const int pg = __builtin_amdgcn_readfirstlane(r.table[(c0 + lo) * r.table_stride + colm]);
      if (pg < 0 || pg >= r.pages) {
        if (lane == 0) atomicOr(r.err, 2);
        continue;
      }
      f(p0, (int)(o0 + (p0 - start)), o0, o1, pg, h0, min(hpu, r.nkv - h0));
    }
  }
}

// The lanes of a wave over a quad: D / 8 lanes a position, eight neighbouring
// elements each.
template <int D>
struct QuadLanes {
  static constexpr int L = D / 8;
  static constexpr int TP = 64 / L < 4 ? 64 / L : 4, PASS = 4 / TP;  // positions at a time
  static constexpr int HW = D == 64 ? 2 : 1;                         // heads at a time
};

// A wave takes a quad and the heads of one unit: D / 8 lanes a position with eight
// neighbouring values each, so four lanes share a group.  blockIdx.y: keys, values.
// Keys leave as they are, a word a lane.  The u16 of a value's layout gathers the
// nibbles of four lanes (c, c ^ 2, c ^ 4, c ^ 6), and a quad's four positions
// share 16-byte pieces: they are put together in LDS and stored whole where all
// four are appended, and as u16 where they are not.
//
// 14460 BF16 rows of 8 heads of 128 (59 MB in, 18.5 MB out, interleaved rotation): 32.6 us
// behind a gather, 2.4 TB/s, 28.9 where the input lies in the caches; f32 (118 MB in) 37.6.
// Latency: a wave loads, codes and stores one head after the other, so that 28 vector
// instructions a value (ranges, quotients, codes, places), 55% of the issue slots, and waits,
// 53% of its cycles, do not overlap enough (a position a lane took 77 us;
// quads with correctly rounded quotients by a division 38, by a corrected reciprocal 33).
// One row: 4 us, the chain of offsets, page id and table.
template <typename T, int D, int MODE, bool VAL>
__device__ __forceinline__ void append_part(const AppendArgs& a, int units, int hpu, int* s_q, int* s_wsum, int* s_tot,
                                            uint16_t* s_v) {
  using P = KvParts<D>;
  constexpr int NG = D / kKvGroup, HN = D / 64, L = QuadLanes<D>::L;
  constexpr int TP = QuadLanes<D>::TP, PASS = QuadLanes<D>::PASS, HW = QuadLanes<D>::HW;
  const int lane = threadIdx.x & 63, c = lane % L, j = c >> 2, g = c & 3;
  const int sub = D == 64 ? lane >> 5 : 0, tp = (lane / L) % TP;
  const int ps = 1 << a.r.ps_log2;
  const bool vec = VAL ? a.vvec : a.kvec;
  const int64_t srow = VAL ? a.vs : a.ks, shead = VAL ? a.vh : a.kh;
  const T* src = static_cast<const T*>(VAL ? a.v : a.k) + tp * srow + 8 * c;
  const bool first_half = 8 * c < (a.rot >> 1);
  const bool turns = MODE == kRotHalf || MODE == kRotInterleaved ? 8 * c < a.rot : false;
  const int other = first_half ? a.rot >> 1 : -(a.rot >> 1);  // the pairs' other elements (kRotHalf)
  walk_quads(a.r, units, hpu, s_q, s_wsum, s_tot, [&](int64_t p0, int t0, int o0, int o1, int pg, int h0, int nh) {
      const int at0 = (int)(p0 & (ps - 1));
      // the lane's positions
      bool on[PASS];
      const float2* tab[PASS];
      float2 cs[MODE == kRotHalf || MODE == kRotInterleaved ? PASS : 1][8];
      bool mine = true;
#pragma unroll
      for (int k = 0; k < PASS; ++k) {
        const int t = t0 + k * TP + tp;
        on[k] = t >= o0 && t < o1;
        tab[k] = nullptr;
        if (a.table && on[k]) {  // a row without a rotation is not appended at all
          const int64_t r = a.pos ? a.pos[t] : p0 + k * TP + tp;
          if (r < 0 || r >= a.max_pos) {
            if (!VAL) atomicOr(a.rope_err, 1);
            on[k] = false;
          } else
            tab[k] = a.table + r * (a.rot >> 1);
        }
        mine = mine && on[k];
        // the pairs of the lane's piece, for every head
        if (MODE == kRotHalf && on[k] && turns) {
          const int e = first_half ? 8 * c : 8 * c - (a.rot >> 1);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            cs[k][i] = tab[k][e + i];
            cs[k][i].y = first_half ? -cs[k][i].y : cs[k][i].y;
          }
        }
        if (MODE == kRotInterleaved && on[k] && turns) {
#pragma unroll
          for (int i = 0; i < 4; ++i) cs[k][i] = tab[k][4 * c + i];
        }
      }
      const bool all = __ballot(!mine) == 0;
      const T* x0 = src + t0 * srow + (h0 + sub) * shead;
      char* blk = a.r.pool + ((int64_t)pg * a.r.nkv + h0 + sub) * a.r.block;
      for (int h1 = 0; h1 < nh; h1 += HW, x0 += HW * shead, blk += HW * a.r.block) {
        const bool there = HW == 1 || h1 + sub < nh;
#pragma unroll
        for (int k = 0; k < PASS; ++k) {
          const bool act = on[k] && there;
          const int at = at0 + k * TP + tp;
          float f[8] = {0, 0, 0, 0, 0, 0, 0, 0};
          if (act) {
            const T* x = x0 + k * TP * srow;
            if (MODE == kRotAny) {
              rotated8(x - 8 * c, 8 * c, a.rot, a.half_layout, vec, tab[k], f);
            } else {
              load8(x, vec, f);
              if (MODE == kRotHalf && turns) {
                float o[8];
                load8(x + other, vec, o);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = f[i] * cs[k][i].x + o[i] * cs[k][i].y;
              }
              if (MODE == kRotInterleaved && turns) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float y0 = f[2 * i], y1 = f[2 * i + 1];
                  f[2 * i] = y0 * cs[k][i].x - y1 * cs[k][i].y;
                  f[2 * i + 1] = y1 * cs[k][i].x + y0 * cs[k][i].y;
                }
              }
            }
          }
          float lo8 = fminf(fminf(fminf(f[0], f[1]), fminf(f[2], f[3])), fminf(fminf(f[4], f[5]), fminf(f[6], f[7])));
          float hi8 = fmaxf(fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])), fmaxf(fmaxf(f[4], f[5]), fmaxf(f[6], f[7])));
          int bad = __builtin_isunordered(f[0], f[1]) | __builtin_isunordered(f[2], f[3]) |
                    __builtin_isunordered(f[4], f[5]) | __builtin_isunordered(f[6], f[7]);
          lo8 = fminf(lo8, dppf<kDppQuadSwap1>(lo8));
          hi8 = fmaxf(hi8, dppf<kDppQuadSwap1>(hi8));
          bad |= dpp<kDppQuadSwap1>(bad);
          lo8 = fminf(lo8, dppf<kDppQuadSwap2>(lo8));
          hi8 = fmaxf(hi8, dppf<kDppQuadSwap2>(hi8));
          bad |= dpp<kDppQuadSwap2>(bad);
          const bool nan = bad || too_large(lo8) || too_large(hi8);
          const uint32_t pair = kv_pair(lo8, hi8, nan);
          const uint32_t w = nan ? 0 : kv_codes8(f, pair);
          if (!VAL) {
            if (act) {
              *reinterpret_cast<uint32_t*>(blk + P::kc() + at * (D / 2) + (g * NG + j) * 4) = w;
              if (g == 0) *reinterpret_cast<uint32_t*>(blk + P::kp(ps) + (at * NG + j) * 4) = pair;
            }
            continue;
          }
          // d = 8 c + i = 64 hf + 16 n + r: nibble n of the u16 of r = 8 (c & 1) + i
          const int n = (c >> 1) & 3, hf = c >> 3;
          uint32_t v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t x = w >> (8 * i);
            v[i] = ((x & 15u) | (x & 0xf0u) << 12) << (4 * n);
            v[i] |= (uint32_t)dpp<kDppQuadSwap2>((int)v[i]);
            // lane c ^ 4: the mirror of eight lanes, then of four
            v[i] |= (uint32_t)dpp<0x1B>(dpp<kDppRowHalfMirror>((int)v[i]));
          }
          // of the four lanes that now hold the same eight u16, each takes two
          const uint32_t two = n == 0 ? v[0] : n == 1 ? v[1] : n == 2 ? v[2] : v[3];
          const int r = 8 * (c & 1) + 2 * n, tk = at & 3;
          const int o = ((r * 2 + (tk >> 1)) * HN + hf) * 2 + (tk & 1);
          if (all) {
            s_v[sub * D + o] = (uint16_t)two;
            s_v[sub * D + o + 4 * HN] = (uint16_t)(two >> 16);
          } else if (act) {
            uint16_t* vc = reinterpret_cast<uint16_t*>(blk + P::vc(ps)) + (at >> 2) * D;
            vc[o] = (uint16_t)two;
            vc[o + 4 * HN] = (uint16_t)(two >> 16);
          }
          if (act && g == 0) *reinterpret_cast<uint32_t*>(blk + P::vp(ps) + (j * ps + at) * 4) = pair;
        }
        if (VAL && all) {
          __builtin_amdgcn_wave_barrier();
          const int l = lane & (D == 64 ? 31 : 63);
          if (l < D / 8 && there)
            *reinterpret_cast<uint4*>(blk + P::vc(ps) + (at0 >> 2) * (2 * D) + l * 16) =
                *reinterpret_cast<const uint4*>(&s_v[sub * D + l * 8]);
          __builtin_amdgcn_wave_barrier();
        }
      }
  });
}

template <typename T, int D, int MODE>
__global__ __launch_bounds__(kKvThreads) void kv_append_kernel(AppendArgs a, int units, int hpu) {
  __shared__ int s_q[kSeqChunk], s_wsum[kKvThreads / 64], s_tot;
  __shared__ __align__(16) uint16_t s_v[kKvThreads / 64][D == 64 ? 2 * D : D];
  if (blockIdx.y == 0) append_part<T, D, MODE, false>(a, units, hpu, s_q, s_wsum, &s_tot, nullptr);
  else append_part<T, D, kRotNone, true>(a, units, hpu, s_q, s_wsum, &s_tot, s_v[threadIdx.x >> 6]);
}

struct GatherArgs {
  KvRows r;
  void *k, *v;
};

// The inverse: the same quads and lanes.  Of the four lanes that need the same eight
// u16 of a value's codes each loads two, and they exchange them.  14460 rows of 8 heads of
// 128 to BF16 (18.5 MB in, 59 MB out): 22.0 us, 3.5 TB/s (23.7 behind an append), 3.6 us for
// one; to f32 (118 MB out) 27.5 us, 5.0 TB/s.  Waits are 57% of a wave's cycles: the next
// head's loads are not under way.  The rows stay in the caches for whoever reads them next: with a
// copy of them behind, 40.8 us and to f32 76.4, where stores past the caches took 44.9 and
// 88.8 (alone 21.1 and 39.5).
template <typename T, int D, bool VAL>
__device__ __forceinline__ void gather_part(const GatherArgs& a, int units, int hpu, int* s_q, int* s_wsum, int* s_tot) {
  using P = KvParts<D>;
  constexpr int NG = D / kKvGroup, HN = D / 64, L = QuadLanes<D>::L;
  constexpr int TP = QuadLanes<D>::TP, PASS = QuadLanes<D>::PASS, HW = QuadLanes<D>::HW;
  const int lane = threadIdx.x & 63, c = lane % L, j = c >> 2, g = c & 3;
  const int sub = D == 64 ? lane >> 5 : 0, tp = (lane / L) % TP;
  const int ps = 1 << a.r.ps_log2;
  const int64_t srow = (int64_t)a.r.nkv * D;
  T* dst = static_cast<T*>(VAL ? a.v : a.k) + tp * srow + 8 * c;
  const int n = (c >> 1) & 3, hf = c >> 3, r = 8 * (c & 1) + 2 * n;
  walk_quads(a.r, units, hpu, s_q, s_wsum, s_tot, [&](int64_t p0, int t0, int o0, int o1, int pg, int h0, int nh) {
    const int at0 = (int)(p0 & (ps - 1));
    T* y0 = dst + t0 * srow + (int64_t)(h0 + sub) * D;
    const char* blk = a.r.pool + ((int64_t)pg * a.r.nkv + h0) * a.r.block;
    for (int h1 = 0; h1 < nh; h1 += HW, y0 += HW * D, blk += HW * a.r.block) {
      const bool there = HW == 1 || h1 + sub < nh;
      const char* mine = blk + (there ? sub : 0) * a.r.block;  // lanes without a head read the first one's
#pragma unroll
      for (int k = 0; k < PASS; ++k) {
        const int t = t0 + k * TP + tp, at = at0 + k * TP + tp;
        const bool act = there && t >= o0 && t < o1;
        uint32_t pr, q[4];
        if (VAL) {
          const uint16_t* vc = reinterpret_cast<const uint16_t*>(mine + P::vc(ps)) + (at >> 2) * D;
          const int o = ((r * 2 + ((at >> 1) & 1)) * HN + hf) * 2 + (at & 1);
          const uint32_t w0 = vc[o] | (uint32_t)vc[o + 4 * HN] << 16;
          pr = *reinterpret_cast<const uint32_t*>(mine + P::vp(ps) + (j * ps + at) * 4);
          // of lanes c, c ^ 2, c ^ 4, c ^ 6, put in the order of their n
          const uint32_t w1 = (uint32_t)dpp<kDppQuadSwap2>((int)w0);
          const uint32_t w2 = (uint32_t)dpp<0x1B>(dpp<kDppRowHalfMirror>((int)w0));
          const uint32_t w3 = (uint32_t)dpp<kDppQuadSwap2>((int)w2);
          const uint32_t a0 = (n & 1) ? w1 : w0, a1 = (n & 1) ? w0 : w1, a2 = (n & 1) ? w3 : w2, a3 = (n & 1) ? w2 : w3;
          q[0] = (n & 2) ? a2 : a0;
          q[1] = (n & 2) ? a3 : a1;
          q[2] = (n & 2) ? a0 : a2;
          q[3] = (n & 2) ? a1 : a3;
        } else {
          const uint32_t w = *reinterpret_cast<const uint32_t*>(mine + P::kc() + at * (D / 2) + (g * NG + j) * 4);
          pr = *reinterpret_cast<const uint32_t*>(mine + P::kp(ps) + (at * NG + j) * 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) q[i] = w >> (8 * i);
        }
        const float s = __uint_as_float(pr & 0xffff0000u), m = __uint_as_float(pr << 16);
        float f[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f[2 * i] = s * (float)(VAL ? (q[i] >> (4 * n)) & 15 : q[i] & 15) + m;
          f[2 * i + 1] = s * (float)(VAL ? (q[i] >> (4 * n + 16)) & 15 : (q[i] >> 4) & 15) + m;
        }
        if (act) store8(y0 + k * TP * srow, true, f);
      }
    }
  });
}

template <typename T, int D>
__global__ __launch_bounds__(kKvThreads) void kv_gather_kernel(GatherArgs a, int units, int hpu) {
  __shared__ int s_q[kSeqChunk], s_wsum[kKvThreads / 64], s_tot;
  if (blockIdx.y == 0) gather_part<T, D, false>(a, units, hpu, s_q, s_wsum, &s_tot);
  else gather_part<T, D, true>(a, units, hpu, s_q, s_wsum, &s_tot);
}

template <typename T, int D>
static void append_launch_m(const AppendArgs& a, dim3 g, int units, int hpu, hipStream_t st) {
  const dim3 blk(kKvThreads);
  if (a.mode == kRotNone) hipLaunchKernelGGL((kv_append_kernel<T, D, kRotNone>), g, blk, 0, st, a, units, hpu);
  else if (a.mode == kRotHalf) hipLaunchKernelGGL((kv_append_kernel<T, D, kRotHalf>), g, blk, 0, st, a, units, hpu);
  else if (a.mode == kRotInterleaved)
    hipLaunchKernelGGL((kv_append_kernel<T, D, kRotInterleaved>), g, blk, 0, st, a, units, hpu);
  else hipLaunchKernelGGL((kv_append_kernel<T, D, kRotAny>), g, blk, 0, st, a, units, hpu);
}
template <typename T>
static void append_launch(int d, const AppendArgs& a, dim3 g, int units, int hpu, hipStream_t st) {
  if (d == 64) append_launch_m<T, 64>(a, g, units, hpu, st);
  else if (d == 128) append_launch_m<T, 128>(a, g, units, hpu, st);
  else append_launch_m<T, 256>(a, g, units, hpu, st);
}
template <typename T>
static void gather_launch(int d, const GatherArgs& a, dim3 g, int units, int hpu, hipStream_t st) {
  if (d == 64) hipLaunchKernelGGL((kv_gather_kernel<T, 64>), g, dim3(kKvThreads), 0, st, a, units, hpu);
  else if (d == 128) hipLaunchKernelGGL((kv_gather_kernel<T, 128>), g, dim3(kKvThreads), 0, st, a, units, hpu);
  else hipLaunchKernelGGL((kv_gather_kernel<T, 256>), g, dim3(kKvThreads), 0, st, a, units, hpu);
}

// The grid: one head (two of 64 elements) a wave until there are waves enough,
// then up to eight in turn, which share the search for the quad's sequence and page.
static int quad_grid(const kh_paged_kv* c, int64_t rows, int64_t batch, int* units, int* hpu, dim3* g) {
  const int hw = c->d == 64 ? 2 : 1;
  const int64_t waves = (rows / 4 + batch) * ((c->nkv + hw - 1) / hw);
  int n = hw;
  while (n < 8 && n < c->nkv && waves * hw / n > 16384) n *= 2;
  *hpu = n;
  *units = (c->nkv + n - 1) / n;
  const int64_t blocks = ((rows / 4 + 2 * batch) * *units + 3) / 4;
  KH_CHECK_ARG(blocks < (int64_t)1 << 28, "too many rows for one call");
  *g = dim3((unsigned)(blocks < 1024 ? blocks : 1024), 2);
  return KH_OK;
}

// The arguments every call over rows of sequences checks.
static int rows_args(const kh_paged_kv* c, int dtype, int64_t rows, const int64_t* off, int64_t batch,
                     const int64_t* start, const int32_t* table, int64_t cols, int64_t table_stride, KvRows* r) {
  KH_CHECK_ARG(c != nullptr, "null handle");
  KH_CHECK_ARG(dtype == KH_DT_F32 || dtype == KH_DT_BF16, "dtype %d: f32 and BF16 are supported", dtype);
  KH_CHECK_ARG(rows >= 0 && batch >= 0, "rows %lld, batch %lld", (long long)rows, (long long)batch);
  KH_CHECK_ARG(rows < (int64_t)1 << 31, "%lld rows: too many for one call", (long long)rows);
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
    return paged_attn_prepare(c->d);
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
  // cleared before any other stream records again: streams need not wait for the null stream
  KH_HIP(hipStreamSynchronize(nullptr));
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
  a.mode = !rope ? kRotNone
           : rope->rot % (a.half_layout ? 16 : 8) ? kRotAny
           : a.half_layout ? kRotHalf : kRotInterleaved;
  a.rope_err = rope ? rope->err : nullptr;
  a.kvec = aligned16(k_dev, dtype, k_row_stride, k_head_stride) ? 1 : 0;
  a.vvec = aligned16(v_dev, dtype, v_row_stride, v_head_stride) ? 1 : 0;
  int units, hpu;
  dim3 g;
  const int grc = quad_grid(c, rows, batch, &units, &hpu, &g);
  if (grc != KH_OK) return grc;
  if (dtype == KH_DT_F32) append_launch<float>(c->d, a, g, units, hpu, as_stream(stream));
  else append_launch<uint16_t>(c->d, a, g, units, hpu, as_stream(stream));
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
  int units, hpu;
  dim3 g;
  const int grc = quad_grid(c, rows, batch, &units, &hpu, &g);
  if (grc != KH_OK) return grc;
  if (dtype == KH_DT_F32) gather_launch<float>(c->d, a, g, units, hpu, as_stream(stream));
  else gather_launch<uint16_t>(c->d, a, g, units, hpu, as_stream(stream));
  KH_LAUNCHED();
  return KH_OK;
}
