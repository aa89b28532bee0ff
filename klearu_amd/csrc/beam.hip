// beam.hip -- the best continuations of beams over a vocabulary (gfx950).
//
//   y[i][v] = scores[i] + x[i][v] - log sum_w exp(x[i][w]),   top k of y over (i, v)
//
// One pass over the logits: a wave takes a part of a row and leaves the sum of exp(x - m) and its
// k largest logits; a second kernel joins a sequence's parts.  Within a beam y orders as x does, so
// parts compare logits as integers, of equal ones the first.  Between beams the log-sum-exps
// decide: they are f64, of f32 exponentials with what log2 e and the rounded maximum lack put back, since
// sums that are 1e-7 off swap continuations of a batch of beams now and then.  The order of a row's sums depends on
// the call's sizes only, so that beams that are alike tie.
//
// The k largest: of W waves that share a row, the smallest of their own (k / W)-th largest logits, T, has k logits at
// or above it, so that no others can be among the k largest.  Waves tell each other theirs: of the first tile's
// lanes' maxima before any list begins, later whenever a wave's list has doubled.  A wave's own k-th largest of its
// lanes' maxima bounds what one tile can add (16 a lane) where the others' logits are smaller.  What passes goes to a list in
// LDS, which is cut to k when it fills and at the end: the k-th largest is found bit by bit, counted with
// ballots.  When a wave sees what another tells changes its list, not the k largest of all.
//
// Both kernels, 512 rows of 131071 BF16 logits, k 16: 56 us (48 and 7), 2.4 TB/s of logits.  The first one's 210 instructions
// for 1024 logits, of which 16 are exponentials at a quarter of the rate, take the SIMDs 27 us, and a copy reads as much in
// 28: loads and work hardly overlap, with one tile ahead and chains of ballots in between.  k 32 takes 76 us, and 64,
// which nobody has looked into, 404.  One pass is all that a row needs; waves take its tiles side by side (59 us with a
// range each).
#include <algorithm>

#include "paged_kv.hpp"

namespace kh {

constexpr int kBmThreads = 512, kBmWaves = kBmThreads / 64;
constexpr int kBmEach = 16;             // logits of a lane
constexpr int kBmTile = 64 * kBmEach;   // of a wave
// Waves that the chip holds at once, in us with 2048 / 4096 / 8192 of them: 512 rows of 131071 BF16 logits 71 / 53 / 70, of
// 32000 35 / 31 / 36; 64 rows of 131071 23.3 / 22.9 / 28.3; 1200 of 32000 77 / 66 / 63.
constexpr int64_t kBmFill = 4096;

struct BeamArgs {
  const void* x;
  int64_t row_stride, batch, vocab;
  int beams, k, parts;  // parts of a row: every parts-th tile
  int slots;            // waves of a row: parts, rounded up so that whole rows or whole blocks go together
  const float* scores;
  const uint8_t* done;
  int64_t end;
  float* out_y;
  int32_t *out_i, *out_v;
  uint64_t* top;  // [rows][parts][k] f32_key << 32 | ~token; 0: none
  double* sum;    // [rows][parts] of exp(x - max)
  float* max;
};

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m);
  return v;
}

// log2 e is 0x1.715476p+0f and 1.9e-8 more.  Sums of z = exp2(y), y = x log2 e - c rounded once, have the rest of log2 e and
// of c put back: the sum of z y times ln 2 (rest / log2 e).
constexpr float kBmHi = 0x1.715476p+0f;
constexpr double kBmLo = 0x1.62e42fefa39efp-1 * (0x1.4ae0bf85ddf44p-26 / 0x1.715476p+0);
// exp(t), t <= 88, within 1e-7 and without a bias, for logits of any size.  Not for -inf.
__device__ __forceinline__ float beam_exp(float t) {
  const float lo = 0x1.4ae0cp-26f;
  const float y = t * kBmHi, r = fmaf(t, lo, fmaf(t, kBmHi, -y));
  const float e = __builtin_amdgcn_exp2f(y);
  return fmaf(e, r * 0x1.62e43p-1f, e);
}

// 16 bytes of a row from any element on.  Tiles begin with the row and not at a 16-byte border, so that where a row
// starts does not change how its exponentials are grouped: beams that are alike have the same sums.
template <typename T>
__device__ __forceinline__ uint4 beam_load(const T* p) {
  uint4 w;
  __builtin_memcpy(&w, p, sizeof w);
  return w;
}

// The largest T of which `count(T)` entries are at or above it: the k-th largest of 32-bit entries; all
// bits below `last` are zero in T (they say nothing of the entries).
template <typename F>
__device__ __forceinline__ uint32_t kth_largest(int k, int last, F count) {
  uint32_t T = 0;
  for (int bit = 31; bit >= last; --bit) {
    const uint32_t c = T | 1u << bit;
    if (count(c) >= k) T = c;
  }
  return T;
}
__device__ __forceinline__ int ballots(bool p) { return __popcll(__ballot(p)); }

template <int KC>
constexpr int kBmList = (18 * KC + 63) / 64 * 64;  // less than 2 k before a tile, and what it adds
// Cuts a wave's list of n > k different entries to its k largest, in any order; returns the upper word of
// the smallest of them.
template <int KC>
__device__ __forceinline__ uint32_t beam_cut(uint64_t* list, int n, int k, int last, int lane) {
  constexpr int C = kBmList<KC> / 64;  // entries of a lane
  __builtin_amdgcn_wave_barrier();  // the wave's writes are in order before its reads
  uint64_t x[C];
#pragma unroll
  for (int c = 0; c < C; ++c) x[c] = c * 64 + lane < n ? list[c * 64 + lane] : 0;
  const uint32_t T = kth_largest(k, last, [&](uint32_t v) {
    int m = 0;
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (c * 64 < n) m += ballots((uint32_t)(x[c] >> 32) >= v);
    return m;
  });
  const auto high = [&](uint64_t y) { return (uint32_t)(y >> 32) >> last; };
  int above = 0, same = 0;
#pragma unroll
  for (int c = 0; c < C; ++c)
    if (c * 64 < n) {
      above += ballots(high(x[c]) > T >> last);
      same += ballots(x[c] != 0 && high(x[c]) == T >> last);
    }
  uint32_t least = 0;  // of those equal to T, the lower word that the last one kept has
  if (same > k - above)
    least = kth_largest(k - above, 0, [&](uint32_t v) {
      int m = 0;
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (c * 64 < n) m += ballots(x[c] != 0 && high(x[c]) == T >> last && (uint32_t)x[c] >= v);
      return m;
    });
  int at = 0;
  uint32_t key = 0;
#pragma unroll
  for (int c = 0; c < C; ++c)
    if (c * 64 < n) {
      const bool keep = x[c] != 0 && (high(x[c]) > T >> last || (high(x[c]) == T >> last && (uint32_t)x[c] >= least));
      const uint64_t b = __ballot(keep);
      if (keep) list[at + __popcll(b & ((1ull << lane) - 1))] = x[c];
      at += __popcll(b);
      const uint64_t least_ones = __ballot(keep && high(x[c]) == T >> last);
      if (least_ones) key = __builtin_amdgcn_readlane((uint32_t)(x[c] >> 32), __builtin_ctzll(least_ones));
    }
  __builtin_amdgcn_wave_barrier();
  return key;
}

// KC: at least k; a tile adds no more than 16 k entries to the list.  It is cut as soon as it holds 2 k: the
// higher T, the fewer of the next logits pass it (with the first tile's T 16 of every tile do).
template <typename T, int KC>
__global__ __launch_bounds__(kBmThreads) void beam_part_kernel(BeamArgs a) {
  constexpr int V = 16 / sizeof(T), Q = kBmEach / V, LAST = sizeof(T) == 2 ? 16 : 0;
  extern __shared__ __align__(16) uint64_t s_lists[];  // [waves][kBmList]
  __shared__ uint32_t s_told[2][kBmWaves];             // of a row and of the next one
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint64_t* list = s_lists + wave * kBmList<KC>;
  const int64_t waves = a.batch * a.beams * a.slots;
  int turn = 0;
  for (int64_t block = (int64_t)blockIdx.x * kBmWaves; block < waves; block += (int64_t)gridDim.x * kBmWaves, turn ^= 1) {
    const int64_t slot = block + wave, r = min(slot, waves - 1) / a.slots;
    const int part = slot < waves ? (int)(slot - r * a.slots) : a.parts;
    const int64_t id = r * a.parts + part;
    // the waves of the block that share the row, and how many of their largest all of them together need
    const int group = min(a.slots, kBmWaves), leader = wave & ~(group - 1), shared = min(group, a.parts - (part & ~(group - 1)));
    const int few = shared > 0 ? (a.k + shared - 1) / shared : a.k;
    uint32_t* told = s_told[turn];
    const T* row = static_cast<const T*>(a.x) + r * a.row_stride;
    const int end = (int)a.vocab;
    const int first = part * kBmTile, last = part < a.parts ? end : 0, step = a.parts * kBmTile;  // waves side by side
    // What the wave's exponentials are taken from, near its largest logit, so that those that count have small exponents and
    // small rounding errors of them; times log2 e; what its rounding makes of the sums.
    float ref = -INFINITY, c = -INFINITY;
    double scale = 1.0;
    double sum = 0.0;
    int n = 0, next_n = 2 * few;
    uint32_t tk = 0, tv = 0;  // T, and its token (inverted): entries below it are of no use
    const auto tell = [&](uint32_t v) { __hip_atomic_store(&told[wave], v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP); };
    const auto hear = [&] {
      const uint32_t v = __hip_atomic_load(&told[leader + min(lane, max(shared, 1) - 1)], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      uint32_t all = wave_min_u32(v);
      if (LAST == 16 && all != 0 && all >> 31 == 0) all |= 0xffffu;  // the whole key of a negative BF16
      if (all > tk) tk = all, tv = 0;  // equal ones may come before those that were counted
    };
    if (first >= last) {
      if (lane == 0) tell(0);
      __syncthreads();
    }
    uint4 next[Q];
    const auto inside = [&](int p) { return p + kBmTile <= end; };
    const auto fetch = [&](int p) {
      if (inside(p)) {
#pragma unroll
        for (int q = 0; q < Q; ++q) next[q] = beam_load(row + p + (q * 64 + lane) * V);
      }
    };
    if (first < last) fetch(first);
    for (int p = first; p < last; p += step) {
      float x[kBmEach];
      const bool whole = inside(p);
      if (whole) {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          const uint4 w = next[q];
          if constexpr (V == 4) {
            x[4 * q] = __uint_as_float(w.x); x[4 * q + 1] = __uint_as_float(w.y);
            x[4 * q + 2] = __uint_as_float(w.z); x[4 * q + 3] = __uint_as_float(w.w);
          } else {
            x[8 * q] = bf16_lo(w.x); x[8 * q + 1] = bf16_hi(w.x); x[8 * q + 2] = bf16_lo(w.y); x[8 * q + 3] = bf16_hi(w.y);
            x[8 * q + 4] = bf16_lo(w.z); x[8 * q + 5] = bf16_hi(w.z); x[8 * q + 6] = bf16_lo(w.w); x[8 * q + 7] = bf16_hi(w.w);
          }
        }
        if (p + step < last) fetch(p + step);
      } else {
#pragma unroll
        for (int e = 0; e < kBmEach; ++e) {
          const int at = p + (e / V * 64 + lane) * V + e % V;
          x[e] = at < end ? load_f32(row + at) : -INFINITY;
        }
        if (p + step < last) fetch(p + step);
      }
      float m = x[0];
#pragma unroll
      for (int e = 1; e < kBmEach; ++e) m = fmaxf(m, x[e]);
      if (__ballot(m > ref + 2.0f)) {
        const float most = wave_max(fmaxf(m, ref));
        sum = sum == 0.0 ? 0.0 : sum * exp((double)ref - (double)most);
        ref = most;
        c = ref * kBmHi;
        const double d = (double)fmaf(ref, kBmHi, -c) * 0x1.62e42fefa39efp-1;
        scale = 1.0 - d + 0.5 * d * d;
      }
      float s = 0.0f, sy = 0.0f;
#pragma unroll
      for (int e = 0; e < kBmEach; ++e) {
        const float y = fmaf(x[e], kBmHi, -c), z = __builtin_amdgcn_exp2f(y);
        s += z;
        sy = fmaf(z, y, sy);
      }
      const float both = s + sy;
      if (__ballot(both != both || !(__builtin_fabsf(ref) <= 4096.0f))) {
        // -inf or the type's lowest value among them, or what makes the sum NaN, or large ones
        float none = -150.0f;
        asm volatile("" : "+v"(none));  // keeps this behind its branch
        s = 0.0f;
#pragma unroll
        for (int e = 0; e < kBmEach; ++e) s += x[e] == -INFINITY || x[e] - ref < none ? 0.0f : beam_exp(x[e] - ref);
        sum += (double)s;
      } else {
        sum += (double)s * scale + (double)sy * kBmLo;
      }

      // the lane's largest (of the row's own: those past its end are -inf, too, but no entries)
      const uint32_t mk = f32_key(m);
      const auto passes = [&] { return mk >= tk + (tv == ~0u ? 1 : 0); };
      if (p == first) {
        const uint32_t v = few == 1 ? wave_max_u32(mk) : kth_largest(few, LAST, [&](uint32_t v) { return ballots(mk >= v); });
        if (lane == 0) tell(v);
        __syncthreads();
        hear();
      } else if (__ballot(passes())) {
        hear();
      }
      bool mine = passes();
      const uint64_t better = __ballot(mine);
      if (!better) continue;
      const auto there = [&](int e) {
        const int at = p + (e / V * 64 + lane) * V + e % V;
        return whole || at < end;
      };
      const auto token = [&](int e) { return ~(uint32_t)(p + (e / V * 64 + lane) * V + e % V); };
      if (__popcll(better) >= a.k) {
        uint32_t bk = 0, bv = 0;
#pragma unroll
        for (int e = 0; e < kBmEach; ++e) {
          const uint32_t key = f32_key(x[e]);
          if (there(e) && key > bk) bk = key, bv = token(e);
        }
        const uint32_t kth = kth_largest(a.k, LAST, [&](uint32_t v) { return ballots(bk >= v); }) >> LAST;
        if (kth != 0 && kth >= tk >> LAST) {
          // of the lanes whose maximum is T the first ones, by their tokens
          const int above = ballots(bk >> LAST > kth);
          const uint64_t same = __ballot(bk >> LAST == kth);
          tv = 0;
          if (__popcll(same) > a.k - above)
            tv = kth_largest(a.k - above, 0, [&](uint32_t v) { return ballots(bk >> LAST == kth && bv >= v); });
          tk = __builtin_amdgcn_readlane(bk, __builtin_ctzll(same));
          mine = true;
        }
      }
      // at or above T, as floats (a NaN is not); then exactly
      const float from = !mine ? INFINITY : tk == 0 ? -INFINITY : __uint_as_float(tk >> 31 ? tk & 0x7fffffffu : ~tk);
#pragma unroll
      for (int e = 0; e < kBmEach; ++e) {
        if (!__ballot(x[e] >= from)) continue;
        const uint32_t key = f32_key(x[e]);
        const bool take = mine && x[e] >= from && there(e) && (key > tk || token(e) >= tv);
        const uint64_t b = __ballot(take);
        if (b) {
          if (take) list[n + __popcll(b & ((1ull << lane) - 1))] = (uint64_t)key << 32 | token(e);
          n += __popcll(b);
        }
      }
      if (n >= 2 * a.k) {
        tk = beam_cut<KC>(list, n, a.k, LAST, lane);
        n = a.k;
        tv = ~0u;  // the next ones have to be above it
      }
      if (n >= next_n && n <= 64 && p + step < last) {
        next_n = 2 * n;
        __builtin_amdgcn_wave_barrier();
        const uint32_t key = lane < n ? (uint32_t)(list[lane] >> 32) : 0;
        const uint32_t v = kth_largest(few, LAST, [&](uint32_t v) { return ballots(key >= v); });
        if (lane == 0) tell(v);
      }
    }
    if (n > a.k) beam_cut<KC>(list, n, a.k, LAST, lane), n = a.k;
    if (part >= a.parts) continue;
    uint64_t* top = a.top + id * a.k;
    if (lane < a.k) top[lane] = lane < n ? list[lane] : 0;
    const double total = wave_sum_f64(sum);
    if (lane == 0) {
      a.max[id] = ref;
      a.sum[id] = total;
    }
  }
}

// A score as an integer of the same order.
__device__ __forceinline__ uint64_t f64_key(double y) {
  const uint64_t u = (uint64_t)__double_as_longlong(y + 0.0);
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ double key_f64(uint64_t k) {
  return __longlong_as_double((long long)(k >> 63 ? k & 0x7fffffffffffffffull : ~k));
}

// Block: a sequence.  A chain of loads: what its threads need of the parts is asked for at once, before
// the log-sum-exps that it is scored with.
constexpr int kBjThreads = 512, kBjEach = 4, kBjList = 1024;

__global__ __launch_bounds__(kBjThreads) void beam_join_kernel(BeamArgs a) {
  constexpr int W = kBjThreads / 64;
  __shared__ double s_score[KH_MAX_BEAMS], s_top[KH_MAX_BEAMS], s_log[KH_MAX_BEAMS];  // and the log-sum-exp's parts
  __shared__ int s_kind[KH_MAX_BEAMS];  // 0: its parts' logits, 1: none, 2: at its end
  // a continuation's score, and what orders equal ones, from the first: the beam, its logit (the largest
  // first: a score may have no digits for the difference), the token
  __shared__ uint64_t s_key[kBjList], s_tie[kBjList], s_bk[W], s_bt[W];
  __shared__ uint32_t s_t;
  __shared__ int s_n;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int each = a.parts * a.k, all = a.beams * each;
  for (int64_t b = blockIdx.x; b < a.batch; b += gridDim.x) {
    const uint64_t* top = a.top + b * all;
    uint64_t mine[kBjEach];
#pragma unroll
    for (int c = 0; c < kBjEach; ++c) mine[c] = top[min(t + c * kBjThreads, all - 1)];
    for (int i = wave; i < a.beams; i += W) {
      const int64_t r = b * a.beams + i, at = r * a.parts;
      const float m0 = lane < a.parts ? a.max[at + lane] : -INFINITY;
      const double d0 = lane < a.parts ? a.sum[at + lane] : 0.0;
      const double score = (double)a.scores[r];
      const bool ended = a.done && a.done[r];
      float m = m0;
      for (int c = 64 + lane; c < a.parts; c += 64) m = fmaxf(m, a.max[at + c]);
      m = wave_max(m);
      double s = d0 == 0.0 ? 0.0 : d0 * exp((double)m0 - (double)m);
      for (int c = 64 + lane; c < a.parts; c += 64) {
        const double d = a.sum[at + c];
        s += d == 0.0 ? 0.0 : d * exp((double)a.max[at + c] - (double)m);
      }
      s = wave_sum_f64(s);
      if (lane == 0) {
        const double l = log(s);
        const bool fine = __builtin_isfinite(score), has = __builtin_isfinite(m) && __builtin_isfinite(l);
        s_kind[i] = !fine ? 1 : ended ? 2 : has ? 0 : 1;
        s_score[i] = score;
        s_top[i] = (double)m;
        s_log[i] = l;
      }
    }
    if (t == 0) s_n = 0, s_t = 0;
    __syncthreads();
    // continuation j with entry w of its part: its key (0: there is none) and its order among equal ones
    const auto get = [&](int j, uint64_t w, uint64_t& tie) -> uint64_t {
      const int i = (int)((uint32_t)j / (uint32_t)each), e = j - i * each, kind = s_kind[i];
      tie = (uint64_t)i << 56;
      if (kind == 0) {
        const uint32_t k32 = (uint32_t)(w >> 32);
        const double x = (double)__uint_as_float(k32 >> 31 ? k32 & 0x7fffffffu : ~k32);
        tie |= (uint64_t)~k32 << 24 | ~(uint32_t)w;
        return w ? f64_key(s_score[i] + ((x - s_top[i]) - s_log[i])) : 0;  // logits of any size leave the score its bits
      }
      // the first tokens, all of them -inf, but for the end
      if (e >= a.k || e >= a.vocab) return 0;
      tie |= kind == 1 || e > a.end ? e : e == 0 ? (uint32_t)a.end : e - 1;
      return f64_key(kind == 2 && e == 0 ? s_score[i] : -INFINITY);
    };
    uint64_t key[kBjEach];
    uint64_t tie[kBjEach];
    // the k-th largest of the lanes' own maxima, by their upper words
    uint32_t most = 0;
#pragma unroll
    for (int c = 0; c < kBjEach; ++c) {
      const int j = t + c * kBjThreads;
      key[c] = j < all ? get(j, mine[c], tie[c]) : 0;
      most = max(most, (uint32_t)(key[c] >> 32));
    }
    for (int j = t + kBjEach * kBjThreads; j < all; j += kBjThreads) {
      uint64_t f;
      most = max(most, (uint32_t)(get(j, top[j], f) >> 32));
    }
    const uint32_t Tw = kth_largest(a.k, 0, [&](uint32_t v) { return ballots(most >= v); });
    if (lane == 0) atomicMax(&s_t, Tw);
    __syncthreads();
    const uint32_t T = s_t;
    const auto list = [&](uint64_t y, uint64_t f) {
      if (y != 0 && (uint32_t)(y >> 32) >= T) {
        const int at = atomicAdd(&s_n, 1);
        if (at < kBjList) s_key[at] = y, s_tie[at] = f;
      }
    };
#pragma unroll
    for (int c = 0; c < kBjEach; ++c) list(key[c], tie[c]);
    for (int j = t + kBjEach * kBjThreads; j < all; j += kBjThreads) {
      uint64_t f;
      const uint64_t y = get(j, top[j], f);
      list(y, f);
    }
    __syncthreads();
    const int n = s_n;
    const auto put = [&](int at, uint64_t y, uint64_t f) {
      a.out_y[b * a.k + at] = (float)key_f64(y);
      a.out_i[b * a.k + at] = (int32_t)(f >> 56);
      a.out_v[b * a.k + at] = (int32_t)(f & 0xffffffu);
    };
    if (n <= kBjList) {
      for (int i0 = 0; i0 < n; i0 += kBjThreads / 8) {  // eight lanes an entry
        const int i = min(i0 + (t >> 3), n - 1);
        const uint64_t y = s_key[i];
        const uint64_t f = s_tie[i];
        int above = 0;
        for (int j = t & 7; j < n; j += 8) above += s_key[j] > y || (s_key[j] == y && s_tie[j] < f) ? 1 : 0;
        above += dpp<kDppQuadSwap1>(above);
        above += dpp<kDppQuadSwap2>(above);
        above += dpp<kDppRowHalfMirror>(above);
        if ((t & 7) == 0 && i0 + (t >> 3) < n && above < a.k) put(above, y, f);
      }
    } else {  // many equal scores: the best, time after time
      uint64_t lk = ~0ull, lf = 0;  // the last one written
      for (int i = 0; i < a.k; ++i) {
        uint64_t bk = 0, bf = ~0ull;
        for (int j = t; j < all; j += kBjThreads) {
          uint64_t f;
          const uint64_t y = get(j, top[j], f);
          if (y != 0 && (y < lk || (y == lk && f > lf)) && (y > bk || (y == bk && f < bf))) bk = y, bf = f;
        }
#pragma unroll
        for (int m = 32; m > 0; m >>= 1) {
          const uint64_t ok = __shfl_xor((unsigned long long)bk, m);
          const uint64_t of = __shfl_xor((unsigned long long)bf, m);
          if (ok > bk || (ok == bk && of < bf)) bk = ok, bf = of;
        }
        __syncthreads();
        if (lane == 0) s_bk[wave] = bk, s_bt[wave] = bf;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w)
          if (s_bk[w] > bk || (s_bk[w] == bk && s_bt[w] < bf)) bk = s_bk[w], bf = s_bt[w];
        lk = bk;
        lf = bf;
        if (t == 0) put(i, bk, bf);
      }
    }
    __syncthreads();
  }
}

static int beam_shape(int64_t batch, int beams, int64_t vocab, int k) {
  KH_CHECK_ARG(beams >= 1 && beams <= KH_MAX_BEAMS, "%d beams not in [1,%d]", beams, KH_MAX_BEAMS);
  KH_CHECK_ARG(batch >= 0 && batch < ((int64_t)1 << 31) / beams, "batch %lld", (long long)batch);
  KH_CHECK_ARG(vocab >= 1 && vocab <= (int64_t)1 << 24, "vocab %lld not in [1,2^24]", (long long)vocab);
  KH_CHECK_ARG(k >= 1 && k <= KH_MAX_BEAM_K && k <= beams * vocab, "k %d not in [1,%d] or more than there are", k,
               KH_MAX_BEAM_K);
  return KH_OK;
}
// Parts of a row (tiles of a part): as many waves as the chip holds.
struct BeamPlan {
  int parts, slots;
};
static BeamPlan beam_plan(int64_t rows, int64_t vocab) {
  const int64_t all = (vocab + kBmTile - 1) / kBmTile;
  const int64_t want = std::max<int64_t>(std::min(kBmFill / std::max<int64_t>(rows, 1), all), 1);
  BeamPlan p;
  const int64_t tiles = (all + want - 1) / want;  // of a part
  p.parts = (int)((all + tiles - 1) / tiles);
  p.slots = 1;
  while (p.slots < p.parts && p.slots < kBmWaves) p.slots *= 2;
  if (p.parts > kBmWaves) p.slots = (p.parts + kBmWaves - 1) / kBmWaves * kBmWaves;
  return p;
}
static int64_t beam_space(int64_t batch, int beams, int64_t vocab, int k) {
  return batch * beams * beam_plan(batch * beams, vocab).parts * (8 * (int64_t)k + 8 + 4);
}
template <typename T, int KC>
static void beam_launch_k(const BeamArgs& a, hipStream_t st) {
  const int64_t blocks = (a.batch * a.beams * a.slots + kBmWaves - 1) / kBmWaves;
  hipLaunchKernelGGL((beam_part_kernel<T, KC>), dim3((unsigned)std::min<int64_t>(blocks, 1 << 20)), dim3(kBmThreads),
                     kBmWaves * kBmList<KC> * 8, st, a);
}
template <typename T>
static void beam_launch(const BeamArgs& a, hipStream_t st) {
  if (a.k <= 16) beam_launch_k<T, 16>(a, st);
  else if (a.k <= 32) beam_launch_k<T, 32>(a, st);
  else beam_launch_k<T, 64>(a, st);
}

}  // namespace kh

using namespace kh;

extern "C" int kh_beam_select_workspace(int64_t batch, int beams, int64_t vocab, int k, int64_t* bytes) {
  KH_CHECK_ARG(bytes != nullptr, "null output");
  const int rc = beam_shape(batch, beams, vocab, k);
  if (rc != KH_OK) return rc;
  *bytes = beam_space(batch, beams, vocab, k);
  return KH_OK;
}

extern "C" int kh_beam_select(int dtype, const void* logits_dev, int64_t row_stride, int64_t batch, int beams,
                              int64_t vocab, const float* scores_dev, const uint8_t* done_dev, int64_t end, int k,
                              float* out_scores_dev, int32_t* out_beams_dev, int32_t* out_tokens_dev, void* ws_dev,
                              int64_t ws_bytes, void* stream) {
  KH_CHECK_ARG(dtype == KH_DT_F32 || dtype == KH_DT_BF16, "dtype %d: f32 and BF16 are supported", dtype);
  const int rc = beam_shape(batch, beams, vocab, k);
  if (rc != KH_OK) return rc;
  KH_CHECK_ARG(row_stride >= 0, "negative stride");
  KH_CHECK_ARG(!done_dev || (end >= 0 && end < vocab), "end %lld not in [0,%lld)", (long long)end, (long long)vocab);
  if (batch == 0) return KH_OK;
  KH_CHECK_ARG((reinterpret_cast<uintptr_t>(logits_dev) & (dtype_bytes(dtype) - 1)) == 0, "the logits are not aligned");
  KH_CHECK_ARG(logits_dev && scores_dev && out_scores_dev && out_beams_dev && out_tokens_dev, "null argument");
  const int64_t need = beam_space(batch, beams, vocab, k), rows = batch * beams;
  if (!ws_dev || ws_bytes < need) {
    set_error("the workspace holds %lld bytes, %lld are needed", (long long)(ws_dev ? ws_bytes : 0), (long long)need);
    return KH_ERR_CAPACITY;
  }
  KH_CHECK_ARG((reinterpret_cast<uintptr_t>(ws_dev) & 15) == 0, "the workspace must be 16-byte aligned");
  BeamArgs a;
  a.x = logits_dev;
  a.row_stride = row_stride;
  a.batch = batch;
  a.vocab = vocab;
  a.beams = beams;
  a.k = k;
  const BeamPlan p = beam_plan(rows, vocab);
  a.parts = p.parts;
  a.slots = p.slots;
  a.scores = scores_dev;
  a.done = done_dev;
  a.end = end;
  a.out_y = out_scores_dev;
  a.out_i = out_beams_dev;
  a.out_v = out_tokens_dev;
  a.top = static_cast<uint64_t*>(ws_dev);
  a.sum = reinterpret_cast<double*>(a.top + rows * a.parts * k);
  a.max = reinterpret_cast<float*>(a.sum + rows * a.parts);
  const hipStream_t st = as_stream(stream);
  if (dtype == KH_DT_F32) beam_launch<float>(a, st);
  else beam_launch<uint16_t>(a, st);
  hipLaunchKernelGGL(beam_join_kernel, dim3((unsigned)std::min<int64_t>(batch, 1 << 20)), dim3(kBjThreads), 0, st, a);
  KH_LAUNCHED();
  return KH_OK;
}
