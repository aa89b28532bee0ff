// paged_frag.hpp -- what the kernels that read a paged cache's codes through the matrix cores share:
// wide loads, codes and f32 numbers as BF16 terms, exchanges between the lane groups of a column.
#pragma once

#include "mfma.hpp"
#include "paged_kv.hpp"

namespace kh {

constexpr float kLog2e = 1.44269504088896340736f;

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
  // Zeros unless on.
  __device__ __forceinline__ void keep(bool on) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = make_uint4(on ? w[i].x : 0, on ? w[i].y : 0, on ? w[i].z : 0, on ? w[i].w : 0);
  }
  // The largest absolute value, as an f32's bits.
  __device__ __forceinline__ uint32_t largest() const {
    if constexpr (sizeof(T) == 4) {
      const auto m = [](const uint4& v) {
        return max(max(v.x & 0x7fffffffu, v.y & 0x7fffffffu), max(v.z & 0x7fffffffu, v.w & 0x7fffffffu));
      };
      return max(m(w[0]), m(w[1]));
    } else {
      typedef unsigned short pair __attribute__((ext_vector_type(2)));
      const auto p = [](uint32_t u) { return __builtin_bit_cast(pair, u & 0x7fff7fffu); };
      const pair m = __builtin_elementwise_max(__builtin_elementwise_max(p(w[0].x), p(w[0].y)), __builtin_elementwise_max(p(w[0].z), p(w[0].w)));
      return (uint32_t)max(m.x, m.y) << 16;
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

__device__ __forceinline__ uint32_t across_groups_max_u32(uint32_t u) {
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t w = max(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return max(b[0], b[1]);
}

__device__ __forceinline__ uint32_t across_groups_or(uint32_t u) {
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t w = a[0] | a[1];
  const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return b[0] | b[1];
}

typedef _Float16 kh_f16x2 __attribute__((ext_vector_type(2)));

// Nibble n of each half of w as 16 + c, a pair of f16: six bits up it counts ones
// behind the bits of 16.
__device__ __forceinline__ kh_f16x2 codes_f16(uint32_t w, int n) {
  const uint32_t x = n == 0 ? w << 6 : n == 1 ? w << 2 : n == 2 ? w >> 2 : w >> 6;
  return __builtin_bit_cast(kh_f16x2, (x & 0x03c003c0u) | 0x4c004c00u);
}

}  // namespace kh
