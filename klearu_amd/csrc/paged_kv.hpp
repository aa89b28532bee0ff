// paged_kv.hpp -- handles and the page layout shared by the rotary, paged-cache
// and paged-attention kernels.
//
// A page holds `ps` positions of every kv head.  One (page, kv head) is a block
// of contiguous bytes in four parts, laid out so that the attention kernels
// load matrix-core operands as they lie (g = 0..3 and r = 0..15 are a lane's
// row group and row, j a group of 32 values, D = head_dim):
//   K codes [ps][g][j] u32: nibble n is the code of d = 32 j + 8 g + n
//   V codes [ps / 4][r][token / 2 % 2][h][token % 2] u16, h < D / 64: nibble n
//           is the code of d = 64 h + 16 n + r
//   K pairs [ps][j] u32: minimum | scale << 16 (BF16 bits)
//   V pairs [j][ps] u32: the same
// Every part of a position is written by whole u16 or u32 stores of its own, so
// positions of one page may be appended from different blocks.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.hpp"

struct kh_rope {
  int rot = 0;           // rotated elements of a head, even
  int layout = 0;        // KH_ROPE_*
  int64_t max_pos = 0;
  int device = 0;
  float2* table = nullptr;  // [max_pos][rot / 2] (cos, sin), both times the magnitude
  int* err = nullptr;
  // several axes: pairs end[a - 1] .. end[a] - 1 turn by the row's position along axis a
  int axes = 1;
  int end[KH_ROPE_MAX_AXES] = {0, 0, 0, 0};
};

struct kh_paged_kv {
  int nkv = 0, d = 0, ps = 0, ps_log2 = 0;
  int64_t pages = 0;
  int64_t block = 0;  // bytes of one (page, kv head)
  int device = 0;
  char* pool = nullptr;
  int* err = nullptr;
};

namespace kh {

// The pairs' axes of a rotation, and where the positions along the others lie behind the first one's.
struct RopeAxes {
  int n;
  int end[KH_ROPE_MAX_AXES];  // of unused axes: the number of pairs
  int64_t stride;
  __device__ __forceinline__ int of(int pair) const {
    int a = 0;
#pragma unroll
    for (int i = 0; i + 1 < KH_ROPE_MAX_AXES; ++i) a += pair >= end[i] ? 1 : 0;
    return a;
  }
};
inline RopeAxes rope_axes(const kh_rope* r, int64_t stride) {
  RopeAxes x;
  x.n = r->axes;
  x.stride = stride;
  for (int i = 0; i < KH_ROPE_MAX_AXES; ++i) x.end[i] = i < r->axes ? r->end[i] : r->rot / 2;
  return x;
}
// Whether no section ends inside a piece of n pairs.
inline bool rope_axes_whole(const kh_rope* r, int n) {
  for (int i = 0; i < r->axes; ++i)
    if (r->end[i] % n) return false;
  return true;
}

constexpr int kKvGroup = 32;  // values that share a scale and a minimum

constexpr int64_t kv_block_bytes(int ps, int d) { return (int64_t)ps * d + (int64_t)ps * (d / kKvGroup) * 8; }

// Offsets of the parts of a block.
template <int D>
struct KvParts {
  static constexpr int NG = D / kKvGroup;
  static __host__ __device__ constexpr int kc() { return 0; }
  static __host__ __device__ constexpr int vc(int ps) { return ps * (D / 2); }
  static __host__ __device__ constexpr int kp(int ps) { return ps * D; }
  static __host__ __device__ constexpr int vp(int ps) { return ps * D + ps * NG * 4; }
};

// The handle's device must be the current one: its memory and the stream
// belong there.
inline int check_device(int device, const char* what) {
  int cur = 0;
  KH_HIP(hipGetDevice(&cur));
  KH_CHECK_ARG(cur == device, "%s lives on device %d, the current device is %d", what, device, cur);
  return KH_OK;
}
#define KH_ON_DEVICE(device, what)                           \
  do {                                                       \
    const int dev_rc_ = ::kh::check_device((device), (what)); \
    if (dev_rc_ != KH_OK) return dev_rc_;                    \
  } while (0)

// Threads that a grid may have along x: of more the launch keeps the lower 32 bits of
// their number, and reports nothing.
constexpr int64_t kGridThreads = ((int64_t)1 << 32) - 1;

// What the attention kernels of a head_dim need of the current device.
int paged_attn_prepare(int d);
int paged_weights_prepare(int d);

// Whether two ranges of n and m bytes have one in common.
inline bool ranges_meet(const void* a, int64_t n, const void* b, int64_t m) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x <= y ? y - x < (uint64_t)n : x - y < (uint64_t)m;
}

inline size_t dtype_bytes(int dtype) { return dtype == KH_DT_F32 ? 4 : 2; }

// Whether 16-byte accesses of whole 16-byte pieces are aligned: the base and
// every stride (in elements) that is used.
inline bool aligned16(const void* p, int dtype, int64_t s0, int64_t s1) {
  const int64_t e = (int64_t)dtype_bytes(dtype);
  return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(s0 * e) | (uintptr_t)(s1 * e)) & 15) == 0;
}

// Rows [n0][n1][width] with element strides (s0, s1, 1) that no two elements
// share (an output's requirement).
inline bool strides_disjoint(int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t width) {
  if (n0 <= 1 && n1 <= 1) return true;
  if (n0 <= 1) return s1 >= width;
  if (n1 <= 1) return s0 >= width;
  if (s1 <= s0) return s1 >= width && s0 >= (n1 - 1) * s1 + width;
  return s0 >= width && s1 >= (n0 - 1) * s0 + width;
}

__device__ __forceinline__ float load_f32(const float* p) { return *p; }
__device__ __forceinline__ float load_f32(const uint16_t* p) { return bf16_to_f32(*p); }
__device__ __forceinline__ void store_f32(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_f32(uint16_t* p, float v) { *p = f32_to_bf16(v); }

// Eight neighbouring elements; vec: p is 16-byte aligned.
__device__ __forceinline__ void load8(const uint16_t* p, bool vec, float (&f)[8]) {
  if (vec) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    f[0] = bf16_lo(v.x); f[1] = bf16_hi(v.x); f[2] = bf16_lo(v.y); f[3] = bf16_hi(v.y);
    f[4] = bf16_lo(v.z); f[5] = bf16_hi(v.z); f[6] = bf16_lo(v.w); f[7] = bf16_hi(v.w);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = bf16_to_f32(p[i]);
  }
}
__device__ __forceinline__ void load8(const float* p, bool vec, float (&f)[8]) {
  if (vec) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = p[i];
  }
}
__device__ __forceinline__ void store8(uint16_t* p, bool vec, const float (&f)[8]) {
  if (vec) {
    uint4 v;
    v.x = f32_to_bf16(f[0]) | (uint32_t)f32_to_bf16(f[1]) << 16;
    v.y = f32_to_bf16(f[2]) | (uint32_t)f32_to_bf16(f[3]) << 16;
    v.z = f32_to_bf16(f[4]) | (uint32_t)f32_to_bf16(f[5]) << 16;
    v.w = f32_to_bf16(f[6]) | (uint32_t)f32_to_bf16(f[7]) << 16;
    *reinterpret_cast<uint4*>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = f32_to_bf16(f[i]);
  }
}
__device__ __forceinline__ void store8(float* p, bool vec, const float (&f)[8]) {
  if (vec) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = f[i];
  }
}

}  // namespace kh
