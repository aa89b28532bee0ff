// rope.hip -- rotary positions by themselves (gfx950).
//
// For a row at position p and the rotated pair i of a head (x0, x1):
//   y0 = x0 c - x1 s,  y1 = x1 c + x0 s,   c = a cos(p f_i), s = a sin(p f_i)
// and the transposed rotation (the gradient with respect to x) has -s for s.
// Frequencies f_i = theta^(-2i/r), i < r/2, stretched for long contexts as the
// handle says.  The angles are computed once, in f64 (p f_i reaches 1e5 and more,
// where f32 holds 1e-2 of a turn), and kept as an f32 table.
//
// The kernel moves x through registers once, 16 bytes a lane and access, both halves
// of a pair in one thread: bounded by memory for many rows (8191 BF16 rows of 32 heads of
// 128, 138 MB with the table: 24.7 us, 5.6 TB/s, a copy of 4 GiB runs at 4.8; 2049 f32 rows
// of 32 heads of 64, interleaved, half of a head rotated: 7.5 us) and by the launch for one
// (2.4 us of kernel, 6.8 us a call).
#include <algorithm>
#include <cmath>
#include <new>

#include "paged_kv.hpp"

namespace kh {

constexpr int64_t kMostBlocks = kGridThreads / 256;  // larger work is launched in parts

// Entries first and later of the table of n.
__global__ void rope_table_kernel(const double* __restrict__ freq, int half, int64_t first, int64_t n, double mag,
                                  float2* __restrict__ table) {
  const int64_t i = first + (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const double a = (double)(i / half) * freq[i % half];
  double s, c;
  sincos(a, &s, &c);
  table[i] = make_float2((float)(c * mag), (float)(s * mag));
}

struct RopeArgs {
  const void* x;
  void* y;
  const int64_t* pos;
  const float2* table;
  int* err;
  int64_t rows, xs, xh, ys, yh, max_pos;
  int heads, dim, rot;
  float sgn;  // of the sine: -1 for the transposed rotation
  int copy;   // the elements past rot are copied (y is not x)
  RopeAxes ax;
};

// The row's table entries, or nullptr for a row that is skipped: negative
// positions are padding, positions past the table are recorded.
__device__ __forceinline__ const float2* rope_row(const RopeArgs& a, int64_t t) {
  const int64_t p = a.pos[t];
  if (p < 0) return nullptr;
  if (p >= a.max_pos) {
    atomicOr(a.err, 1);
    return nullptr;
  }
  return a.table + p * (a.rot >> 1);
}

// Several axes: whether the row is rotated (any negative position makes it padding), and its positions.
__device__ __forceinline__ bool rope_row_axes(const RopeArgs& a, int64_t t, int64_t (&p)[KH_ROPE_MAX_AXES]) {
  bool pad = false, past = false;
#pragma unroll
  for (int i = 0; i < KH_ROPE_MAX_AXES; ++i) {
    p[i] = i < a.ax.n ? a.pos[i * a.ax.stride + t] : 0;
    pad = pad || p[i] < 0;
    past = past || p[i] >= a.max_pos;
  }
  if (!pad && past) atomicOr(a.err, 1);
  return !pad && !past;
}
// The table's row that pair i of the row reads.
__device__ __forceinline__ const float2* rope_axis(const RopeArgs& a, const int64_t (&p)[KH_ROPE_MAX_AXES], int i) {
  const int x = a.ax.of(i);
  const int64_t r = x == 0 ? p[0] : x == 1 ? p[1] : x == 2 ? p[2] : p[3];
  return a.table + r * (a.rot >> 1);
}

__device__ __forceinline__ void rope_pair(float& x0, float& x1, float c, float s) {
  const float y0 = x0 * c - x1 * s, y1 = x1 * c + x0 * s;
  x0 = y0;
  x1 = y1;
}

// One thread: one piece of eight pairs (or eight elements of four pairs, or
// eight elements past rot) of one head of one row.  AXES: several of them; a piece
// that two sections share looks its rows up pair by pair.
template <typename T, bool HALF, bool AXES>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a, int pieces) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t per_row = (int64_t)pieces * a.heads;
  const int64_t t = id / per_row;
  if (t >= a.rows) return;
  const float2* __restrict__ tab = nullptr;
  int64_t p[KH_ROPE_MAX_AXES];
  if (AXES) {
    if (!rope_row_axes(a, t, p)) return;
  } else {
    tab = rope_row(a, t);
    if (!tab) return;
  }
  const auto pair = [&](int i) -> float2 {
    if (!AXES) return tab[i];
    return rope_axis(a, p, i)[i];
  };
  const int rem = (int)(id - t * per_row), h = rem / pieces, u = rem - h * pieces;
  const T* x = static_cast<const T*>(a.x) + t * a.xs + h * a.xh;
  T* y = static_cast<T*>(a.y) + t * a.ys + h * a.yh;
  const int half = a.rot >> 1;
  float v[8], w[8];
  if (HALF) {
    const int np = half / 8;
    if (u < np) {
      load8(x + 8 * u, true, v);
      load8(x + half + 8 * u, true, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 cs = pair(8 * u + i);
        rope_pair(v[i], w[i], cs.x, a.sgn * cs.y);
      }
      store8(y + 8 * u, true, v);
      store8(y + half + 8 * u, true, w);
      return;
    }
    const int d = a.rot + 8 * (u - np);
    load8(x + d, true, v);
    store8(y + d, true, v);
  } else {
    const int d = 8 * u;
    load8(x + d, true, v);
    if (d < a.rot) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 cs = pair(4 * u + i);
        rope_pair(v[2 * i], v[2 * i + 1], cs.x, a.sgn * cs.y);
      }
    }
    store8(y + d, true, v);
  }
}

// Any alignment and any even rot: one thread per pair, then one per copied
// element.
template <typename T, bool AXES>
__global__ __launch_bounds__(256) void rope_any_kernel(RopeArgs a, int half_layout, int units) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t per_row = (int64_t)units * a.heads;
  const int64_t t = id / per_row;
  if (t >= a.rows) return;
  const float2* __restrict__ tab = nullptr;
  int64_t p[KH_ROPE_MAX_AXES];
  if (AXES) {
    if (!rope_row_axes(a, t, p)) return;
  } else {
    tab = rope_row(a, t);
    if (!tab) return;
  }
  const int rem = (int)(id - t * per_row), h = rem / units, u = rem - h * units;
  const T* x = static_cast<const T*>(a.x) + t * a.xs + h * a.xh;
  T* y = static_cast<T*>(a.y) + t * a.ys + h * a.yh;
  const int half = a.rot >> 1;
  if (u < half) {
    const int i0 = half_layout ? u : 2 * u, i1 = half_layout ? u + half : 2 * u + 1;
    float v = load_f32(x + i0), w = load_f32(x + i1);
    const float2 cs = AXES ? rope_axis(a, p, u)[u] : tab[u];
    rope_pair(v, w, cs.x, a.sgn * cs.y);
    store_f32(y + i0, v);
    store_f32(y + i1, w);
  } else {
    const int d = a.rot + (u - half);
    y[d] = x[d];
  }
}

template <typename T, bool AXES>
static int rope_launch(const RopeArgs& all, int layout, bool vec, hipStream_t st) {
  const int pieces = !vec ? all.rot / 2 + (all.copy ? all.dim - all.rot : 0)
                     : layout == KH_ROPE_HALF ? all.rot / 16 + (all.copy ? (all.dim - all.rot) / 8 : 0)
                                              : (all.copy ? all.dim : all.rot) / 8;
  // rows of a launch; one row is below 2^32 threads (65536 heads of fewer than 65536 pieces)
  const int64_t most = kMostBlocks * 256 / ((int64_t)all.heads * pieces);
  for (int64_t t0 = 0; t0 < all.rows; t0 += most) {
    RopeArgs a = all;
    a.rows = all.rows - t0 < most ? all.rows - t0 : most;
    a.x = static_cast<const T*>(all.x) + t0 * all.xs;
    a.y = static_cast<T*>(all.y) + t0 * all.ys;
    a.pos = all.pos + t0;
    const unsigned blocks = (unsigned)((a.rows * a.heads * pieces + 255) / 256);
    if (!vec)
      hipLaunchKernelGGL((rope_any_kernel<T, AXES>), dim3(blocks), dim3(256), 0, st, a, layout == KH_ROPE_HALF ? 1 : 0, pieces);
    else if (layout == KH_ROPE_HALF)
      hipLaunchKernelGGL((rope_kernel<T, true, AXES>), dim3(blocks), dim3(256), 0, st, a, pieces);
    else
      hipLaunchKernelGGL((rope_kernel<T, false, AXES>), dim3(blocks), dim3(256), 0, st, a, pieces);
    KH_LAUNCHED();
  }
  return KH_OK;
}

}  // namespace kh

using namespace kh;

extern "C" int kh_rope_destroy(kh_rope* r) {
  if (!r) return KH_OK;
  dev_free(r->table);
  dev_free(r->err);
  delete r;
  return KH_OK;
}

extern "C" int kh_rope_create(int rot_dim, int64_t max_pos, int layout, double theta, int scaling, double factor,
                              int64_t original_len, double low, double high, double magnitude, kh_rope** out) {
  const int all = rot_dim / 2;
  return kh_rope_create_axes(rot_dim, max_pos, layout, theta, scaling, factor, original_len, low, high, magnitude, 1,
                             &all, 0, out);
}

extern "C" int kh_rope_create_axes(int rot_dim, int64_t max_pos, int layout, double theta, int scaling, double factor,
                                   int64_t original_len, double low, double high, double magnitude, int axes,
                                   const int32_t* sections_host, int restart, kh_rope** out) {
  KH_CHECK_ARG(out != nullptr, "null output");
  *out = nullptr;
  KH_CHECK_ARG(rot_dim >= 2 && rot_dim <= 1024 && rot_dim % 2 == 0, "rot_dim %d not an even number in [2,1024]",
               rot_dim);
  KH_CHECK_ARG(max_pos >= 1 && max_pos <= ((int64_t)1 << 31), "max_pos %lld not in [1,2^31]", (long long)max_pos);
  KH_CHECK_ARG(layout == KH_ROPE_HALF || layout == KH_ROPE_INTERLEAVED, "unknown layout %d", layout);
  KH_CHECK_ARG(std::isfinite(theta) && theta > 0, "theta must be positive and finite");
  KH_CHECK_ARG(scaling >= KH_ROPE_SCALE_NONE && scaling <= KH_ROPE_SCALE_BY_PARTS, "unknown scaling %d", scaling);
  KH_CHECK_ARG(std::isfinite(magnitude) && magnitude > 0, "magnitude must be positive and finite");
  if (scaling != KH_ROPE_SCALE_NONE)
    KH_CHECK_ARG(std::isfinite(factor) && factor > 0, "factor must be positive and finite");
  KH_CHECK_ARG(scaling != KH_ROPE_SCALE_BASE || rot_dim > 2, "a changed base needs rot_dim > 2");
  if (scaling == KH_ROPE_SCALE_BY_PARTS)
    KH_CHECK_ARG(original_len >= 1 && std::isfinite(low) && std::isfinite(high) && high > low,
                 "scaling by parts needs original_len >= 1 and low < high");
  KH_CHECK_ARG(axes >= 1 && axes <= KH_ROPE_MAX_AXES, "%d axes: 1 to %d are supported", axes, KH_ROPE_MAX_AXES);
  KH_CHECK_ARG(sections_host != nullptr, "null sections");
  const int half = rot_dim / 2;
  int64_t pairs = 0;
  for (int x = 0; x < axes; ++x) {
    KH_CHECK_ARG(sections_host[x] >= 1, "section %d has %d pairs", x, sections_host[x]);
    KH_CHECK_ARG(!restart || scaling != KH_ROPE_SCALE_BASE || sections_host[x] > 1,
                 "a changed base needs sections of more than one pair");
    pairs += sections_host[x];
  }
  KH_CHECK_ARG(pairs == half, "the sections have %lld pairs, rot_dim %d", (long long)pairs, rot_dim);
  double freq[512];
  int first = 0, axis = 0;  // of the section whose frequencies pair i's are: its first pair, its axis
  for (int i = 0; i < half; ++i) {
    if (restart && i == first + sections_host[axis]) first = i, ++axis;
    const int r = restart ? 2 * sections_host[axis] : rot_dim;
    const double base = scaling == KH_ROPE_SCALE_BASE ? theta * std::pow(factor, (double)r / (r - 2)) : theta;
    double f = std::pow(base, -2.0 * (i - first) / r);
    if (scaling == KH_ROPE_SCALE_LINEAR) f /= factor;
    if (scaling == KH_ROPE_SCALE_BY_PARTS) {
      const double turns = f * (double)original_len / (2.0 * 3.14159265358979323846);
      double keep = (turns - low) / (high - low);
      keep = keep < 0 ? 0 : keep > 1 ? 1 : keep;
      f = f * (keep + (1 - keep) / factor);
    }
    freq[i] = f;
  }
  kh_rope* r = new (std::nothrow) kh_rope;
  if (!r) {
    set_error("out of host memory");
    return KH_ERR_ALLOC;
  }
  r->rot = rot_dim;
  r->layout = layout;
  r->max_pos = max_pos;
  r->axes = axes;
  for (int x = 0, n = 0; x < axes; ++x) r->end[x] = n += sections_host[x];
  double* freq_dev = nullptr;
  int rc = KH_OK;
  const int64_t n = max_pos * half;
  const auto fill = [&]() -> int {
    KH_HIP(hipGetDevice(&r->device));
    r->table = static_cast<float2*>(dev_alloc(sizeof(float2) * (size_t)n));
    r->err = static_cast<int*>(dev_alloc(sizeof(int)));
    freq_dev = static_cast<double*>(dev_alloc(sizeof(double) * half));
    if (!r->table || !r->err || !freq_dev) return KH_ERR_ALLOC;
    KH_HIP(hipMemset(r->err, 0, sizeof(int)));
    KH_HIP(hipMemcpy(freq_dev, freq, sizeof(double) * half, hipMemcpyHostToDevice));
    for (int64_t i = 0; i < n; i += kMostBlocks * 256) {
      const int64_t blocks = std::min((n - i + 255) / 256, kMostBlocks);
      hipLaunchKernelGGL(rope_table_kernel, dim3((unsigned)blocks), dim3(256), 0, nullptr, freq_dev, half, i, n,
                         magnitude, r->table);
      KH_LAUNCHED();
    }
    KH_HIP(hipStreamSynchronize(nullptr));
    return KH_OK;
  };
  rc = fill();
  dev_free(freq_dev);
  if (rc != KH_OK) {
    kh_rope_destroy(r);
    return rc;
  }
  *out = r;
  return KH_OK;
}

extern "C" int kh_rope_status(const kh_rope* r) {
  KH_CHECK_ARG(r != nullptr, "null handle");
  KH_ON_DEVICE(r->device, "the rotation");
  KH_HIP(hipDeviceSynchronize());
  int bad = 0;
  KH_HIP(hipMemcpy(&bad, r->err, sizeof(int), hipMemcpyDeviceToHost));
  if (!bad) return KH_OK;
  KH_HIP(hipMemset(r->err, 0, sizeof(int)));
  // cleared before any other stream records again: streams need not wait for the null stream
  KH_HIP(hipStreamSynchronize(nullptr));
  set_error("a row's position was not below max_pos %lld", (long long)r->max_pos);
  return KH_ERR_ARG;
}

extern "C" int kh_rope_apply(const kh_rope* r, int dtype, const void* x_dev, int64_t x_row_stride,
                             int64_t x_head_stride, int64_t rows, int heads, int head_dim, const int64_t* pos_dev,
                             void* y_dev, int64_t y_row_stride, int64_t y_head_stride, int transpose,
                             void* stream) {
  KH_CHECK_ARG(r != nullptr, "null handle");
  KH_CHECK_ARG(dtype == KH_DT_F32 || dtype == KH_DT_BF16, "dtype %d: f32 and BF16 are supported", dtype);
  KH_CHECK_ARG(rows >= 0 && rows < (int64_t)1 << 31 && heads >= 1 && heads <= 65536, "rows %lld, heads %d",
               (long long)rows, heads);
  KH_CHECK_ARG(head_dim >= r->rot && head_dim <= 65536, "head_dim %d not in [%d,65536]", head_dim, r->rot);
  if (rows == 0) return KH_OK;
  KH_CHECK_ARG(x_dev && y_dev && pos_dev, "null argument");
  KH_CHECK_ARG(x_row_stride >= 0 && x_head_stride >= 0, "negative stride");
  KH_CHECK_ARG(strides_disjoint(rows, y_row_stride, heads, y_head_stride, head_dim),
               "output strides (%lld, %lld) let heads overlap", (long long)y_row_stride, (long long)y_head_stride);
  const bool in_place = x_dev == y_dev;
  KH_CHECK_ARG(!in_place || (x_row_stride == y_row_stride && x_head_stride == y_head_stride),
               "a rotation in place needs the same strides on both sides");
  KH_ON_DEVICE(r->device, "the rotation");
  RopeArgs a;
  a.x = x_dev;
  a.y = y_dev;
  a.pos = pos_dev;
  a.table = r->table;
  a.err = r->err;
  a.rows = rows;
  a.xs = x_row_stride;
  a.xh = x_head_stride;
  a.ys = y_row_stride;
  a.yh = y_head_stride;
  a.max_pos = r->max_pos;
  a.heads = heads;
  a.dim = head_dim;
  a.rot = r->rot;
  a.sgn = transpose ? -1.0f : 1.0f;
  a.copy = in_place ? 0 : 1;
  a.ax = rope_axes(r, rows);
  const bool vec = aligned16(x_dev, dtype, x_row_stride, x_head_stride) &&
                   aligned16(y_dev, dtype, y_row_stride, y_head_stride) && head_dim % 8 == 0 &&
                   r->rot % (r->layout == KH_ROPE_HALF ? 16 : 8) == 0;
  const hipStream_t st = as_stream(stream);
  if (r->axes > 1)
    return dtype == KH_DT_F32 ? rope_launch<float, true>(a, r->layout, vec, st) : rope_launch<uint16_t, true>(a, r->layout, vec, st);
  return dtype == KH_DT_F32 ? rope_launch<float, false>(a, r->layout, vec, st) : rope_launch<uint16_t, false>(a, r->layout, vec, st);
}
