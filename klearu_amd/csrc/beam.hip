// beam.hip -- the best continuations of beams over a vocabulary (gfx950).
//
//   y[i][v] = scores[i] + x[i][v] - log sum_w exp(x[i][w]),   top k of y over (i, v)
//
// One pass over the logits: a block takes a chunk of a row, and leaves its maximum M, the sum of
// exp(x - M) and its k largest logits; a second kernel joins a sequence's chunks.  Within a beam y orders
// as x does, so chunks compare logits as integers.  Between beams the log-sum-exps decide: they are f64,
// of f32 exponentials with the rounding of their arguments put back (log2 e in two
// parts), since sums that are 1e-7 off swap continuations of a batch of beams now and then.
//
// The k largest of a chunk: the k-th largest T of the threads' own maxima has k logits at
// or above it, so the k largest are among those, few, which are ranked by counting.
#include <algorithm>

#include "paged_kv.hpp"

namespace kh {

constexpr int kBmThreads = 256;
constexpr int kBmEach = 16;                       // logits of a thread
constexpr int kBmChunk = kBmThreads * kBmEach;
constexpr int kBmList = 512;                      // of a chunk, that are ranked by counting

struct BeamArgs {
  const void* x;
  int64_t row_stride, batch, vocab;
  int beams, k, chunks;
  const float* scores;
  const uint8_t* done;
  int64_t end;
  float* out_y;
  int32_t *out_i, *out_v;
  uint64_t* top;  // [rows][chunks][k] f32_key << 32 | ~token, descending; 0: none
  double* sum;    // [rows][chunks]
  float* max;
};

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m);
  return v;
}
__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) {
    const uint64_t o = __shfl_xor((unsigned long long)v, m);
    v = o > v ? o : v;
  }
  return v;
}

// exp(t), t <= 0, within 1e-7 and without a bias: log2 e is 0x1.715476p+0f and 1.9e-8 more.
__device__ __forceinline__ float beam_exp(float t) {
  const float hi = 0x1.715476p+0f, lo = 0x1.4ae0cp-26f;
  const float y = t * hi, r = fmaf(t, hi, -y) + t * lo;
  const float e = __builtin_amdgcn_exp2f(y);
  return y < -126.0f ? 0.0f : fmaf(e, r * 0x1.62e43p-1f, e);
}

// Elements i0 .. i0 + N - 1 of a row that starts `shift` elements behind a 16-byte
// border, counted from that border: a vector load where all of them are the row's.
template <typename T, int N>
__device__ __forceinline__ void beam_load(const T* row, int shift, int64_t n, int64_t i0, float (&f)[N]) {
  const int64_t v0 = i0 - shift;
  if (v0 >= 0 && v0 + N <= n) {
    const uint4 w = *reinterpret_cast<const uint4*>(row + v0);
    if constexpr (sizeof(T) == 4) {
      f[0] = __uint_as_float(w.x); f[1] = __uint_as_float(w.y); f[2] = __uint_as_float(w.z); f[3] = __uint_as_float(w.w);
    } else {
      f[0] = bf16_lo(w.x); f[1] = bf16_hi(w.x); f[2] = bf16_lo(w.y); f[3] = bf16_hi(w.y);
      f[4] = bf16_lo(w.z); f[5] = bf16_hi(w.z); f[6] = bf16_lo(w.w); f[7] = bf16_hi(w.w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = v0 + i >= 0 && v0 + i < n ? load_f32(row + v0 + i) : -INFINITY;
  }
}

template <typename T>
__global__ __launch_bounds__(kBmThreads) void beam_chunk_kernel(BeamArgs a) {
  constexpr int V = 16 / sizeof(T), W = kBmThreads / 64;
  __shared__ __align__(16) uint32_t s_max[kBmThreads];
  __shared__ uint64_t s_list[kBmList], s_best[W];
  __shared__ float s_m[W];
  __shared__ double s_sum[W];
  __shared__ uint32_t s_t;
  __shared__ int s_n;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  for (int64_t id = blockIdx.x; id < a.batch * a.beams * a.chunks; id += gridDim.x) {
    const int64_t r = id / a.chunks, c0 = (id - r * a.chunks) * kBmChunk;
    const T* row = static_cast<const T*>(a.x) + r * a.row_stride;
    const int shift = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    float x[kBmEach];
    // element e of thread t: (e / V * 256 + t) V + e % V of the chunk
#pragma unroll
    for (int q = 0; q < kBmEach / V; ++q) {
      float f[V];
      beam_load<T, V>(row, shift, a.vocab, c0 + (q * kBmThreads + t) * V, f);
#pragma unroll
      for (int i = 0; i < V; ++i) x[q * V + i] = f[i];
    }
    const auto token = [&](int e) { return (uint32_t)(c0 + ((e / V) * kBmThreads + t) * V + e % V - shift); };
    const auto there = [&](int e) { return token(e) < (uint32_t)a.vocab; };
    float m = x[0];
#pragma unroll
    for (int e = 1; e < kBmEach; ++e) m = fmaxf(m, x[e]);
    // a thread of nothing but NaN has no maximum: its NaN go into the sum
    uint32_t key = 0;
#pragma unroll
    for (int e = 0; e < kBmEach; ++e)
      if (there(e)) key = max(key, f32_key(x[e]));
    s_max[t] = key;
    m = wave_max(m);
    if (lane == 0) s_m[wave] = m;
    if (t == 0) s_n = 0, s_t = 1;
    __syncthreads();
    m = s_m[0];
#pragma unroll
    for (int w = 1; w < W; ++w) m = fmaxf(m, s_m[w]);
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < kBmEach; ++e) s += x[e] == -INFINITY ? 0.0f : beam_exp(x[e] - m);
    const double d = wave_sum_f64((double)s);
    if (lane == 0) s_sum[wave] = d;
    // the rank of the thread's maximum
    int rank = 0;
    for (int i = 0; i < kBmThreads; i += 4) {
      const uint4 o = *reinterpret_cast<const uint4*>(&s_max[i]);
      rank += (o.x > key || (o.x == key && i < t)) + (o.y > key || (o.y == key && i + 1 < t)) +
              (o.z > key || (o.z == key && i + 2 < t)) + (o.w > key || (o.w == key && i + 3 < t));
    }
    if (rank == a.k - 1 && key > 0) s_t = key;
    __syncthreads();
    if (t == 0) {
      a.max[id] = m;
      a.sum[id] = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
    }
    const uint32_t T0 = s_t;
    int n = 0;
#pragma unroll
    for (int e = 0; e < kBmEach; ++e) n += there(e) && f32_key(x[e]) >= T0 ? 1 : 0;
    if (n) {
      int at = atomicAdd(&s_n, n);
#pragma unroll
      for (int e = 0; e < kBmEach; ++e)
        if (there(e) && f32_key(x[e]) >= T0) {
          if (at < kBmList) s_list[at] = (uint64_t)f32_key(x[e]) << 32 | ~token(e);
          ++at;
        }
    }
    __syncthreads();
    n = s_n;
    uint64_t* top = a.top + id * a.k;
    if (n <= kBmList) {
      for (int i = t; i < n; i += kBmThreads) {
        const uint64_t me = s_list[i];
        int above = 0;
        for (int j = 0; j < n; ++j) above += s_list[j] > me ? 1 : 0;
        if (above < a.k) top[above] = me;
      }
      if (t >= n && t < a.k) top[t] = 0;
    } else {  // many equal logits: the largest, time after time
      uint64_t last = ~0ull;
      for (int i = 0; i < a.k; ++i) {
        uint64_t best = 0;
#pragma unroll
        for (int e = 0; e < kBmEach; ++e) {
          const uint64_t y = (uint64_t)f32_key(x[e]) << 32 | ~token(e);
          if (there(e) && y < last && y > best) best = y;
        }
        best = wave_max_u64(best);
        __syncthreads();
        if (lane == 0) s_best[wave] = best;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) best = s_best[w] > best ? s_best[w] : best;
        last = best;
        if (t == 0) top[i] = best;
      }
    }
    __syncthreads();
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

constexpr int kBjThreads = 256, kBjList = 1024;

// Block: a sequence.
__global__ __launch_bounds__(kBjThreads) void beam_join_kernel(BeamArgs a) {
  constexpr int W = kBjThreads / 64;
  __shared__ double s_score[KH_MAX_BEAMS], s_top[KH_MAX_BEAMS], s_log[KH_MAX_BEAMS];  // and the log-sum-exp's parts
  __shared__ int s_kind[KH_MAX_BEAMS];  // 0: its chunks' logits, 1: none, 2: at its end
  __shared__ __align__(16) uint64_t s_max[kBjThreads];
  __shared__ uint64_t s_key[kBjList], s_flat[kBjList], s_bk[W], s_bf[W], s_t;
  __shared__ int s_n;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  for (int64_t b = blockIdx.x; b < a.batch; b += gridDim.x) {
    for (int i = wave; i < a.beams; i += W) {
      const int64_t r = b * a.beams + i, at = r * a.chunks;
      float m = -INFINITY;
      for (int c = lane; c < a.chunks; c += 64) m = fmaxf(m, a.max[at + c]);
      m = wave_max(m);
      double s = 0.0;
      for (int c = lane; c < a.chunks; c += 64) {
        const float mc = a.max[at + c];
        s += mc == -INFINITY ? a.sum[at + c] : a.sum[at + c] * exp((double)mc - (double)m);
      }
      s = wave_sum_f64(s);
      if (lane == 0) {
        const double score = (double)a.scores[r], l = log(s);
        const bool fine = __builtin_isfinite(score), has = __builtin_isfinite(m) && __builtin_isfinite(l);
        s_kind[i] = !fine ? 1 : a.done && a.done[r] ? 2 : has ? 0 : 1;
        s_score[i] = score;
        s_top[i] = (double)m;
        s_log[i] = l;
      }
    }
    if (t == 0) s_n = 0, s_t = 0;
    __syncthreads();
    const int each = a.chunks * a.k, all = a.beams * each;
    // continuation j: its key and its place among all; false: there is none
    const auto get = [&](int j, uint64_t& key, uint64_t& flat) {
      const int i = j / each, e = j - i * each;
      const uint64_t base = (uint64_t)i * (uint64_t)a.vocab;
      const int kind = s_kind[i];
      if (kind == 0) {
        const uint64_t w = a.top[((b * a.beams + i) * a.chunks) * a.k + e];
        const uint32_t k32 = (uint32_t)(w >> 32);
        const double x = (double)__uint_as_float(k32 >> 31 ? k32 & 0x7fffffffu : ~k32);
        key = f64_key(s_score[i] + ((x - s_top[i]) - s_log[i]));  // logits of any size leave the score its bits
        flat = base + (uint32_t)~(uint32_t)w;
        return w != 0;
      }
      // the first tokens, all of them -inf, but for the end
      key = f64_key(-INFINITY);
      int64_t v = e;
      if (kind == 2) {
        if (e == 0) key = f64_key(s_score[i]), v = a.end;
        else if (e <= a.end) v = e - 1;
      }
      flat = base + (uint64_t)v;
      return e < a.k && e < a.vocab;
    };
    uint64_t mine = 0;
    for (int j = t; j < all; j += kBjThreads) {
      uint64_t key, flat;
      if (get(j, key, flat) && key > mine) mine = key;
    }
    s_max[t] = mine;
    __syncthreads();
    int rank = 0;
    for (int i = 0; i < kBjThreads; ++i) rank += s_max[i] > mine || (s_max[i] == mine && i < t) ? 1 : 0;
    if (rank == a.k - 1) s_t = mine;
    __syncthreads();
    const uint64_t T = s_t;
    for (int j = t; j < all; j += kBjThreads) {
      uint64_t key, flat;
      if (get(j, key, flat) && key >= T) {
        const int at = atomicAdd(&s_n, 1);
        if (at < kBjList) s_key[at] = key, s_flat[at] = flat;
      }
    }
    __syncthreads();
    const int n = s_n;
    const auto put = [&](int at, uint64_t key, uint64_t flat) {
      a.out_y[b * a.k + at] = (float)key_f64(key);
      a.out_i[b * a.k + at] = (int32_t)(flat / (uint64_t)a.vocab);
      a.out_v[b * a.k + at] = (int32_t)(flat % (uint64_t)a.vocab);
    };
    if (n <= kBjList) {
      for (int i = t; i < n; i += kBjThreads) {
        const uint64_t key = s_key[i], flat = s_flat[i];
        int above = 0;
        for (int j = 0; j < n; ++j) above += s_key[j] > key || (s_key[j] == key && s_flat[j] < flat) ? 1 : 0;
        if (above < a.k) put(above, key, flat);
      }
    } else {
      uint64_t lk = ~0ull, lf = 0;  // the last one written
      for (int i = 0; i < a.k; ++i) {
        uint64_t bk = 0, bf = ~0ull;
        for (int j = t; j < all; j += kBjThreads) {
          uint64_t key, flat;
          if (get(j, key, flat) && (key < lk || (key == lk && flat > lf)) && (key > bk || (key == bk && flat < bf)))
            bk = key, bf = flat;
        }
#pragma unroll
        for (int m = 32; m > 0; m >>= 1) {
          const uint64_t ok = __shfl_xor((unsigned long long)bk, m), of = __shfl_xor((unsigned long long)bf, m);
          if (ok > bk || (ok == bk && of < bf)) bk = ok, bf = of;
        }
        __syncthreads();
        if (lane == 0) s_bk[wave] = bk, s_bf[wave] = bf;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w)
          if (s_bk[w] > bk || (s_bk[w] == bk && s_bf[w] < bf)) bk = s_bk[w], bf = s_bf[w];
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
// Chunks of a row, wherever it starts between two 16-byte borders.
static int beam_chunks(int64_t vocab) { return ceil_div(vocab + 7, kBmChunk); }
static int64_t beam_space(int64_t batch, int beams, int64_t vocab, int k) {
  return batch * beams * beam_chunks(vocab) * (8 * (int64_t)k + 8 + 4);
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
  a.chunks = beam_chunks(vocab);
  a.scores = scores_dev;
  a.done = done_dev;
  a.end = end;
  a.out_y = out_scores_dev;
  a.out_i = out_beams_dev;
  a.out_v = out_tokens_dev;
  a.top = static_cast<uint64_t*>(ws_dev);
  a.sum = reinterpret_cast<double*>(a.top + rows * a.chunks * k);
  a.max = reinterpret_cast<float*>(a.sum + rows * a.chunks);
  const hipStream_t st = as_stream(stream);
  const dim3 g((unsigned)std::min<int64_t>(rows * a.chunks, 1 << 20));
  if (dtype == KH_DT_F32) hipLaunchKernelGGL(beam_chunk_kernel<float>, g, dim3(kBmThreads), 0, st, a);
  else hipLaunchKernelGGL(beam_chunk_kernel<uint16_t>, g, dim3(kBmThreads), 0, st, a);
  hipLaunchKernelGGL(beam_join_kernel, dim3((unsigned)std::min<int64_t>(batch, 1 << 20)), dim3(kBjThreads), 0, st, a);
  KH_LAUNCHED();
  return KH_OK;
}
