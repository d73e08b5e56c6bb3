// emmy_rotate_append.cu -- rotary positions on new queries and keys, keys and
// values into a paged cache, in one launch.
//
// A pair (x, y) of a head turns by the angle a = position * frequency:
// (x cos a - y sin a, y cos a + x sin a).  Every head of a token turns by the
// same angles, so a CTA takes one token, computes its cosines and sines once
// into shared memory and then moves the token's heads: each element is read
// once and written once, which is the floor of the operator.
//
// The angle is formed in 64 bits as a count of half turns and reduced there:
// at position 2^17 a 32-bit product is already off by 0.008 radians, and the
// reduction of a large 32-bit angle would cost a slow path besides.  Rotation
// is in 32 bits; the one rounding is to the cache's or q_out's type.
#include "../../include/emmy_b200.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <cstdio>

int emmy_internal_fail(int code, const char *msg);   // emmy_runtime.cpp

namespace {

constexpr int kThreads = 256;

struct Params {
  emmy_rotate_append_args a;
  int q_tasks, k_tasks, v_tasks;   // per head
};

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f(float x) { return x; }
template <> __device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f(float x) { return x; }
template <> __device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }

// N elements moved as one access where N * sizeof(T) is 16, else one by one
template <typename T, int N> struct alignas(N * sizeof(T)) Vec { T e[N]; };

// One task of a rotated head: with split pairs, vector i of the first half and
// its partner in the second, then the vectors that do not turn; with
// interleaved pairs, vector i (a scalar task, N = 1, takes a whole pair).
template <typename T, int N>
__device__ __forceinline__ void rotate_task(const T *src, T *dst, int task, int half, bool interleaved,
                                            const float2 *turn) {
  using V = Vec<T, N>;
  if (!interleaved) {
    const int pair_tasks = half / N;
    if (task < pair_tasks) {
      const int i = task * N;
      V x = *reinterpret_cast<const V *>(src + i), y = *reinterpret_cast<const V *>(src + half + i);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float2 cs = turn[i + e];
        const float a = to_f(x.e[e]), b = to_f(y.e[e]);
        x.e[e] = from_f<T>(a * cs.x - b * cs.y);
        y.e[e] = from_f<T>(b * cs.x + a * cs.y);
      }
      *reinterpret_cast<V *>(dst + i) = x;
      *reinterpret_cast<V *>(dst + half + i) = y;
      return;
    }
    const int i = 2 * half + (task - pair_tasks) * N;
    *reinterpret_cast<V *>(dst + i) = *reinterpret_cast<const V *>(src + i);
    return;
  }
  if (N == 1) {
    if (task < half) {
      const float2 cs = turn[task];
      const float a = to_f(src[2 * task]), b = to_f(src[2 * task + 1]);
      dst[2 * task] = from_f<T>(a * cs.x - b * cs.y);
      dst[2 * task + 1] = from_f<T>(b * cs.x + a * cs.y);
    } else {
      dst[task + half] = src[task + half];
    }
    return;
  }
  const int i = task * N;
  V x = *reinterpret_cast<const V *>(src + i);
  if (i < 2 * half) {
#pragma unroll
    for (int e = 0; e + 1 < N; e += 2) {
      const float2 cs = turn[(i + e) / 2];
      const float a = to_f(x.e[e]), b = to_f(x.e[e + 1]);
      x.e[e] = from_f<T>(a * cs.x - b * cs.y);
      x.e[e + 1] = from_f<T>(b * cs.x + a * cs.y);
    }
  }
  *reinterpret_cast<V *>(dst + i) = x;
}

template <typename T, int N>
__global__ void __launch_bounds__(kThreads) rotate_append_kernel(const __grid_constant__ Params p) {
  extern __shared__ float2 turn[];
  const emmy_rotate_append_args &a = p.a;
  const int token = blockIdx.x, half = a.rotary_dim / 2;
  const int *positions = reinterpret_cast<const int *>(a.positions);
  const int *pair_axis = reinterpret_cast<const int *>(a.pair_axis);
  const float *frequencies = reinterpret_cast<const float *>(a.frequencies);
  for (int i = threadIdx.x; i < half; i += kThreads) {
    const int axis = pair_axis ? min(max(pair_axis[i], 0), a.axes - 1) : 0;
    const double turns = double(positions[axis * a.positions_stride + token]) * double(frequencies[i]) *
                         0.31830988618379067154;             // in half turns
    float s, c;
    sincospif(float(turns - 2.0 * rint(0.5 * turns)), &s, &c);
    turn[i] = make_float2(c, s);
  }
  __syncthreads();
  const int64_t slot = a.kv_heads ? reinterpret_cast<const int *>(a.slots)[token] : -1;
  const bool stored = slot >= 0 && slot < int64_t(a.pages) * a.page_size;
  const int64_t page = stored ? slot / a.page_size : 0, within = stored ? slot % a.page_size : 0;
  const int q_end = a.q_heads * p.q_tasks;
  const int k_end = q_end + (stored ? a.kv_heads * p.k_tasks : 0);
  const int v_end = k_end + (stored ? a.kv_heads * p.v_tasks : 0);
  for (int t = threadIdx.x; t < v_end; t += kThreads) {
    if (t < q_end) {
      const int head = t / p.q_tasks, task = t - head * p.q_tasks;
      rotate_task<T, N>(reinterpret_cast<const T *>(a.q) + token * a.q_stride[0] + head * a.q_stride[1],
                        reinterpret_cast<T *>(a.q_out) + token * a.q_out_stride[0] + head * a.q_out_stride[1],
                        task, half, a.interleaved, turn);
    } else if (t < k_end) {
      const int head = (t - q_end) / p.k_tasks, task = (t - q_end) - head * p.k_tasks;
      rotate_task<T, N>(reinterpret_cast<const T *>(a.k) + token * a.k_stride[0] + head * a.k_stride[1],
                        reinterpret_cast<T *>(a.k_cache) + page * a.k_cache_stride[0] +
                            within * a.k_cache_stride[1] + head * a.k_cache_stride[2],
                        task, half, a.interleaved, turn);
    } else {
      const int head = (t - k_end) / p.v_tasks, task = (t - k_end) - head * p.v_tasks;
      using V = Vec<T, N>;
      const T *src = reinterpret_cast<const T *>(a.v) + token * a.v_stride[0] + head * a.v_stride[1];
      T *dst = reinterpret_cast<T *>(a.v_cache) + page * a.v_cache_stride[0] + within * a.v_cache_stride[1] +
               head * a.v_cache_stride[2];
      *reinterpret_cast<V *>(dst + task * N) = *reinterpret_cast<const V *>(src + task * N);
    }
  }
}

int fail(const char *fmt, long a = 0, long b = 0) {
  char buf[256];
  snprintf(buf, sizeof buf, fmt, a, b);
  return emmy_internal_fail(EMMY_EINVAL, buf);
}

template <typename T, int N> int launch(Params &p, cudaStream_t s) {
  const emmy_rotate_append_args &a = p.a;
  const int half = a.rotary_dim / 2;
  p.v_tasks = a.head_dim / N;
  p.q_tasks = p.k_tasks = (a.interleaved && N > 1) ? a.head_dim / N : (half + a.head_dim - a.rotary_dim) / N;
  rotate_append_kernel<T, N><<<a.tokens, kThreads, half * sizeof(float2), s>>>(p);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    char buf[256];
    snprintf(buf, sizeof buf, "emmy_rotate_append: launch failed: %s", cudaGetErrorString(e));
    return emmy_internal_fail(static_cast<int>(e), buf);
  }
  return 0;
}

// 16-byte accesses need every address and stride to be a multiple of 16 bytes
// and heads, halves and the part that stays to be whole vectors.
template <typename T> int dispatch(Params &p, cudaStream_t s) {
  constexpr int N = 16 / sizeof(T);
  const emmy_rotate_append_args &a = p.a;
  uint64_t addr = 0;
  int64_t strides = 0;
  if (a.q_heads) {
    addr |= a.q | a.q_out;
    for (int i = 0; i < 2; ++i) strides |= a.q_stride[i] | a.q_out_stride[i];
  }
  if (a.kv_heads) {
    addr |= a.k | a.v | a.k_cache | a.v_cache;
    for (int i = 0; i < 2; ++i) strides |= a.k_stride[i] | a.v_stride[i];
    for (int i = 0; i < 3; ++i) strides |= a.k_cache_stride[i] | a.v_cache_stride[i];
  }
  const int unit = a.interleaved ? a.rotary_dim : a.rotary_dim / 2;
  if (addr % 16 == 0 && strides % N == 0 && a.head_dim % N == 0 && unit % N == 0)
    return launch<T, N>(p, s);
  return launch<T, 1>(p, s);
}

}  // namespace

extern "C" EMMY_API int emmy_rotate_append(const emmy_rotate_append_args *a, void *stream) {
  if (!a) return fail("emmy_rotate_append: bad argument");
  if (a->dtype != 6 && a->dtype != 7 && a->dtype != 9)
    return fail("emmy_rotate_append: dtype %ld (f16, f32 or bf16)", a->dtype);
  if (a->tokens < 0 || a->q_heads < 0 || a->kv_heads < 0 || a->q_heads > 65536 || a->kv_heads > 65536)
    return fail("emmy_rotate_append: bad count of tokens or heads");
  if (a->head_dim < 1 || a->head_dim > 1024)
    return fail("emmy_rotate_append: head_dim %ld outside 1..1024", a->head_dim);
  if (a->rotary_dim < 0 || a->rotary_dim > a->head_dim || a->rotary_dim % 2)
    return fail("emmy_rotate_append: rotary_dim %ld must be even and at most head_dim %ld", a->rotary_dim, a->head_dim);
  if (a->axes < 1 || a->axes > 16) return fail("emmy_rotate_append: %ld position axes (1..16)", a->axes);
  if (a->kv_heads && (a->pages < 0 || a->page_size < 1))
    return fail("emmy_rotate_append: a cache of %ld pages of %ld tokens", a->pages, a->page_size);
  if (a->tokens == 0 || (a->q_heads == 0 && a->kv_heads == 0)) return 0;
  if ((a->q_heads && (!a->q || !a->q_out)) ||
      (a->kv_heads && (!a->k || !a->v || !a->slots || (a->pages && (!a->k_cache || !a->v_cache)))) ||
      (a->rotary_dim && (!a->positions || !a->frequencies)))
    return fail("emmy_rotate_append: null address");
  const uint64_t elements = (a->q_heads ? a->q | a->q_out : 0) |
                            (a->kv_heads ? a->k | a->v | a->k_cache | a->v_cache : 0);
  if (elements % (a->dtype == 7 ? 4 : 2) || (a->kv_heads ? a->slots % 4 : 0) ||
      (a->rotary_dim ? (a->positions | a->frequencies | a->pair_axis) % 4 : 0))
    return fail("emmy_rotate_append: address not a multiple of its element's size");
  Params p{*a, 0, 0, 0};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->dtype == 6) return dispatch<__half>(p, s);
  if (a->dtype == 7) return dispatch<float>(p, s);
  return dispatch<__nv_bfloat16>(p, s);
}
