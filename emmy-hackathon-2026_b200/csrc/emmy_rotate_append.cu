// emmy_rotate_append.cu -- rotary positions on new queries and keys, keys and
// values into a paged cache, in one launch.
//
// A pair (x, y) of a head turns by the angle a = position * frequency:
// (x cos a - y sin a, y cos a + x sin a).  Every head of a token turns by the
// same angles, so the threads of a token compute its cosines and sines once
// into shared memory and then move the token's heads: each element is read once
// and written once, which is the floor of the operator.
//
// Half a head's vectors are a row of threads.  A thread has the same two vectors
// -- one of the first half and its partner in the second, or two that hold their
// pairs or stay as they are -- of the same head of every token it moves, so that
// what it does for a token is two loads, the turn and two stores: the operator
// is bound by instructions as soon as addresses are worked out head by head (298
// a pair of vectors then, 4,000 GB/s at 16,384 tokens of 32 + 8 heads of 128).
// Blocks stay for many tokens.  The vectors, position and slot of the next two
// are on their way to shared memory, each to its thread's own place, while one
// is turned: with one token ahead in registers 1,024 threads an SM kept too few
// bytes in flight (4,700 GB/s).  Blocks of 384 threads take the 48 heads of the
// video case in one share, with its angles formed once: 65 us, 6,150 GB/s, against
// 70 us of 256 in two; 4,095 tokens of 32 + 32 heads 35 us, 5,700 GB/s (replayed from a
// graph; called again and again 71 and 37 us).
//
// The angle is formed in 64 bits as a count of half turns and reduced there:
// at position 2^17 a 32-bit product is already off by 0.008 radians, and the
// reduction of a large 32-bit angle would cost a slow path besides.  Rotation
// is in 32 bits; the one rounding is to the cache's or q_out's type.
#include "../../include/emmy_b200.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <cstdio>

int emmy_internal_fail(int code, const char *msg);   // emmy_runtime.cpp

namespace {

constexpr int kThreads = 384, kBlocks = 3;      // at most a block; at least an SM
constexpr int kAhead = 3;                       // tokens in flight or being turned

struct Params {
  emmy_rotate_append_args a;
  int lanes;                       // threads of a row: a head's vectors by two
};

// N elements moved as one access: 16 bytes, or one element
template <typename T, int N> struct alignas(N * sizeof(T)) Vec { T e[N]; };

template <int N> __device__ __forceinline__ void widen(const Vec<float, N> &v, float *f) {
#pragma unroll
  for (int e = 0; e < N; ++e) f[e] = v.e[e];
}
template <int N> __device__ __forceinline__ void round_to(const float *f, Vec<float, N> &v) {
#pragma unroll
  for (int e = 0; e < N; ++e) v.e[e] = f[e];
}
template <int N> __device__ __forceinline__ void widen(const Vec<__half, N> &v, float *f) {
  if constexpr (N == 1) {
    f[0] = __half2float(v.e[0]);
  } else {
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const float2 p = __half22float2(__halves2half2(v.e[e], v.e[e + 1]));
      f[e] = p.x, f[e + 1] = p.y;
    }
  }
}
template <int N> __device__ __forceinline__ void round_to(const float *f, Vec<__half, N> &v) {
  if constexpr (N == 1) {
    v.e[0] = __float2half_rn(f[0]);
  } else {
#pragma unroll
    for (int e = 0; e < N; e += 2) *reinterpret_cast<__half2 *>(v.e + e) = __floats2half2_rn(f[e], f[e + 1]);
  }
}
template <int N> __device__ __forceinline__ void widen(const Vec<__nv_bfloat16, N> &v, float *f) {
  if constexpr (N == 1) {
    f[0] = __bfloat162float(v.e[0]);
  } else {
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const uint32_t two = *reinterpret_cast<const uint32_t *>(v.e + e);     // a bfloat16 is a float's upper half
      f[e] = __uint_as_float(two << 16), f[e + 1] = __uint_as_float(two & 0xffff0000u);
    }
  }
}
template <int N> __device__ __forceinline__ void round_to(const float *f, Vec<__nv_bfloat16, N> &v) {
  if constexpr (N == 1) {
    v.e[0] = __float2bfloat16_rn(f[0]);
  } else {
#pragma unroll
    for (int e = 0; e < N; e += 2) *reinterpret_cast<__nv_bfloat162 *>(v.e + e) = __floats2bfloat162_rn(f[e], f[e + 1]);
  }
}

template <int BYTES> __device__ __forceinline__ void copy_async(void *to, const void *from) {
  const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(to));
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(from), "n"(BYTES) : "memory");
}

// blockDim = (lanes, heads, tokens); blockIdx.y: the block's share of the heads
// of queries, keys and values.  WITHIN: the pairs lie inside a vector
// (interleaved, N > 1); otherwise a pair is one element of each of the thread's
// two vectors.
template <typename T, int N, bool WITHIN>
__global__ void __launch_bounds__(kThreads, kBlocks) rotate_append_kernel(const __grid_constant__ Params p) {
  using V = Vec<T, N>;
  extern __shared__ __align__(16) float angles[];
  const emmy_rotate_append_args &a = p.a;
  const int half = a.rotary_dim / 2, heads = a.q_heads + 2 * a.kv_heads;
  const int lane = threadIdx.x, step = gridDim.x * blockDim.z;
  const int head = blockIdx.y * blockDim.y + threadIdx.y;

  // where this thread's head comes from and goes to
  const bool query = head < a.q_heads, turns = head < a.q_heads + a.kv_heads, moves = head < heads;
  const T *src;
  T *dst;
  int64_t src_token, dst_page, dst_token;      // queries: dst_token of q_out, no pages
  if (query) {
    src = reinterpret_cast<const T *>(a.q) + head * a.q_stride[1];
    dst = reinterpret_cast<T *>(a.q_out) + head * a.q_out_stride[1];
    src_token = a.q_stride[0], dst_page = 0, dst_token = a.q_out_stride[0];
  } else if (turns) {
    src = reinterpret_cast<const T *>(a.k) + (head - a.q_heads) * a.k_stride[1];
    dst = reinterpret_cast<T *>(a.k_cache) + (head - a.q_heads) * a.k_cache_stride[2];
    src_token = a.k_stride[0], dst_page = a.k_cache_stride[0], dst_token = a.k_cache_stride[1];
  } else {
    src = reinterpret_cast<const T *>(a.v) + (head - a.q_heads - a.kv_heads) * a.v_stride[1];
    dst = reinterpret_cast<T *>(a.v_cache) + (head - a.q_heads - a.kv_heads) * a.v_cache_stride[2];
    src_token = a.v_stride[0], dst_page = a.v_cache_stride[0], dst_token = a.v_cache_stride[1];
  }
  // its two vectors, `apart` elements from one another
  bool turn_one, turn_two;
  int apart, first_pair, second_pair;         // pairs of the first and (WITHIN) the second
  {
    int one, two;
    if (WITHIN) {
      one = lane * N;
      two = (lane + p.lanes) * N;
      turn_one = one < a.rotary_dim;
      turn_two = two < a.rotary_dim;
      first_pair = one / 2, second_pair = two / 2;
    } else {
      turn_one = turn_two = lane * N < half;
      // (threads next to one another move vectors next to one another: two of
      // one thread side by side would ask for every 32-byte sector twice)
      one = !turn_one ? half + lane * N : a.interleaved ? lane * 2 : lane * N;
      two = !turn_one ? one + p.lanes * N - half : a.interleaved ? one + 1 : half + lane * N;
      first_pair = second_pair = lane * N;
    }
    turn_one = turn_one && turns;
    turn_two = turn_two && turns;
    apart = two < a.head_dim ? two - one : 0;   // an odd head ends with one: moved twice
    src += one;
    dst += one;
  }

  // the pair whose angle this thread forms (more than one where heads are few)
  const int pair = threadIdx.y * blockDim.x + lane, pairs_at_once = blockDim.x * blockDim.y;
  auto axis_of = [&](int i) {
    return a.pair_axis ? min(max(reinterpret_cast<const int *>(a.pair_axis)[i], 0), a.axes - 1) : 0;
  };
  const int *const positions = reinterpret_cast<const int *>(a.positions) + (pair < half ? axis_of(pair) * a.positions_stride : 0);
  const float frequency = pair < half ? reinterpret_cast<const float *>(a.frequencies)[pair] : 0.f;
  const int *const slots = reinterpret_cast<const int *>(a.slots);
  const int64_t n_slots = int64_t(a.pages) * a.page_size;
  auto turn = [&](float *to, int i, int position, float f) {
    const double turned = double(position) * double(f) * 0.31830988618379067154;     // half turns
    float s, c;
    sincospif(float(turned - 2.0 * rint(0.5 * turned)), &s, &c);
    to[i] = c;
    to[half + i] = s;
  };

  // single elements (N = 1) are read where they are used: too small to copy
  constexpr bool COPIED = N * sizeof(T) == 16;
  const int threads = blockDim.x * blockDim.y * blockDim.z, me = (threadIdx.z * blockDim.y + threadIdx.y) * blockDim.x + lane;
  V *const vectors = reinterpret_cast<V *>(angles + blockDim.z * 2 * a.rotary_dim) + me;       // [kAhead][2][threads]
  int *const numbers = reinterpret_cast<int *>(vectors - me + (COPIED ? kAhead * 2 * threads : 0)) + me;   // [kAhead][2][threads]
  auto fetch = [&](int token, int stage) {
    if (COPIED && token < a.tokens) {
      if (moves) {
        const T *at = src + token * src_token;
        copy_async<16>(vectors + stage * 2 * threads, at);
        copy_async<16>(vectors + (stage * 2 + 1) * threads, at + apart);
        if (!query) copy_async<4>(numbers + stage * 2 * threads, slots + token);
      }
      if (pair < half) copy_async<4>(numbers + (stage * 2 + 1) * threads, positions + token);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int token = blockIdx.x * blockDim.z + threadIdx.z, stage = 0;
#pragma unroll
  for (int k = 0; k + 1 < kAhead; ++k) fetch(token + k * step, k);
  float *angle = angles + threadIdx.z * 2 * a.rotary_dim;      // of this token and the next in turn
  const bool turning = blockIdx.y * int(blockDim.y) < a.q_heads + a.kv_heads;
  int flip = a.rotary_dim;
  for (int base = blockIdx.x * blockDim.z; base < a.tokens; base += step) {
    fetch(token + (kAhead - 1) * step, (stage + kAhead - 1) % kAhead);
    asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
    if (turning) {
      if (token < a.tokens && pair < half) {
        turn(angle, pair, COPIED ? numbers[(stage * 2 + 1) * threads] : positions[token], frequency);
        for (int i = pair + pairs_at_once; i < half; i += pairs_at_once)
          turn(angle, i, reinterpret_cast<const int *>(a.positions)[axis_of(i) * a.positions_stride + token],
               reinterpret_cast<const float *>(a.frequencies)[i]);
      }
      __syncthreads();
    }
    if (token < a.tokens && moves) {
      const T *at = src + token * src_token;
      V u = COPIED ? vectors[stage * 2 * threads] : *reinterpret_cast<const V *>(at);
      V v = COPIED ? vectors[(stage * 2 + 1) * threads] : *reinterpret_cast<const V *>(at + apart);
      const int slot = query ? 0 : COPIED ? numbers[stage * 2 * threads] : slots[token];
      if (turn_one) {
        float f[N], g[N], c[N], s[N];
        widen(u, f);
        widen(v, g);
        constexpr int M = N == 1 ? 1 : WITHIN ? N / 2 : 4;
        using Angles = Vec<float, M>;
#pragma unroll
        for (int e = 0; e < N; e += M) {
          // cosines and sines of N pairs; WITHIN: half of them for each vector
          const int i = !WITHIN ? first_pair + e : e < N / 2 ? first_pair + e : second_pair + e - N / 2;
          const bool used = !WITHIN || e < N / 2 || turn_two;
          const Angles ce = *reinterpret_cast<const Angles *>(angle + (used ? i : 0));
          const Angles se = *reinterpret_cast<const Angles *>(angle + half + (used ? i : 0));
#pragma unroll
          for (int k = 0; k < M; ++k) c[e + k] = ce.e[k], s[e + k] = se.e[k];
        }
        if (WITHIN) {
#pragma unroll
          for (int e = 0; e < N; e += 2) {
            const float f0 = f[e], f1 = f[e + 1], g0 = g[e], g1 = g[e + 1], ce = c[e / 2], se = s[e / 2],
                        cg = c[N / 2 + e / 2], sg = s[N / 2 + e / 2];
            f[e] = f0 * ce - f1 * se;
            f[e + 1] = f1 * ce + f0 * se;
            g[e] = g0 * cg - g1 * sg;
            g[e + 1] = g1 * cg + g0 * sg;
          }
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const float fe = f[e], ge = g[e];
            f[e] = fe * c[e] - ge * s[e];
            g[e] = ge * c[e] + fe * s[e];
          }
        }
        round_to(f, u);
        if (turn_two) round_to(g, v);
      }
      if (query || (slot >= 0 && slot < n_slots)) {
        T *to;
        if (query) {
          to = dst + token * dst_token;
        } else {
          const int page = slot / a.page_size;
          to = dst + page * dst_page + (slot - page * a.page_size) * dst_token;
        }
        *reinterpret_cast<V *>(to) = u;
        *reinterpret_cast<V *>(to + apart) = v;
      }
    }
    token += step;
    stage = (stage + 1) % kAhead;
    angle += flip;
    flip = -flip;
  }
}

int fail(const char *fmt, long a = 0, long b = 0) {
  char buf[256];
  snprintf(buf, sizeof buf, fmt, a, b);
  return emmy_internal_fail(EMMY_EINVAL, buf);
}

int failed(cudaError_t e) {
  char buf[256];
  snprintf(buf, sizeof buf, "emmy_rotate_append: launch failed: %s", cudaGetErrorString(e));
  return emmy_internal_fail(static_cast<int>(e), buf);
}

template <typename T, int N, bool WITHIN> int launch(Params &p, cudaStream_t s) {
  const emmy_rotate_append_args &a = p.a;
  p.lanes = (a.head_dim / N + 1) / 2;
  // heads in shares of equal size, and a few tokens a block where one is small
  const int heads = a.q_heads + 2 * a.kv_heads, most = p.lanes < kThreads ? kThreads / p.lanes : 1;
  const int shares = (heads + most - 1) / most, rows = (heads + shares - 1) / shares;
  int tokens = kThreads / 2 / (p.lanes * rows);
  tokens = tokens < 1 ? 1 : tokens > 64 ? 64 : tokens;
  if (tokens > a.tokens) tokens = a.tokens;
  static std::atomic<int> known[64];         // SMs of each device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return failed(e);
  int sms = dev < 64 ? known[dev].load() : 0;
  if (!sms) {
    e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return failed(e);
    if (dev < 64) known[dev].store(sms);
  }
  const int want = (a.tokens + tokens - 1) / tokens;
  int resident = sms * (kBlocks * kThreads / (p.lanes * rows * tokens)) / shares;
  if (resident < 1) resident = 1;
  const dim3 grid(want < resident ? want : resident, shares), block(p.lanes, rows, tokens);
  // angles of two turns; vectors, slots and positions on their way (N > 1): with
  // 256 components and 384 threads 47 KiB, under the 48 that need no asking
  const size_t smem = size_t(tokens) * 2 * a.rotary_dim * sizeof(float) +
                      (N > 1 ? size_t(kAhead) * 2 * p.lanes * rows * tokens * (16 + 4) : 0);
  rotate_append_kernel<T, N, WITHIN><<<grid, block, smem, s>>>(p);
  e = cudaGetLastError();
  return e == cudaSuccess ? 0 : failed(e);
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
  const bool whole = addr % 16 == 0 && strides % N == 0 && a.head_dim % (2 * N) == 0;
  // (vectors of angles: 16 bytes of shared memory hold the cosines of 4 pairs)
  if (whole && a.interleaved && a.rotary_dim % N == 0 && a.rotary_dim % 8 == 0) return launch<T, N, true>(p, s);
  if (whole && !a.interleaved && a.rotary_dim / 2 % N == 0) return launch<T, N, false>(p, s);
  return launch<T, 1, false>(p, s);
}

}  // namespace

extern "C" EMMY_API int emmy_rotate_append(const emmy_rotate_append_args *a, void *stream) {
  if (!a) return fail("emmy_rotate_append: bad argument");
  if (a->dtype != 6 && a->dtype != 7 && a->dtype != 9)
    return fail("emmy_rotate_append: dtype %ld (f16, f32 or bf16)", a->dtype);
  if (a->tokens < 0 || a->tokens > (1 << 30) || a->q_heads < 0 || a->kv_heads < 0 || a->q_heads > 1024 || a->kv_heads > 1024)
    return fail("emmy_rotate_append: bad count of tokens or heads");
  if (a->head_dim < 1 || a->head_dim > 256)
    return fail("emmy_rotate_append: head_dim %ld outside 1..256", a->head_dim);
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
  Params p;
  p.a = *a;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->dtype == 6) return dispatch<__half>(p, s);
  if (a->dtype == 7) return dispatch<float>(p, s);
  return dispatch<__nv_bfloat16>(p, s);
}
