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
//
// With norms (queries and keys of each head times the reciprocal of their root mean
// square and a weight) or a cache of 8-bit floats (times a power of two -- exactly -- and
// rounded once), each element takes twice the instructions, and that walk waited at its
// barrier of each token: 8,191 tokens of 32 + 8 heads of 128 in 57 us, whatever the
// tokens ahead.  Heads of vectors go through append_kernel instead, a warp a token: its
// angles and weights stay in registers for all heads, the squares' sums meet by shuffles,
// arithmetic is on pairs of floats (fma.rn.f32x2), the norm's factor and the cache's power
// of two are one at the end, and nothing waits for another warp: 34.5 us, 5,400 GB/s.
// Heads that are no whole vectors, or of which a part turns that is none (halves of 12 of 96
// components, say), take the walk above an element at a time, with the squares in shared
// memory: right, and slow, as each element is a load and a store of its own (8,191 tokens of
// 32 + 8 heads of 96, bfloat16: 276 us, 39 where all of a head turns).
#include "../../include/emmy_b200.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <cstdio>
#include <type_traits>

int emmy_internal_fail(int code, const char *msg);   // emmy_runtime.cpp

// SMs of the current device, which is asked once; a cudaError_t
int emmy_internal_sms(int *sms) {
  static std::atomic<int> known[64];
  int dev = 0;
  if (const cudaError_t e = cudaGetDevice(&dev)) return e;
  *sms = dev < 64 ? known[dev].load() : 0;
  if (*sms) return cudaSuccess;
  if (const cudaError_t e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev)) return e;
  if (dev < 64) known[dev].store(*sms);
  return cudaSuccess;
}

namespace {

constexpr int kThreads = 384, kBlocks = 3;      // at most a block; at least an SM
constexpr int kNormBlocks = 2;                  // with norms, whose weights take registers
constexpr int kAhead = 3;                       // tokens in flight or being turned

struct Params {
  emmy_rotate_append_args a;
  int lanes;                       // threads of a row: a head's vectors by two
  uint64_t q_weight, k_weight, exponents;
  float eps;
  uint32_t page_inverse;           // slot / page_size = slot * page_inverse >> page_shift
  int page_shift;
};

struct E4M3 { uint8_t bits; };     // an 8-bit float: 4 exponent bits, largest 448

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

// the largest 8-bit float for what is larger; NaN stays
template <int N> __device__ __forceinline__ void round_to(const float *f, Vec<E4M3, N> &v) {
  uint16_t two;
  if constexpr (N == 1) {
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(two) : "f"(0.f), "f"(f[0]));
    v.e[0].bits = static_cast<uint8_t>(two);
  } else {
    uint32_t words[N / 4];
#pragma unroll
    for (int e = 0; e < N; e += 4) {
      uint16_t more;
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(two) : "f"(f[e + 1]), "f"(f[e]));
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(more) : "f"(f[e + 3]), "f"(f[e + 2]));
      words[e / 4] = two | uint32_t(more) << 16;
    }
    if constexpr (N == 8)
      *reinterpret_cast<uint2 *>(&v) = make_uint2(words[0], words[1]);
    else
      *reinterpret_cast<uint32_t *>(&v) = words[0];
  }
}

// ---- pairs of floats
__device__ __forceinline__ uint64_t pair_of(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
template <typename T, int N> __device__ __forceinline__ void widen2(const Vec<T, N> &v, uint64_t *f) {
  float x[N];
  widen(v, x);
#pragma unroll
  for (int e = 0; e < N; e += 2) f[e / 2] = pair_of(x[e], x[e + 1]);
}
template <typename T, int N> __device__ __forceinline__ void round2(const uint64_t *f, float by, Vec<T, N> &v) {
  float x[N];
#pragma unroll
  for (int e = 0; e < N; e += 2) {
    const float2 t = unpair(mul2(f[e / 2], pair_of(by, by)));
    x[e] = t.x, x[e + 1] = t.y;
  }
  round_to(x, v);
}

// Cosine and sine of position * frequency.  The angle is formed in 64 bits as half turns
// and goes on as 32 bits and the rest, a first-order step: left out, that is up to 2^-25
// half turns, 9e-8 radians, as much as the other roundings of a key together (of 8 million
// 8-bit keys 17 to 27 went to the other neighbour, 4 to 16 with it; the time is the same).
// Without norms and 8 bits the walk ends at 32 bits, and rotate_append's results stay as they are.
__device__ __forceinline__ void angle_of(int position, float frequency, float &c, float &s) {
  double turned = double(position) * double(frequency) * 0.31830988618379067154;
  turned -= 2.0 * rint(0.5 * turned);
  const float near = float(turned), rest = float(turned - double(near)) * 3.14159265f;
  float c0, s0;
  sincospif(near, &s0, &c0);
  c = fmaf(-s0, rest, c0);
  s = fmaf(c0, rest, s0);
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
// two vectors.  C: the cache's elements, T or 8-bit floats.  With norms or an 8-bit
// cache: single elements only (append_kernel has the vectors).
template <typename T, typename C, int N, bool WITHIN, bool NORM>
__global__ void __launch_bounds__(kThreads, NORM ? kNormBlocks : kBlocks) rotate_append_kernel(const __grid_constant__ Params p) {
  using V = Vec<T, N>;
  constexpr bool SMALL = !std::is_same<T, C>::value;
  static_assert(N == 1 || !(NORM || SMALL), "vectors with norms or 8 bits are append_kernel's");
  extern __shared__ __align__(16) float angles[];
  const emmy_rotate_append_args &a = p.a;
  const int half = a.rotary_dim / 2, heads = a.q_heads + 2 * a.kv_heads;
  const int lane = threadIdx.x, step = gridDim.x * blockDim.z;
  const int head = blockIdx.y * blockDim.y + threadIdx.y;

  // where this thread's head comes from and goes to
  const bool query = head < a.q_heads, turns = head < a.q_heads + a.kv_heads, moves = head < heads;
  const T *src;
  T *dst;
  [[maybe_unused]] C *small = nullptr;         // a cache of another type
  [[maybe_unused]] float small_scale = 1.f;
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
  [[maybe_unused]] V weight_one{}, weight_two{};
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
    if constexpr (SMALL) {
      if (!query && moves) {
        const int kv_head = head - a.q_heads - (turns ? 0 : a.kv_heads);
        small = (turns ? reinterpret_cast<C *>(a.k_cache) + kv_head * a.k_cache_stride[2]
                       : reinterpret_cast<C *>(a.v_cache) + kv_head * a.v_cache_stride[2]) + one;
        const int e = p.exponents ? reinterpret_cast<const int *>(p.exponents)[kv_head + (turns ? 0 : a.kv_heads)] : 0;
        small_scale = exp2f(float(-min(max(e, EMMY_MIN_EXPONENT), EMMY_MAX_EXPONENT)));      // (exact)
      }
    }
    if constexpr (NORM) {
      if (turns) {
        const T *w = reinterpret_cast<const T *>(query ? p.q_weight : p.k_weight) + one;
        weight_one = *reinterpret_cast<const V *>(w);
        weight_two = *reinterpret_cast<const V *>(w + apart);
      }
    }
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
    if constexpr (NORM || SMALL) {
      angle_of(position, f, to[i], to[half + i]);
    } else {
      const double turned = double(position) * double(f) * 0.31830988618379067154;     // half turns
      float s, c;
      sincospif(float(turned - 2.0 * rint(0.5 * turned)), &s, &c);
      to[i] = c;
      to[half + i] = s;
    }
  };

  // single elements (N = 1) are read where they are used: too small to copy
  constexpr bool COPIED = N * sizeof(T) == 16;
  const int threads = blockDim.x * blockDim.y * blockDim.z, me = (threadIdx.z * blockDim.y + threadIdx.y) * blockDim.x + lane;
  V *const vectors = reinterpret_cast<V *>(angles + blockDim.z * 2 * a.rotary_dim) + me;       // [kAhead][2][threads]
  int *const numbers = reinterpret_cast<int *>(vectors - me + (COPIED ? kAhead * 2 * threads : 0)) + me;   // [kAhead][2][threads]
  // (NORM, where nothing is copied) sums of squares of this token and the next in turn, [2][threads]
  [[maybe_unused]] float *const squares = reinterpret_cast<float *>(vectors - me) + me;
  [[maybe_unused]] int odd = 0;
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
    [[maybe_unused]] V read_one{}, read_two{};   // (q_out may be q: read before any of the head is written)
    if constexpr (NORM) {
      float sum = 0.f;
      if (token < a.tokens && moves) {
        const T *at = src + token * src_token;
        read_one = *reinterpret_cast<const V *>(at);
        read_two = *reinterpret_cast<const V *>(at + apart);
        float f[N], g[N];
        widen(read_one, f);
        widen(read_two, g);
#pragma unroll
        for (int e = 0; e < N; ++e) sum += f[e] * f[e];
        if (apart) {
#pragma unroll
          for (int e = 0; e < N; ++e) sum += g[e] * g[e];
        }
      }
      squares[odd] = sum;
    }
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
      V u, v;
      if constexpr (NORM) {
        u = read_one;
        v = read_two;
      } else {
        const T *at = src + token * src_token;
        u = COPIED ? vectors[stage * 2 * threads] : *reinterpret_cast<const V *>(at);
        v = COPIED ? vectors[(stage * 2 + 1) * threads] : *reinterpret_cast<const V *>(at + apart);
      }
      const int slot = query ? 0 : COPIED ? numbers[stage * 2 * threads] : slots[token];
      float f[N], g[N];
      if constexpr (NORM || SMALL) {
        widen(u, f);
        widen(v, g);
      }
      if constexpr (NORM) {
        if (turns) {
          const float *of_head = squares - lane + odd;
          float sum = 0.f;
          if (p.lanes % 4 == 0) {
            for (int i = 0; i < p.lanes; i += 4) {
              const float4 x = *reinterpret_cast<const float4 *>(of_head + i);
              sum += (x.x + x.y) + (x.z + x.w);
            }
          } else {
            for (int i = 0; i < p.lanes; ++i) sum += of_head[i];
          }
          const float by = __frsqrt_rn(sum / float(a.head_dim) + p.eps);
          float w[N];
          widen(weight_one, w);
#pragma unroll
          for (int e = 0; e < N; ++e) f[e] = f[e] * by * w[e];
          widen(weight_two, w);
#pragma unroll
          for (int e = 0; e < N; ++e) g[e] = g[e] * by * w[e];
        }
      }
      if (turn_one) {
        float c[N], s[N];
        if constexpr (!NORM && !SMALL) {
          widen(u, f);
          widen(v, g);
        }
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
            g[e] = g0 * cg - g1 * sg;      // (left out below where it does not turn)
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
        if constexpr (!NORM) {
          round_to(f, u);
          if (turn_two) round_to(g, v);
        }
      }
      if constexpr (NORM) {
        if (turns) {
          round_to(f, u);
          round_to(g, v);
        }
      }
      if (SMALL && !query) {
        if constexpr (SMALL) {
          if (slot >= 0 && slot < n_slots) {
            const int page = slot / a.page_size;
            C *to = small + page * dst_page + (slot - page * a.page_size) * dst_token;
            Vec<C, N> r;
#pragma unroll
            for (int e = 0; e < N; ++e) f[e] *= small_scale, g[e] *= small_scale;
            round_to(f, r);
            *reinterpret_cast<Vec<C, N> *>(to) = r;
            round_to(g, r);
            *reinterpret_cast<Vec<C, N> *>(to + apart) = r;
          }
        }
      } else if (query || (slot >= 0 && slot < n_slots)) {
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
    if constexpr (NORM) odd = threads - odd;
    token += step;
    stage = (stage + 1) % kAhead;
    angle += flip;
    flip = -flip;
  }
}

constexpr int kWarps = 4, kGroups = 4;      // of a block of append_kernel; groups of heads on their way or being turned

// A warp has a token (of 4 a block) and every gridDim.y-th group of heads, `lanes` threads
// a head, 32 at most (256 components of 4 bytes).  A thread's vectors and pairs as above.
// LANES: `lanes` where it is one of the common ones, else 0.
template <typename T, typename C, int N, bool WITHIN, bool NORM, int LANES>
__global__ void __launch_bounds__(32 * kWarps, 5) append_kernel(const __grid_constant__ Params p) {
  using V = Vec<T, N>;
  constexpr bool SMALL = !std::is_same<T, C>::value;
  extern __shared__ __align__(16) float angles[];           // vectors [kWarps][kGroups][2][32], angles [kWarps][2][half]
  const emmy_rotate_append_args &a = p.a;
  const int half = a.rotary_dim / 2, heads = a.q_heads + 2 * a.kv_heads, lanes = LANES ? LANES : p.lanes;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, token = blockIdx.x * kWarps + warp;
  if (token >= a.tokens) return;
  const int at_once = 32 / lanes, mine = lane % lanes, step = at_once * gridDim.y;
  // (of 32 lanes, those that are too few for another head have none)
  int head = lane / lanes < at_once ? blockIdx.y * at_once + lane / lanes : heads;
  // its two vectors, `apart` elements from one another, and their first pairs
  bool turn_one, turn_two;
  int one, apart, first_pair, second_pair;
  if (WITHIN) {
    one = mine * N;
    apart = lanes * N;
    turn_one = one < a.rotary_dim;
    turn_two = one + apart < a.rotary_dim;
    first_pair = one / 2, second_pair = (one + apart) / 2;
  } else {
    turn_one = turn_two = mine * N < half;
    one = turn_one ? mine * N : half + mine * N;
    apart = turn_one ? half : lanes * N - half;
    first_pair = second_pair = mine * N;
  }
  // a head's vectors go to shared memory, each to its thread's own place, some groups ahead
  V *const ring = reinterpret_cast<V *>(angles) + warp * kGroups * 2 * 32 + lane;
  auto fetch = [&](int h, int stage) {
    if (h < heads) {
      const T *at;
      if (h < a.q_heads)
        at = reinterpret_cast<const T *>(a.q) + token * a.q_stride[0] + h * a.q_stride[1];
      else if (h < a.q_heads + a.kv_heads)
        at = reinterpret_cast<const T *>(a.k) + token * a.k_stride[0] + (h - a.q_heads) * a.k_stride[1];
      else
        at = reinterpret_cast<const T *>(a.v) + token * a.v_stride[0] + (h - a.q_heads - a.kv_heads) * a.v_stride[1];
      copy_async<16>(ring + stage * 64, at + one);
      copy_async<16>(ring + stage * 64 + 32, at + one + apart);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int k = 0; k + 1 < kGroups; ++k) fetch(head + k * step, k);
  int stage = 0;
  int64_t k_at = 0, v_at = 0;                   // where the token's keys and values go
  bool stored = false;
  if (a.kv_heads) {
    const int slot = __ldg(reinterpret_cast<const int *>(a.slots) + token);
    if (slot >= 0 && slot < int64_t(a.pages) * a.page_size) {
      const int page = static_cast<int>(uint64_t(slot) * p.page_inverse >> p.page_shift), within = slot - page * a.page_size;
      stored = true;
      k_at = page * a.k_cache_stride[0] + within * a.k_cache_stride[1];
      v_at = page * a.v_cache_stride[0] + within * a.v_cache_stride[1];
    }
  }
  // this token's angles, and of them those of this thread's pairs: c[0..N) and s[0..N);
  // WITHIN: the first half of the first vector, the others of the second
  float *const angle = angles + kWarps * kGroups * 64 * (sizeof(V) / 4) + warp * 2 * half;
  for (int i = lane; i < half; i += 32) {
    const int axis = a.pair_axis ? min(max(__ldg(reinterpret_cast<const int *>(a.pair_axis) + i), 0), a.axes - 1) : 0;
    angle_of(__ldg(reinterpret_cast<const int *>(a.positions) + axis * a.positions_stride + token),
             __ldg(reinterpret_cast<const float *>(a.frequencies) + i), angle[i], angle[half + i]);
  }
  __syncwarp();
  float c[N], s[N], minus[N];
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const int i = !WITHIN ? first_pair + e : e < N / 2 ? first_pair + e : second_pair + e - N / 2;
    const bool used = !WITHIN || e < N / 2 ? turn_one : turn_two;
    c[e] = used ? angle[i] : 1.f;
    s[e] = used ? angle[half + i] : 0.f;
    minus[e] = -s[e];
  }
  uint64_t weight[NORM ? N : 1];                // of both vectors, of queries or keys
  int weights_of = -1;
  const float reciprocal = 1.f / float(a.head_dim);
#pragma unroll 1
  for (int n = 0; blockIdx.y * at_once + n * step < heads; ++n, head += step) {
    const bool query = head < a.q_heads, turns = head < a.q_heads + a.kv_heads;
    uint64_t f[N / 2], g[N / 2];
    fetch(head + (kGroups - 1) * step, (stage + kGroups - 1) % kGroups);
    asm volatile("cp.async.wait_group %0;" ::"n"(kGroups - 1) : "memory");
    const V left = ring[stage * 64], right = ring[stage * 64 + 32];
    stage = (stage + 1) % kGroups;
    widen2(left, f);
    widen2(right, g);
    float by = 1.f;
    if constexpr (NORM) {
      uint64_t x = mul2(f[0], f[0]), y = mul2(g[0], g[0]);
#pragma unroll
      for (int e = 1; e < N / 2; ++e) x = fma2(f[e], f[e], x), y = fma2(g[e], g[e], y);
      const float2 sx = unpair(x), sy = unpair(y);
      float sum = (sx.x + sx.y) + (sy.x + sy.y);
      if constexpr (LANES != 0) {
#pragma unroll
        for (int k = 1; k < LANES; k *= 2) sum += __shfl_xor_sync(~0u, sum, k);
      } else {
        float all = 0.f;
        for (int k = 0; k < lanes; ++k) all += __shfl_sync(~0u, sum, lane - mine + k);
        sum = all;
      }
      const int kind = turns ? !query : weights_of;
      if (kind != weights_of) {
        const T *w = reinterpret_cast<const T *>(kind ? p.k_weight : p.q_weight) + one;
        widen2(*reinterpret_cast<const V *>(w), weight);
        widen2(*reinterpret_cast<const V *>(w + apart), weight + N / 2);
        weights_of = kind;
      }
      if (turns) {
        by = rsqrtf(fmaf(sum, reciprocal, p.eps));
#pragma unroll
        for (int e = 0; e < N / 2; ++e) f[e] = mul2(f[e], weight[e]), g[e] = mul2(g[e], weight[N / 2 + e]);
      }
    }
    if (turns && turn_one) {
      if (WITHIN) {
#pragma unroll
        for (int e = 0; e < N / 2; ++e) {
          const float2 x = unpair(f[e]), y = unpair(g[e]);
          f[e] = fma2(f[e], pair_of(c[e], c[e]), mul2(pair_of(x.y, x.x), pair_of(minus[e], s[e])));
          // (by an angle of 0 an infinity that does not turn would make its neighbour NaN)
          if (turn_two) g[e] = fma2(g[e], pair_of(c[N / 2 + e], c[N / 2 + e]), mul2(pair_of(y.y, y.x), pair_of(minus[N / 2 + e], s[N / 2 + e])));
        }
      } else {
#pragma unroll
        for (int e = 0; e < N; e += 2) {
          const uint64_t cosine = pair_of(c[e], c[e + 1]), x = f[e / 2], y = g[e / 2];
          f[e / 2] = fma2(x, cosine, mul2(y, pair_of(minus[e], minus[e + 1])));
          g[e / 2] = fma2(y, cosine, mul2(x, pair_of(s[e], s[e + 1])));
        }
      }
    }
    if (head >= heads) continue;
    if (query) {
      T *to = reinterpret_cast<T *>(a.q_out) + token * a.q_out_stride[0] + head * a.q_out_stride[1] + one;
      V r;
      round2(f, by, r);
      *reinterpret_cast<V *>(to) = r;
      round2(g, by, r);
      *reinterpret_cast<V *>(to + apart) = r;
    } else if (stored) {
      const int kv_head = head - a.q_heads - (turns ? 0 : a.kv_heads);
      C *to = (turns ? reinterpret_cast<C *>(a.k_cache) + k_at + kv_head * a.k_cache_stride[2] : reinterpret_cast<C *>(a.v_cache) + v_at + kv_head * a.v_cache_stride[2]) + one;
      Vec<C, N> r, t;
      if constexpr (SMALL) {
        const int e = p.exponents ? __ldg(reinterpret_cast<const int *>(p.exponents) + kv_head + (turns ? 0 : a.kv_heads)) : 0;
        const float scale = by * __uint_as_float(uint32_t(127 - min(max(e, EMMY_MIN_EXPONENT), EMMY_MAX_EXPONENT)) << 23);
        round2(f, scale, r);
        round2(g, scale, t);
      } else if (turns) {
        round2(f, by, r);
        round2(g, by, t);
      } else {
        r = left, t = right;
      }
      *reinterpret_cast<Vec<C, N> *>(to) = r;
      *reinterpret_cast<Vec<C, N> *>(to + apart) = t;
    }
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

template <typename T, typename C, int N, bool WITHIN, bool NORM> int launch(Params &p, cudaStream_t s) {
  const emmy_rotate_append_args &a = p.a;
  p.lanes = (a.head_dim / N + 1) / 2;
  int sms = 0;
  if (const int e = emmy_internal_sms(&sms)) return failed(static_cast<cudaError_t>(e));
  if constexpr (N > 1 && (NORM || !std::is_same<T, C>::value)) {
    // a token's heads go to more warps where tokens are few: 16 warps an SM at least
    const int groups = (a.q_heads + 2 * a.kv_heads + 32 / p.lanes - 1) / (32 / p.lanes);
    const int64_t wanted = sms * 32;
    const int shares = static_cast<int>(std::min<int64_t>(groups, std::max<int64_t>(1, (wanted + a.tokens - 1) / a.tokens)));
    const dim3 grid((a.tokens + kWarps - 1) / kWarps, shares);
    const size_t smem = size_t(kWarps) * (kGroups * 64 * 16 + a.rotary_dim * sizeof(float));
    if (p.lanes == 4)
      append_kernel<T, C, N, WITHIN, NORM, 4><<<grid, 32 * kWarps, smem, s>>>(p);
    else if (p.lanes == 8)
      append_kernel<T, C, N, WITHIN, NORM, 8><<<grid, 32 * kWarps, smem, s>>>(p);
    else if (p.lanes == 16)
      append_kernel<T, C, N, WITHIN, NORM, 16><<<grid, 32 * kWarps, smem, s>>>(p);
    else
      append_kernel<T, C, N, WITHIN, NORM, 0><<<grid, 32 * kWarps, smem, s>>>(p);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : failed(e);
  } else {
    // heads in shares of equal size, and a few tokens a block where one is small
    const int heads = a.q_heads + 2 * a.kv_heads, most = p.lanes < kThreads ? kThreads / p.lanes : 1;
    const int shares = (heads + most - 1) / most, rows = (heads + shares - 1) / shares;
    int tokens = kThreads / 2 / (p.lanes * rows);
    tokens = tokens < 1 ? 1 : tokens > 64 ? 64 : tokens;
    if (tokens > a.tokens) tokens = a.tokens;
    const int want = (a.tokens + tokens - 1) / tokens;
    int resident = sms * ((NORM ? kNormBlocks : kBlocks) * kThreads / (p.lanes * rows * tokens)) / shares;
    if (resident < 1) resident = 1;
    const dim3 grid(want < resident ? want : resident, shares), block(p.lanes, rows, tokens);
    // angles of two turns; vectors, slots and positions on their way (N > 1): with
    // 256 components and 384 threads 47 KiB, under the 48 that need no asking
    const size_t smem = size_t(tokens) * 2 * a.rotary_dim * sizeof(float) +
                        (N > 1 ? size_t(kAhead) * 2 * p.lanes * rows * tokens * (16 + 4) : 0) +
                        (NORM ? size_t(2) * p.lanes * rows * tokens * sizeof(float) : 0);
    rotate_append_kernel<T, C, N, WITHIN, NORM><<<grid, block, smem, s>>>(p);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : failed(e);
  }
}

// 16-byte accesses need every address and stride to be a multiple of 16 bytes
// and heads, halves and the part that stays to be whole vectors.
template <typename T, typename C, bool NORM> int dispatch(Params &p, cudaStream_t s) {
  constexpr int N = 16 / sizeof(T);
  const emmy_rotate_append_args &a = p.a;
  uint64_t addr = 0;
  int64_t strides = 0;
  if (a.q_heads) {
    addr |= a.q | a.q_out;
    for (int i = 0; i < 2; ++i) strides |= a.q_stride[i] | a.q_out_stride[i];
  }
  if (a.kv_heads) {
    addr |= a.k | a.v | (a.k_cache | a.v_cache) * (sizeof(T) / sizeof(C));     // (N elements of 8 bits are N bytes)
    for (int i = 0; i < 2; ++i) strides |= a.k_stride[i] | a.v_stride[i];
    for (int i = 0; i < 3; ++i) strides |= a.k_cache_stride[i] | a.v_cache_stride[i];
  }
  if (NORM) addr |= (a.q_heads ? p.q_weight : 0) | (a.kv_heads ? p.k_weight : 0);
  const bool whole = addr % 16 == 0 && strides % N == 0 && a.head_dim % (2 * N) == 0;
  // (vectors of angles: 16 bytes of shared memory hold the cosines of 4 pairs)
  if (whole && a.interleaved && a.rotary_dim % N == 0 && a.rotary_dim % 8 == 0) return launch<T, C, N, true, NORM>(p, s);
  if (whole && !a.interleaved && a.rotary_dim / 2 % N == 0) return launch<T, C, N, false, NORM>(p, s);
  return launch<T, C, 1, false, NORM>(p, s);
}

template <typename T> int dispatch(Params &p, bool small, bool norm, cudaStream_t s) {
  if (small) return norm ? dispatch<T, E4M3, true>(p, s) : dispatch<T, E4M3, false>(p, s);
  return norm ? dispatch<T, T, true>(p, s) : dispatch<T, T, false>(p, s);
}

// `name`: the entry's, for messages
int run(const char *name, Params &p, bool small, bool norm, void *stream) {
  const emmy_rotate_append_args *const a = &p.a;
  // 2^shift / page_size rounded up is too large by less than 1, which a slot times that,
  // below 2^shift, forgives
  int log = 0;
  while ((int64_t(1) << log) < a->page_size) ++log;
  p.page_shift = 31 + log;
  p.page_inverse = a->page_size > 0 ? static_cast<uint32_t>(((uint64_t(1) << p.page_shift) + a->page_size - 1) / a->page_size) : 0;
  auto bad = [&](const char *fmt, long x = 0, long y = 0) {
    char with[256];
    snprintf(with, sizeof with, "%s: %s", name, fmt);
    return fail(with, x, y);
  };
  if (a->dtype != 6 && a->dtype != 7 && a->dtype != 9) return bad("dtype %ld (f16, f32 or bf16)", a->dtype);
  if (a->tokens < 0 || a->tokens > (1 << 30) || a->q_heads < 0 || a->kv_heads < 0 || a->q_heads > 1024 || a->kv_heads > 1024)
    return bad("bad count of tokens or heads");
  if (a->head_dim < 1 || a->head_dim > 256) return bad("head_dim %ld outside 1..256", a->head_dim);
  if (a->rotary_dim < 0 || a->rotary_dim > a->head_dim || a->rotary_dim % 2)
    return bad("rotary_dim %ld must be even and at most head_dim %ld", a->rotary_dim, a->head_dim);
  if (a->axes < 1 || a->axes > 16) return bad("%ld position axes (1..16)", a->axes);
  if (a->kv_heads && (a->pages < 0 || a->page_size < 1)) return bad("a cache of %ld pages of %ld tokens", a->pages, a->page_size);
  if (norm && !(p.eps >= 0.f)) return bad("eps must not be negative");
  if (a->tokens == 0 || (a->q_heads == 0 && a->kv_heads == 0)) return 0;
  if ((a->q_heads && (!a->q || !a->q_out)) ||
      (a->kv_heads && (!a->k || !a->v || !a->slots || (a->pages && (!a->k_cache || !a->v_cache)))) ||
      (a->rotary_dim && (!a->positions || !a->frequencies)) ||
      (norm && ((a->q_heads && !p.q_weight) || (a->kv_heads && !p.k_weight))))
    return bad("null address");
  const uint64_t elements = (a->q_heads ? a->q | a->q_out : 0) | (a->kv_heads ? a->k | a->v : 0) |
                            (a->kv_heads && !small ? a->k_cache | a->v_cache : 0) |
                            (norm ? (a->q_heads ? p.q_weight : 0) | (a->kv_heads ? p.k_weight : 0) : 0);
  if (elements % (a->dtype == 7 ? 4 : 2) || (a->kv_heads ? (a->slots | p.exponents) % 4 : 0) ||
      (a->rotary_dim ? (a->positions | a->frequencies | a->pair_axis) % 4 : 0))
    return bad("address not a multiple of its element's size");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->dtype == 6) return dispatch<__half>(p, small, norm, s);
  if (a->dtype == 7) return dispatch<float>(p, small, norm, s);
  return dispatch<__nv_bfloat16>(p, small, norm, s);
}

}  // namespace

extern "C" EMMY_API int emmy_rotate_append(const emmy_rotate_append_args *a, void *stream) {
  if (!a) return fail("emmy_rotate_append: bad argument");
  Params p{};
  p.a = *a;
  return run("emmy_rotate_append", p, false, false, stream);
}

extern "C" EMMY_API int emmy_norm_rotate_append(const emmy_norm_rotate_append_args *a, void *stream) {
  if (!a) return fail("emmy_norm_rotate_append: bad argument");
  if (a->cache_bits8 != 0 && a->cache_bits8 != 1) return fail("emmy_norm_rotate_append: cache_bits8 %ld (0 or 1)", a->cache_bits8);
  Params p{};
  p.a = a->a;
  p.q_weight = a->q_weight;
  p.k_weight = a->k_weight;
  p.eps = a->eps;
  p.exponents = a->cache_bits8 ? a->exponents : 0;
  return run("emmy_norm_rotate_append", p, a->cache_bits8 != 0, a->q_weight || a->k_weight, stream);
}
