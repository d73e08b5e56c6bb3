// emmy_quantised_attention.cu -- attention over a paged cache of 8-bit floats.
//
//   s_j = scale 2^e q.k_j,  o = 2^f sum_j p_j v_j / l,  p_j = 2^(c (s_j - m)),  l = sum_j p_j
//
// with the powers of two of a head's keys and values (e, f) outside the products.
//
// Few query rows of a key head (decoding, drafted tokens): bound by reading the cache.
// A warp takes slices of 16 keys on its own: it copies their 8-bit rows to its ring of
// shared memory some slices ahead, widens them to f16 in registers -- every 8-bit
// float is an f16 -- and multiplies with mma.sync, which has no bytes of f16 to fetch
// from shared memory: 6 KiB a slice of 128 components instead of 20 with 16-bit tiles
// written back for tcgen05, whose throughput 8 rows could not use (a slice's products
// take 120 cycles of the 700 that its bytes take to arrive).
//
// The products are transposed, S^T = K Q^T and O^T = V^T P^T, so that keys and
// components fill the 16 rows of an instruction and 8 query rows its columns.  What a
// thread holds of S^T goes to P^T by movmatrix.  Neither keys nor components have to
// be in order within a sum, so a thread reads 16 bytes of a row at once: component
// order is permuted alike in K and Q, and key order (row r of S^T is key
// 4 (r & 1) + (r >> 1 & 3) + (r & 8)) so that the rows of V that a thread pairs by
// bytes lie without bank conflicts.
//
// Queries of any 16-bit type become f16 with a power of two that brings the row's
// largest to 2^14..2^15: exact for components down to 2^-29 of it, and within 2^-40 of
// it below, far under the rounding of the sums in 32 bits.  Weights are rounded to
// f16; they start at 2^6 and grow to 2^14 before the base moves, so that small ones
// keep their bits.
//
// Many rows: bound by the tensor cores.  The keys are read back to 16 bits once, into
// pages of 128 tokens (unscaled values, exact in either type; read_back_kernel), and go
// through the 16-bit cache's tcgen05 attention.
#include "emmy_quantised.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include <cstdint>
#include <cstdio>

int emmy_internal_fail(int code, const char *msg);   // emmy_runtime.cpp

using namespace emmy_quantised;

namespace {

constexpr float kNoMax = -FLT_MAX;      // base of a row that has seen no key
constexpr float kShift = 6.f, kGrow = 8.f;      // log2 of the weight at the base, and growth before it moves
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Params {
  const Piece *pieces;
  const int *cta_first;
  unsigned *counters;
  const int *table, *exponents;
  const uint8_t *k, *v;
  const void *q;
  void *out;
  float *lse, *part_o;
  float2 *part_ml;
  int64_t table_stride, q_stride[2], out_stride[2], k_stride[3], v_stride[3];
  int pages, page_size, page_shift;       // key / page_size = key * page_inverse >> page_shift
  uint32_t page_inverse;
  int q_heads, kv_heads, group, group_inverse, causal, window, bf16;
  float scale_log2;
};

// NT: tiles of 8 query rows
template <int D, int NT> struct Shape {
  static constexpr int kWarps = NT == 1 ? 8 : 4, kThreads = 32 * kWarps;
  static constexpr int kHalf = kSlice * D, kStage = 2 * kHalf;             // bytes: keys, then values
  static constexpr int kStages = (NT == 1 ? 3 : 5) * (128 / D);            // slices of a warp in flight or in use
  static constexpr int kSteps = D / 16;                                    // products of 16 components
  static constexpr int kRounds = D / 32;                                   // of 4 of a thread's components, at a unit's end
  static constexpr int kAtOnce = NT == 1 ? 2 : 1;                          // rounds between two barriers
  static constexpr int kQuery = kWarps * kStages * kStage;                 // offsets: f16 queries (NT > 1)
  static constexpr int kJoin = kQuery + (NT > 1 ? NT * kSteps * 256 : 0);  // the warps' parts of a round
  static constexpr int kSums = kJoin + kWarps * NT * 1024 * kAtOnce;       // (base, sum) of a warp's rows
  static constexpr int kScales = kSums + kWarps * NT * 8 * 8;              // c of each row
  static constexpr int kFlag = kScales + NT * 8 * 4, kBytes = kFlag + 16;
  static_assert(2 * (kBytes + 1024) <= 228 * 1024, "two CTAs an SM");
};

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
// 16 bytes, or zeros without reading
__device__ __forceinline__ void copy_or_zero(uint32_t to, const void *from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void load4(uint32_t at, uint32_t *r) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void load2(uint32_t at, uint32_t *r) {
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(at) : "memory");
}
// the two 8-bit floats of a word's lower or upper half
__device__ __forceinline__ uint32_t widen_low(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t widen_high(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ void mma(float *d, const uint32_t *a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t r) {
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %0;" : "+r"(r));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(uint32_t(e + 127) << 23); }       // -126..127
__device__ __forceinline__ int exponent_of(const Params &p, int which, int head) {
  return p.exponents ? min(max(__ldg(p.exponents + which * p.kv_heads + head), EMMY_MIN_EXPONENT), EMMY_MAX_EXPONENT) : 0;
}
// Reciprocal of a row's sum: 0 for a row that saw no key, NaN stays.
__device__ __forceinline__ float reciprocal(float l) { return l > 0.f ? __frcp_rn(l) : l; }
__device__ __forceinline__ float log_sum(float m, float c, float l) {
  return l > 0.f ? (__fmul_rn(m, c) - kShift + log2f(l)) * kLn2 : (l == 0.f ? -INFINITY : l);
}
// what a sum over base m weighs over base `top`
__device__ __forceinline__ float weight(float m, float top, float c) { return m == top ? 1.f : exp2_approx((m - top) * c); }

__device__ __forceinline__ Piece read_piece(const Params &p, int i) {
  Piece u;
  const int4 *at = reinterpret_cast<const int4 *>(p.pieces + i);
  int4 *to = reinterpret_cast<int4 *>(&u);
#pragma unroll
  for (int k = 0; k < 4; ++k) to[k] = __ldg(at + k);
  return u;
}

// What a warp copies next: slices first_slice + warp, + warp + kWarps, .. of a piece,
// then those of the next piece.
template <int D, int NT> struct Feed {
  using S = Shape<D, NT>;
  static constexpr int kLanes = D / 16, kKeys = kSlice * kLanes / 32;    // lanes of a row; rows of a lane
  const Params &p;
  int piece, last, slice, end, lo, hi;      // slices of the whole sequence
  const int *row;
  const uint8_t *k, *v;
  int page[kKeys];                   // of the slice to come; -1: nothing to read

  __device__ __forceinline__ int key(int i) const { return slice * kSlice + (threadIdx.x % 32) / kLanes + i * (32 / kLanes); }
  __device__ __forceinline__ int page_of(int key) const { return static_cast<int>(uint64_t(key) * p.page_inverse >> p.page_shift); }
  __device__ __forceinline__ void enter(int warp) {      // the first piece from `piece` on with a slice for this warp
    for (; piece < last; ++piece) {
      const Piece u = read_piece(p, piece);
      if (warp >= u.nslices) continue;
      slice = u.slice0 + warp;
      end = u.slice0 + u.nslices;
      lo = u.lo;
      hi = u.hi;
      row = p.table + u.seq * p.table_stride;
      k = p.k + u.kvh * p.k_stride[2];
      v = p.v + u.kvh * p.v_stride[2];
      break;
    }
  }
  __device__ __forceinline__ void look_up() {
    if (piece >= last) return;
#pragma unroll
    for (int i = 0; i < kKeys; ++i) {
      const int at = key(i);
      page[i] = at >= lo && at < hi ? __ldg(row + page_of(at)) : -1;
    }
  }
  __device__ __forceinline__ Feed(const Params &params, int first, int end_piece, int warp) : p(params), piece(first), last(end_piece) {
    enter(warp);
    look_up();
  }
  // copies the slice to `stage` (keys in the rows of S^T, with the 16-byte pieces of a
  // row in an order of its own for the reads below) and looks the next one's pages up
  __device__ __forceinline__ void next(uint32_t stage, int warp) {
    if (piece < last) {
      const int lane = threadIdx.x % 32, chunk = lane % kLanes;
#pragma unroll
      for (int i = 0; i < kKeys; ++i) {
        const int j = lane / kLanes + i * (32 / kLanes), at = key(i);
        const bool there = page[i] >= 0 && page[i] < p.pages;
        const int64_t pg = there ? page[i] : 0, token = there ? at - page_of(at) * p.page_size : 0;
        const int r = 2 * (j & 3) + (j >> 2 & 1) + (j & 8);
        const int k_chunk = D == 128 ? chunk ^ (r & 1) << 2 : chunk, v_chunk = D == 128 ? chunk ^ (j & 3) << 1 : chunk ^ (j >> 1 & 1) << 1;
        copy_or_zero(stage + r * D + k_chunk * 16, k + pg * p.k_stride[0] + token * p.k_stride[1] + chunk * 16, there);
        copy_or_zero(stage + S::kHalf + j * D + v_chunk * 16, v + pg * p.v_stride[0] + token * p.v_stride[1] + chunk * 16, there);
      }
      slice += S::kWarps;
      if (slice >= end) {
        ++piece;
        enter(warp);
      }
      look_up();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
};

template <int D, int NT>
__global__ void __launch_bounds__(Shape<D, NT>::kThreads, 2) few_rows_kernel(const __grid_constant__ Params p) {
  using S = Shape<D, NT>;
  constexpr int W = S::kWarps, DP = D / 8;          // DP: components of a thread
  extern __shared__ __align__(128) char raw[];
  const uint32_t base = smem_addr(raw);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int first = __ldg(p.cta_first + blockIdx.x), last = __ldg(p.cta_first + blockIdx.x + 1);
  const uint32_t ring = base + warp * S::kStages * S::kStage;
  float *const scales = reinterpret_cast<float *>(raw + S::kScales);
  float2 *const sums = reinterpret_cast<float2 *>(raw + S::kSums);
  volatile int *const flag = reinterpret_cast<volatile int *>(raw + S::kFlag);

  Feed<D, NT> feed(p, first, last, warp);
  int stage = 0;                      // the slice in use; those after it are on their way
#pragma unroll 1
  for (int k = 0; k + 1 < S::kStages; ++k) feed.next(ring + k * S::kStage, warp);

  for (int i = first; i < last; ++i) {
    const Piece u = read_piece(p, i);
    const int tiles = NT == 1 ? 1 : (u.rows + 7) / 8;
    // ------------------------------------------------------------ queries
    uint32_t q[NT == 1 ? 2 * S::kSteps : 1];
    float c[NT == 1 ? 2 : 1];
    if (NT == 1 || warp < tiles) {
      const int r = (NT == 1 ? 0 : 8 * warp) + g;
      uint32_t w[2 * S::kSteps];
      float top = 0.f;
      const int at = u.row0 + min(r, u.rows - 1), token = at * p.group_inverse >> 16, head = u.kvh * p.group + at - token * p.group;
      const uint16_t *src = static_cast<const uint16_t *>(p.q) + (u.tok0 + token) * p.q_stride[0] + head * p.q_stride[1] + 16 * t;
#pragma unroll
      for (int k = 0; k < 2 * S::kSteps; k += 4) {
        const uint4 x = *reinterpret_cast<const uint4 *>(src + 2 * k + (k >= 8 ? 48 : 0));      // (64 + 16 t on)
        w[k] = x.x, w[k + 1] = x.y, w[k + 2] = x.z, w[k + 3] = x.w;
      }
      auto both = [&](uint32_t x) {
        if (p.bf16) return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
        return __half22float2(*reinterpret_cast<__half2 *>(&x));
      };
#pragma unroll
      for (int k = 0; k < 2 * S::kSteps; ++k) {
        const float2 f = both(w[k]);
        top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
      }
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
      const int up = top == 0.f ? 0 : min(14 - (int(__float_as_uint(top) >> 23) - 127), 120);
      const float by = power_of_two(up);
#pragma unroll
      for (int k = 0; k < 2 * S::kSteps; ++k) {
        const float2 f = both(w[k]);
        w[k] = pack_f16(f.x * by, f.y * by);
      }
      // (finite and not 0: a difference of scores of 0, or one that is infinite, stays what it is)
      const float of_row = fminf(fmaxf(ldexpf(p.scale_log2, exponent_of(p, 0, u.kvh) - up), FLT_MIN), FLT_MAX);
      if (NT == 1) {
#pragma unroll
        for (int k = 0; k < 2 * S::kSteps; ++k) q[NT == 1 ? k : 0] = w[k];
        c[0] = __shfl_sync(~0u, of_row, 8 * t);
        c[NT == 1 ? 1 : 0] = __shfl_sync(~0u, of_row, 8 * t + 4);
        if (warp == 0 && t == 0) scales[r] = of_row;
      } else {
#pragma unroll
        for (int s = 0; s < S::kSteps; ++s)
          asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(base + S::kQuery + ((warp * S::kSteps + s) * 32 + lane) * 8), "r"(w[2 * s]), "r"(w[2 * s + 1]) : "memory");
        if (t == 0) scales[r] = of_row;
      }
    }
    if (NT > 1) __syncthreads();
    auto scale_of = [&](int nt, int e) { return NT == 1 ? c[NT == 1 ? e : 0] : scales[8 * nt + 2 * t + e]; };
    // the keys that this thread's row 2 t + e of a tile sees; rows after the last take its place
    auto seen_by = [&](int nt, int e, int &lo, int &hi) {
      const int at = u.row0 + min(8 * nt + 2 * t + e, u.rows - 1), pos = u.pos0 + (at * p.group_inverse >> 16);
      hi = p.causal ? min(u.kv_len, pos + 1) : u.kv_len;
      lo = p.window ? max(0, pos - p.window + 1) : 0;
    };
    // every row sees the keys between
    int min_hi, max_lo;
    {
      const int from = u.pos0 + (u.row0 * p.group_inverse >> 16), to = u.pos0 + ((u.row0 + u.rows - 1) * p.group_inverse >> 16);
      min_hi = p.causal ? min(u.kv_len, from + 1) : u.kv_len;
      max_lo = p.window ? max(0, to - p.window + 1) : 0;
    }

    float o[NT][S::kSteps][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int k = 0; k < S::kSteps; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][k][e] = 0.f;
      m[nt][0] = m[nt][1] = kNoMax;
      l[nt][0] = l[nt][1] = 0.f;
    }
#pragma unroll 1
    for (int slice = u.slice0 + warp; slice < u.slice0 + u.nslices; slice += W) {
      asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 2) : "memory");
      __syncwarp();
      const uint32_t keys = ring + stage * S::kStage, values = keys + S::kHalf;
      feed.next(ring + (stage ? stage - 1 : S::kStages - 1) * S::kStage, warp);
      stage = stage + 1 == S::kStages ? 0 : stage + 1;

      // ---------------------------------------------------------- S^T = K Q^T
      float s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
      for (int h = 0; h < D / 64; ++h) {
        const uint32_t at = keys + g * D + (D == 128 ? (4 * h + t) ^ (g & 1) << 2 : t) * 16;
        uint32_t x[4], y[4];
        load4(at, x);
        load4(at + 8 * D, y);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t a[4] = {widen_low(x[k]), widen_low(y[k]), widen_high(x[k]), widen_high(y[k])};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if (NT > 1 && nt >= tiles) break;
            uint32_t b[2];
            if (NT == 1)
              b[0] = q[NT == 1 ? 2 * (4 * h + k) : 0], b[1] = q[NT == 1 ? 2 * (4 * h + k) + 1 : 0];
            else
              load2(base + S::kQuery + ((nt * S::kSteps + 4 * h + k) * 32 + lane) * 8, b);
            mma(s[nt], a, b[0], b[1]);
          }
        }
      }

      // ---------------------------------------------------------- softmax
      const int key0 = slice * kSlice;
      if (key0 < max_lo || key0 + kSlice > min_hi) {
        const int key = key0 + (g >> 1 & 3) + 4 * (g & 1);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (NT > 1 && nt >= tiles) break;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            int lo, hi;
            seen_by(nt, e, lo, hi);
            if (key < lo || key >= hi) s[nt][e] = -INFINITY;
            if (key + 8 < lo || key + 8 >= hi) s[nt][2 + e] = -INFINITY;
          }
        }
      }
      // the base follows the largest score when that has grown by more than 2^8
      bool grown = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (NT > 1 && nt >= tiles) break;
#pragma unroll
        for (int e = 0; e < 2; ++e) grown |= (fmaxf(s[nt][e], s[nt][2 + e]) - m[nt][e]) * scale_of(nt, e) > kGrow;
      }
      if (__any_sync(~0u, grown)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (NT > 1 && nt >= tiles) break;
          float by[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = fmaxf(s[nt][e], s[nt][2 + e]);
            top = fmaxf(top, __shfl_xor_sync(~0u, top, 4));
            top = fmaxf(top, __shfl_xor_sync(~0u, top, 8));
            top = fmaxf(fmaxf(top, __shfl_xor_sync(~0u, top, 16)), m[nt][e]);
            by[e] = weight(m[nt][e], top, scale_of(nt, e));
            m[nt][e] = top;
            l[nt][e] *= by[e];
          }
#pragma unroll
          for (int k = 0; k < S::kSteps; ++k) o[nt][k][0] *= by[0], o[nt][k][1] *= by[1], o[nt][k][2] *= by[0], o[nt][k][3] *= by[1];
        }
      }
      uint32_t w[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (NT > 1 && nt >= tiles) break;
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = exp2_approx(fmaf(s[nt][e] - m[nt][e & 1], scale_of(nt, e & 1), kShift));
        l[nt][0] += x[0] + x[2];
        l[nt][1] += x[1] + x[3];
        w[nt][0] = transposed(pack_f16(x[0], x[1]));
        w[nt][1] = transposed(pack_f16(x[2], x[3]));
      }

      // ---------------------------------------------------------- O^T += V^T P^T
      uint32_t v[4][DP / 4];           // of keys t, t + 4, t + 8, t + 12
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t row = values + (t + 4 * j) * D;
        if (D == 128)
          load4(row + (g ^ t << 1) * 16, v[j]);
        else
          load2(row + (g / 2 ^ (t >> 1) << 1) * 16 + (g & 1) * 8, v[j]);
      }
#pragma unroll
      for (int k = 0; k < DP / 4; ++k) {
        const uint32_t p0 = __byte_perm(v[0][k], v[1][k], 0x5140), p1 = __byte_perm(v[0][k], v[1][k], 0x7362);
        const uint32_t p2 = __byte_perm(v[2][k], v[3][k], 0x5140), p3 = __byte_perm(v[2][k], v[3][k], 0x7362);
        const uint32_t a[4] = {widen_low(p0), widen_high(p0), widen_low(p2), widen_high(p2)};
        const uint32_t b[4] = {widen_low(p1), widen_high(p1), widen_low(p3), widen_high(p3)};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (NT > 1 && nt >= tiles) break;
          mma(o[nt][2 * k], a, w[nt][0], w[nt][1]);
          mma(o[nt][2 * k + 1], b, w[nt][0], w[nt][1]);
        }
      }
    }

    // ------------------------------------------------------------ the piece's end
    // a thread has components DP g to DP g + DP - 1 of rows 2 t and 2 t + 1 of a tile
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[nt][e] += __shfl_xor_sync(~0u, l[nt][e], 4);
        l[nt][e] += __shfl_xor_sync(~0u, l[nt][e], 8);
        l[nt][e] += __shfl_xor_sync(~0u, l[nt][e], 16);
        if (g == 0) sums[warp * NT * 8 + 8 * nt + 2 * t + e] = make_float2(m[nt][e], l[nt][e]);
      }
    __syncthreads();
    // (base, sum) of a row over all warps
    auto joined = [&](int r, float scale) {
      float2 all = make_float2(kNoMax, 0.f);
#pragma unroll
      for (int w = 0; w < W; ++w) all.x = fmaxf(all.x, sums[w * NT * 8 + r].x);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float2 x = sums[w * NT * 8 + r];
        all.y += weight(x.x, all.x, scale) * x.y;
      }
      return all;
    };
    const bool split = u.nsplit > 1;
    const int64_t part = u.part_row + int64_t(u.split) * u.rows;
    const float unscaled = power_of_two(exponent_of(p, 1, u.kvh));
    if (threadIdx.x < u.rows) {
      const int r = threadIdx.x;
      const float2 all = joined(r, scales[r]);
      if (split) {
        __stcg(p.part_ml + part + r, all);
      } else if (p.lse) {
        const int at = u.row0 + r, token = at * p.group_inverse >> 16;
        p.lse[int64_t(u.tok0 + token) * p.q_heads + u.kvh * p.group + at - token * p.group] = log_sum(all.x, scales[r], all.y);
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (NT > 1 && nt >= tiles) break;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * nt + 2 * t + e;
        const float2 all = joined(r, scale_of(nt, e));
        const float by = weight(m[nt][e], all.x, scale_of(nt, e)) * (split ? 1.f : reciprocal(all.y) * unscaled);
#pragma unroll
        for (int k = 0; k < S::kSteps; ++k) o[nt][k][e] *= by, o[nt][k][2 + e] *= by;
      }
    }
    const uint32_t join = base + S::kJoin;
#pragma unroll
    for (int from = 0; from < S::kRounds; from += S::kAtOnce) {
      if (from) __syncthreads();
#pragma unroll
      for (int a = 0; a < S::kAtOnce; ++a)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = 8 * nt + 2 * t + e, k = 2 * (from + a);
            const uint32_t to = join + (((warp * S::kAtOnce + a) * NT * 8 + r) * 8 + (g ^ t << 1)) * 16;
            asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(o[nt][k][e]), "f"(o[nt][k][2 + e]), "f"(o[nt][k + 1][e]), "f"(o[nt][k + 1][2 + e]) : "memory");
          }
      __syncthreads();
      for (int item = threadIdx.x; item < u.rows * 8 * S::kAtOnce; item += S::kThreads) {
        const int a = item / (u.rows * 8), r = item / 8 - a * u.rows, of = item % 8;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; ++w) {
          float4 x;
          const uint32_t at = join + (((w * S::kAtOnce + a) * NT * 8 + r) * 8 + (of ^ (r >> 1 & 3) << 1)) * 16;
          asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(at) : "memory");
          sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
        }
        const int component = DP * of + 4 * (from + a);
        if (split) {
          __stcg(reinterpret_cast<float4 *>(p.part_o + (part + r) * D + component), sum);
        } else {
          const int at = u.row0 + r, token = at * p.group_inverse >> 16;
          uint16_t *to = static_cast<uint16_t *>(p.out) + (u.tok0 + token) * p.out_stride[0] + (u.kvh * p.group + at - token * p.group) * p.out_stride[1] + component;
          *reinterpret_cast<uint2 *>(to) = p.bf16 ? make_uint2(pack_bf16(sum.x, sum.y), pack_bf16(sum.z, sum.w)) : make_uint2(pack_f16(sum.x, sum.y), pack_f16(sum.z, sum.w));
        }
      }
    }
    if (split) {
      // the CTA that arrives last joins the parts, in their order
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        unsigned *counter = p.counters + u.item;
        const bool is_last = atomicAdd(counter, 1u) == unsigned(u.nsplit - 1);
        if (is_last) *counter = 0;
        __threadfence();
        *flag = is_last;
      }
      __syncthreads();
      if (*flag) {
        for (int item = threadIdx.x; item < u.rows * (D / 4); item += S::kThreads) {
          const int r = item / (D / 4), component = item % (D / 4) * 4;
          const int64_t row = u.part_row + r;
          const float scale = scales[r];
          float top = kNoMax, total = 0.f;
#pragma unroll 8
          for (int k = 0; k < u.nsplit; ++k) top = fmaxf(top, __ldcg(p.part_ml + row + int64_t(k) * u.rows).x);
          float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
          for (int k = 0; k < u.nsplit; ++k) {
            const float2 ml = __ldcg(p.part_ml + row + int64_t(k) * u.rows);
            const float4 x = __ldcg(reinterpret_cast<const float4 *>(p.part_o + (row + int64_t(k) * u.rows) * D + component));
            const float by = weight(ml.x, top, scale);
            total += by * ml.y;
            sum.x += by * x.x, sum.y += by * x.y, sum.z += by * x.z, sum.w += by * x.w;
          }
          const float inv = reciprocal(total) * unscaled;
          const int at = u.row0 + r, token = at * p.group_inverse >> 16, head = u.kvh * p.group + at - token * p.group;
          uint16_t *to = static_cast<uint16_t *>(p.out) + (u.tok0 + token) * p.out_stride[0] + head * p.out_stride[1] + component;
          *reinterpret_cast<uint2 *>(to) = p.bf16 ? make_uint2(pack_bf16(sum.x * inv, sum.y * inv), pack_bf16(sum.z * inv, sum.w * inv))
                                                  : make_uint2(pack_f16(sum.x * inv, sum.y * inv), pack_f16(sum.z * inv, sum.w * inv));
          if (component == 0 && p.lse) p.lse[int64_t(u.tok0 + token) * p.q_heads + head] = log_sum(top, scale, total);
        }
      }
    }
    __syncthreads();      // sums, scales and queries have been read
  }
}

struct ReadParams {
  const Job *jobs;
  const int *table, *exponents;
  const uint8_t *k, *v;
  uint16_t *k_out, *v_out;              // [page][head][kBlock][D]
  int64_t table_stride, k_stride[3], v_stride[3];
  int pages, page_size, page_shift;
  uint32_t page_inverse;
  int kv_heads, bf16;
};

// One job's keys or values of a head, blockIdx = (job, head, keys or values); 16 bytes
// a thread at once.
template <int D> __global__ void __launch_bounds__(256) read_back_kernel(const __grid_constant__ ReadParams p) {
  const int4 words = __ldg(reinterpret_cast<const int4 *>(p.jobs) + blockIdx.x);
  const Job job{words.x, words.y, words.z, words.w};
  const int head = blockIdx.y;
  const bool value = blockIdx.z;
  const uint8_t *const from = value ? p.v + head * p.v_stride[2] : p.k + head * p.k_stride[2];
  const int64_t page_step = value ? p.v_stride[0] : p.k_stride[0], token_step = value ? p.v_stride[1] : p.k_stride[1];
  uint16_t *const to = (value ? p.v_out : p.k_out) + (int64_t(job.page) * p.kv_heads + head) * kBlock * D;
  const int e = p.exponents ? min(max(__ldg(p.exponents + (value ? p.kv_heads : 0) + head), EMMY_MIN_EXPONENT), EMMY_MAX_EXPONENT) : 0;
  const float by = power_of_two(e);
  const int *const row = p.table + job.seq * p.table_stride;
#pragma unroll
  for (int i = threadIdx.x; i < kBlock * (D / 16); i += 256) {
    const int token = i / (D / 16), chunk = i % (D / 16), key = job.first + token;
    if (token >= job.count) break;
    const int index = static_cast<int>(uint64_t(key) * p.page_inverse >> p.page_shift), page = __ldg(row + index);
    uint32_t in[4] = {0, 0, 0, 0}, out[8];
    if (page >= 0 && page < p.pages) {
      const uint4 x = __ldg(reinterpret_cast<const uint4 *>(from + page * page_step + (key - index * p.page_size) * token_step + chunk * 16));
      in[0] = x.x, in[1] = x.y, in[2] = x.z, in[3] = x.w;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t two = k % 2 ? widen_high(in[k / 2]) : widen_low(in[k / 2]);
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&two));
      out[k] = p.bf16 ? pack_bf16(f.x * by, f.y * by) : pack_f16(f.x * by, f.y * by);
    }
    uint4 *dst = reinterpret_cast<uint4 *>(to + token * D + chunk * 16);
    dst[0] = make_uint4(out[0], out[1], out[2], out[3]);
    dst[1] = make_uint4(out[4], out[5], out[6], out[7]);
  }
}

// ---------------------------------------------------------------- host
int fail(const char *fmt, long a = 0, long b = 0) {
  char buf[256];
  snprintf(buf, sizeof buf, fmt, a, b);
  return emmy_internal_fail(EMMY_EINVAL, buf);
}
int cuda_fail(const char *what, cudaError_t e) {
  char buf[256];
  snprintf(buf, sizeof buf, "%s: %s", what, cudaGetErrorString(e));
  return emmy_internal_fail(static_cast<int>(e), buf);
}

bool bad_stride(int64_t stride, int64_t extent, int grid) {
  return extent != 1 && (stride <= 0 || stride % grid || stride >= (int64_t(1) << 38));
}

template <int D, int NT> int launch(const Params &p, int ctas, cudaStream_t s) {
  using S = Shape<D, NT>;
  static std::atomic<uint64_t> ready{0};     // a bit for each device
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return cuda_fail("emmy_quantised_attention: cudaGetDevice", e);
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (dev > 63 || !(ready.load() & bit)) {
    if (cudaError_t e = cudaFuncSetAttribute(few_rows_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes))
      return cuda_fail("emmy_quantised_attention: shared memory", e);
    if (dev <= 63) ready.fetch_or(bit);
  }
  few_rows_kernel<D, NT><<<ctas, S::kThreads, S::kBytes, s>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : cuda_fail("emmy_quantised_attention: launch", e);
}

}  // namespace

extern "C" EMMY_API int emmy_quantised_attention(emmy_quantised_plan_t plan, const emmy_quantised_attention_args *args, void *stream) {
  if (!plan || !args) return fail("emmy_quantised_attention: bad argument");
  const emmy_paged_attention_args *a = &args->a;
  if (a->dtype != 6 && a->dtype != 9) return fail("emmy_quantised_attention: dtype %ld (f16 or bf16)", a->dtype);
  if (!(a->scale > 0.f) || !std::isfinite(a->scale * kLog2e)) return fail("emmy_quantised_attention: scale must be positive and finite");
  if (plan->tokens == 0) return 0;
  const bool reads = plan->reads;
  if (a->page_size < 1 || a->page_size > (1 << 30)) return fail("emmy_quantised_attention: page_size %ld (1 or more)", a->page_size);
  if (a->pages < (reads ? 1 : 0)) return fail("emmy_quantised_attention: a cache of %ld pages", a->pages);
  if (a->table_width < 0 || int64_t(a->table_width) * a->page_size < plan->max_kv)
    return fail("emmy_quantised_attention: a table of %ld pages a sequence does not hold %ld tokens", a->table_width, plan->max_kv);
  const bool scratch = plan->part_rows || (plan->others && (plan->others->part_rows || plan->workspace_pages));
  if (!a->q || !a->out || (reads && (!a->k_cache || !a->v_cache || !a->table)) || !a->plan_words || (scratch && !a->scratch))
    return fail("emmy_quantised_attention: null address");
  if ((a->q | a->out | a->k_cache | a->v_cache | a->plan_words) % 16 || a->scratch % 128 || (a->table | a->lse | args->exponents) % 4)
    return fail("emmy_quantised_attention: address not a multiple of 16 bytes (scratch: 128)");
  const int64_t extent[3] = {a->pages, a->page_size, plan->kv_heads};
  for (int i = 0; i < 3 && reads; ++i)
    if (bad_stride(a->k_cache_stride[i], extent[i], 16) || bad_stride(a->v_cache_stride[i], extent[i], 16))
      return fail("emmy_quantised_attention: cache stride %ld not a positive multiple of 16 elements", i);
  const int64_t rows[2] = {plan->tokens, plan->q_heads};
  for (int i = 0; i < 2; ++i)
    if (bad_stride(a->q_stride[i], rows[i], 8) || bad_stride(a->out_stride[i], rows[i], 8))
      return fail("emmy_quantised_attention: q or out stride %ld not a positive multiple of 8 elements", i);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int d = plan->head_dim;
  int *words = reinterpret_cast<int *>(a->plan_words);
  char *scratch_at = reinterpret_cast<char *>(a->scratch);
  auto whole = [](size_t bytes) { return (bytes + 127) / 128 * 128; };
  const size_t row = (d + 2) * sizeof(float);
  // key * inverse >> shift is key / page_size for keys up to 2^30: 2^shift / page_size
  // rounded up is too large by less than 1, which key times that, under 2^shift, forgives
  int log = 0;
  while ((int64_t(1) << log) < a->page_size) ++log;
  const int shift = 30 + log;
  const uint32_t inverse = static_cast<uint32_t>(((uint64_t(1) << shift) + a->page_size - 1) / a->page_size);

  if (plan->at.ctas) {
    Params p{};
    p.cta_first = words;
    p.counters = reinterpret_cast<unsigned *>(words + plan->at.counters);
    p.pieces = reinterpret_cast<const Piece *>(words + plan->at.pieces);
    p.table = reinterpret_cast<const int *>(a->table);
    p.exponents = reinterpret_cast<const int *>(args->exponents);
    p.k = reinterpret_cast<const uint8_t *>(a->k_cache);
    p.v = reinterpret_cast<const uint8_t *>(a->v_cache);
    p.q = reinterpret_cast<const void *>(a->q);
    p.out = reinterpret_cast<void *>(a->out);
    p.lse = reinterpret_cast<float *>(a->lse);
    p.part_o = reinterpret_cast<float *>(scratch_at);
    p.part_ml = reinterpret_cast<float2 *>(p.part_o + plan->part_rows * d);
    p.table_stride = a->table_stride;
    for (int i = 0; i < 2; ++i) p.q_stride[i] = a->q_stride[i], p.out_stride[i] = a->out_stride[i];
    for (int i = 0; i < 3; ++i) p.k_stride[i] = a->k_cache_stride[i], p.v_stride[i] = a->v_cache_stride[i];
    p.pages = a->pages;
    p.page_size = a->page_size;
    p.page_shift = shift;
    p.page_inverse = inverse;
    p.q_heads = plan->q_heads;
    p.kv_heads = plan->kv_heads;
    p.group = plan->q_heads / plan->kv_heads;
    p.group_inverse = (65536 + p.group - 1) / p.group;
    p.causal = plan->causal;
    p.window = plan->window;
    p.bf16 = a->dtype == 9;
    p.scale_log2 = a->scale * kLog2e;
    const int n = plan->at.ctas;
    const int e = d == 128 ? (plan->tiles == 1 ? launch<128, 1>(p, n, s) : launch<128, 4>(p, n, s))
                           : (plan->tiles == 1 ? launch<64, 1>(p, n, s) : launch<64, 4>(p, n, s));
    if (e) return e;
  }
  if (!plan->others) return 0;
  emmy_paged_attention_args b = *a;
  const size_t at_others = whole(plan->part_rows * row), at_workspace = at_others + whole(plan->others->part_rows * row);
  const int64_t page = int64_t(kBlock) * plan->kv_heads * d;
  b.page_size = kBlock;
  b.pages = static_cast<int32_t>(plan->workspace_pages);
  b.table_width = plan->table_width;
  b.table = reinterpret_cast<uint64_t>(words + plan->at.table);
  b.table_stride = plan->table_width;
  b.plan_words = reinterpret_cast<uint64_t>(words + plan->at.others);
  b.scratch = a->scratch + at_others;
  b.k_cache = a->scratch + at_workspace;
  b.v_cache = b.k_cache + plan->workspace_pages * page * 2;
  const int64_t strides[3] = {page, d, int64_t(kBlock) * d};
  for (int i = 0; i < 3; ++i) b.k_cache_stride[i] = b.v_cache_stride[i] = strides[i];
  if (plan->n_jobs) {
    ReadParams p{};
    p.jobs = reinterpret_cast<const Job *>(words + plan->at.jobs);
    p.table = reinterpret_cast<const int *>(a->table);
    p.exponents = reinterpret_cast<const int *>(args->exponents);
    p.k = reinterpret_cast<const uint8_t *>(a->k_cache);
    p.v = reinterpret_cast<const uint8_t *>(a->v_cache);
    p.k_out = reinterpret_cast<uint16_t *>(b.k_cache);
    p.v_out = reinterpret_cast<uint16_t *>(b.v_cache);
    p.table_stride = a->table_stride;
    for (int i = 0; i < 3; ++i) p.k_stride[i] = a->k_cache_stride[i], p.v_stride[i] = a->v_cache_stride[i];
    p.pages = a->pages;
    p.page_size = a->page_size;
    p.page_shift = shift;
    p.page_inverse = inverse;
    p.kv_heads = plan->kv_heads;
    p.bf16 = a->dtype == 9;
    const dim3 grid(plan->n_jobs, plan->kv_heads, 2);
    if (d == 128)
      read_back_kernel<128><<<grid, 256, 0, s>>>(p);
    else
      read_back_kernel<64><<<grid, 256, 0, s>>>(p);
    if (const cudaError_t e = cudaGetLastError()) return cuda_fail("emmy_quantised_attention: launch", e);
  }
  return emmy_paged_attention(plan->others, &b, stream);
}

extern "C" EMMY_API int emmy_quantised_plan_status(emmy_quantised_plan_t plan, uint64_t plan_words, void *stream) {
  if (!plan || !plan_words) return fail("emmy_quantised_plan_status: bad argument");
  // (the kernel for few rows waits for nothing)
  if (!plan->others) return emmy_stream_sync(stream);
  return emmy_paged_plan_status(plan->others, plan_words + 4 * uint64_t(plan->at.others), stream);
}
