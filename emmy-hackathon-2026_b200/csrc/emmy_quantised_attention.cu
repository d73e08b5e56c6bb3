// emmy_quantised_attention.cu -- attention over a paged cache of 8-bit floats.
//
//   s_j = scale 2^e q.k_j,  o = 2^f sum_j p_j v_j / l,  p_j = 2^(c (s_j - m)),  l = sum_j p_j
//
// with the powers of two of a head's keys and values (e, f) outside the products.
//
// Few query rows of a key head (decoding, drafted tokens): bound by reading the cache.
// A warp takes slices of 2 KiB of keys on its own: TMA copies their 8-bit rows, page by
// page, to its ring of shared memory some slices ahead; it widens them to f16 in
// registers -- every 8-bit float is an f16 -- and multiplies with mma.sync, which has no
// f16 to fetch from shared memory: 6 KiB a slice of 128 components instead of 20 with
// 16-bit tiles written back for tcgen05, whose throughput 8 rows could not use (a
// slice's products take 120 cycles of the 700 that its bytes take to arrive).
//
// The products are transposed, S^T = K Q^T and O^T = V^T P^T, so that keys and
// components fill the 16 rows of an instruction and 8 query rows its columns.  What a
// thread holds of S^T goes to P^T by movmatrix.  Neither keys nor components have to
// be in order within a sum, so a thread reads 16 bytes of a row at once: component
// order is permuted alike in K and Q, and the key order of 64 components (key_of) keeps
// the reads of K and of V, whose rows a thread pairs byte by byte, off one another's
// banks.
//
// Queries of any 16-bit type become f16 with a power of two that brings the row's
// largest to 2^14..2^15: exact for components down to 2^-29 of it, and within 2^-40 of
// it below, far under the rounding of the sums in 32 bits.  Weights are rounded to
// f16; they start at 2^6 and grow to 2^14 before the base moves, so that small ones
// keep their bits.
//
// What bounds it: the memory, where sequences are long: 64 of 517 to 8,191 keys, 32 + 8
// heads of 128, 95 us (1.09 of reading them once), a key's 256 bytes taking each SM 11
// cycles where the work on it takes 8.  A warp on its own needs no barrier and joins
// nothing in shared memory; pieces that eight warps shared, with a thread fence, a counter
// and the joining of parts at their ends, took 120 us, since each such step takes 3 us
// while the memory is busy.  Short calls are bound by their latencies: about 4 us from
// the launch to the first keys (lists, piece, page, keys, each behind the one before).
//
// More rows go through the 16-bit cache's tcgen05 attention, which widens 8-bit tiles
// itself, or, with many, over keys and values that read_back_kernel reads back to 16 bits
// once, in pages of 128 tokens (times their power of two: exact in either type).
#include "emmy_quantised.h"

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>

int emmy_internal_fail(int code, const char *msg);   // emmy_runtime.cpp

using namespace emmy_quantised;

namespace {

constexpr float kNoMax = -FLT_MAX;      // base of a row that has seen no key
constexpr float kShift = 6.f, kGrow = 8.f;      // log2 of the weight at the base, and growth before it moves
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct alignas(64) Params {
  CUtensorMap k, v;
  const Piece *pieces;
  const int *first;
  unsigned *status;
  const int *table, *exponents;
  const void *q;
  void *out;
  float *lse, *part_o;
  float4 *part_ml;                 // base, sum and c of a part's row
  int64_t table_stride, q_stride[2], out_stride[2];
  int page_size, box, page_shift;         // key / page_size = key * page_inverse >> page_shift; box: rows of a copy
  uint32_t page_inverse;
  int q_heads, kv_heads, group, group_inverse, causal, window, bf16;
  float scale_log2;
};

// NT: tiles of 8 query rows.  Shared memory: the warps' rings of slices, their pieces'
// queries in f16 (where they are not in registers) and c of each row, what a shared
// piece's results meet in, barriers.
template <int D, int NT> struct Shape {
  static constexpr int kWarps = warps_of(NT), kThreads = 32 * kWarps;
  static constexpr int kKeys = slice_keys(D), kSubs = kKeys / 16;          // keys of a slice, by 16 of a product
  static constexpr int kHalf = 16 * D, kStage = kSubs * 2 * kHalf;         // bytes: 16 keys, then their values
  static constexpr int kSteps = D / 16;                                    // products of 16 components
  static constexpr int kRounds = D / 32;                                   // of 4 of a thread's components, at a unit's end
  static constexpr bool kQueryRegs = NT * D <= 128;                        // queries in registers
  static constexpr int kStages = 3;                                        // slices of a warp in flight or in use
  static constexpr int kRing = kStages * kStage, kQueryBytes = kQueryRegs ? 0 : NT * kSteps * 256;
  static constexpr int kQuery = kWarps * kRing;
  static constexpr int kScales = kQuery + kWarps * kQueryBytes;
  static constexpr int kJoin = kScales + kWarps * NT * 8 * 4;              // the warps' parts of a round
  static constexpr int kSums = kJoin + kWarps * 1024;                      // (base, sum) of a warp's rows
  static constexpr int kBars = kSums + kWarps * NT * 8 * 8;
  static constexpr int kBytes = kBars + kWarps * kStages * 8 + 1024;
  static_assert(kRing % 1024 == 0 && 2 * (kBytes + 1024) <= 228 * 1024, "two CTAs an SM");
};

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void bar_init(uint32_t bar) { asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar)); }
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok;
}
__device__ __forceinline__ uint64_t now_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// false, in all of the warp, where a copy does not come within 2 s
__device__ __noinline__ bool wait_slow(uint32_t bar, uint32_t parity) {
  const uint64_t t0 = now_ns();
  bool ok = false;
  while (!ok && now_ns() - t0 < 2000000000ull) ok = bar_try(bar, parity);
  return __all_sync(~0u, ok);
}
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(map), "r"(bar), "r"(0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
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
  asm(
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

// What a warp copies next: every kWarps-th slice of the pieces that it shares, then
// those of its own.  Lane b copies box b of a slice, a page's 8 or 16 tokens; boxes
// that no row sees anything of are left out.
template <int D, int NT> struct Feed {
  using S = Shape<D, NT>;
  const Params &p;
  int piece, shared_end, own, last;  // the pieces from `piece` to shared_end, then from own to last
  int slice, step, end, lo, hi, kvh;
  const int *row;
  int page;                          // of this lane's box of the slice to come; INT_MIN: none

  __device__ __forceinline__ bool more() const { return own >= 0 || piece < last; }
  __device__ __forceinline__ int key() const { return slice * S::kKeys + threadIdx.x % 32 * p.box; }
  __device__ __forceinline__ int page_of(int key) const { return static_cast<int>(uint64_t(key) * p.page_inverse >> p.page_shift); }
  __device__ __forceinline__ void enter(int warp) {      // the first piece from `piece` on with a slice for this warp
    for (;; ++piece) {
      if (piece == shared_end && own >= 0) {
        piece = own;
        own = -1;
      }
      if (own < 0 && piece >= last) return;
      const Piece u = read_piece(p, piece);
      const int from = own < 0 ? 0 : warp;
      if (from >= u.nslices) continue;
      step = own < 0 ? 1 : S::kWarps;
      slice = u.slice0 + from;
      end = u.slice0 + u.nslices;
      lo = u.lo;
      hi = u.hi;
      kvh = u.kvh;
      row = p.table + u.seq * p.table_stride;
      // while the slices before it go on: the piece after it, and this one's queries
      if (piece + 1 < last) asm volatile("prefetch.global.L1 [%0];" ::"l"(p.pieces + piece + 1));
      const int lane = threadIdx.x % 32;
#pragma unroll
      for (int r = lane / (D / 64); r < 8 * NT; r += 32 / (D / 64)) {
        const int at = u.row0 + r, token = at * p.group_inverse >> 16;
        if (r < u.rows)
          asm volatile("prefetch.global.L1 [%0];" ::"l"(static_cast<const uint16_t *>(p.q) + (u.tok0 + token) * p.q_stride[0] +
                                                         (u.kvh * p.group + at - token * p.group) * p.q_stride[1] + lane % (D / 64) * 64));
      }
      break;
    }
  }
  __device__ __forceinline__ void look_up() {
    if (!more()) return;
    const int at = key();
    const bool wanted = threadIdx.x % 32 * p.box < S::kKeys && at < hi && at + p.box > lo;
    page = wanted ? max(-1, __ldg(row + page_of(at))) : INT_MIN;
  }
  __device__ __forceinline__ Feed(const Params &params, int shared, int shared_last, int first, int end_piece, int warp)
      : p(params), piece(shared), shared_end(shared_last), own(first), last(end_piece) {
    enter(warp);
    look_up();
  }
  // copies the slice to `stage` and looks the next one's pages up
  __device__ __forceinline__ void next(uint32_t stage, uint32_t bar, int warp) {
    if (!more()) return;
    const bool wanted = page != INT_MIN;
    const uint32_t bytes = __popc(__ballot_sync(~0u, wanted)) * p.box * (2 * D);
    if (threadIdx.x % 32 == 0) bar_expect(bar, bytes);
    __syncwarp();
    if (wanted) {
      const int at = key(), in_slice = threadIdx.x % 32 * p.box;
      const uint32_t to = stage + in_slice / 16 * (2 * S::kHalf) + in_slice % 16 * D;
      const int token = at - page_of(at) * p.page_size;
      load_box(to, &p.k, bar, token, kvh, page);
      load_box(to + S::kHalf, &p.v, bar, token, kvh, page);
    }
    __syncwarp();
    slice += step;
    if (slice >= end) {
      ++piece;
      enter(warp);
    }
    look_up();
  }
};

// The key of 16 that row m of S^T is, which column m of V^T is as well.  Rows of 128
// bytes are stored with their 16-byte pieces exchanged by the row's last three bits,
// which keeps all reads apart; those of 64 with the pieces of two rows exchanged alike,
// so that what is read together is taken from rows of different halves.
template <int D> __device__ __forceinline__ int key_of(int m) {
  const int t = m / 2 % 4;
  return D == 128 ? m : (((t & 1) + 4 * (t >> 1)) ^ (m & 1) * 3) + (m & 8);
}

template <int D, int NT>
__global__ void __launch_bounds__(Shape<D, NT>::kThreads, 2) few_rows_kernel(const __grid_constant__ Params p) {
  using S = Shape<D, NT>;
  constexpr int W = S::kWarps, DP = D / 8;          // DP: components of a thread
  extern __shared__ __align__(128) char raw[];
  const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
  char *const shared = raw + (base - smem_addr(raw));
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  // where this CTA's pieces begin, and this warp's
  const int *const lists = p.first + blockIdx.x * (W + 1);
  const int shared_end = __ldg(lists + 1), own = __ldg(lists + 1 + warp), last = __ldg(lists + 2 + warp);
  const uint32_t ring = base + warp * S::kRing, queries = base + S::kQuery + warp * S::kQueryBytes, bars = base + S::kBars + warp * S::kStages * 8;
  float *const scales = reinterpret_cast<float *>(shared + S::kScales) + warp * NT * 8;
  float2 *const sums = reinterpret_cast<float2 *>(shared + S::kSums);
  // after a call that gave up nothing more is done
  if (__syncthreads_or(threadIdx.x == 0 && __ldcg(p.status))) return;
  if (lane == 0) {
    for (int k = 0; k < S::kStages; ++k) bar_init(bars + 8 * k);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncwarp();

  int i = __ldg(lists);
  Feed<D, NT> feed(p, i, shared_end, own, last, warp);
  int stage = 0;                      // the slice in use; those after it are on their way
  uint32_t phase = 0;
  bool alive = true;
#pragma unroll 1
  for (int k = 0; k + 1 < S::kStages; ++k) feed.next(ring + k * S::kStage, bars + 8 * k, warp);

  bool alone = false;                 // at this warp's own pieces
  for (;; ++i) {
    if (!alone && i == shared_end) {
      alone = true;
      i = own;
    }
    if (alone && i >= last) break;
    const Piece u = read_piece(p, i);
    // ------------------------------------------------------------ queries
    uint32_t q[S::kQueryRegs ? NT * 2 * S::kSteps : 1];
    float c[S::kQueryRegs ? 2 * NT : 1];
    // a tile's row g: its components in the order of the products below, and c
    auto take_row = [&](int tile, uint32_t *w) {
      float top = 0.f;
      const int at = u.row0 + min(8 * tile + g, u.rows - 1), token = at * p.group_inverse >> 16, head = u.kvh * p.group + at - token * p.group;
      const uint16_t *src = static_cast<const uint16_t *>(p.q) + (u.tok0 + token) * p.q_stride[0] + head * p.q_stride[1] + D / 4 * t;
#pragma unroll
      for (int k = 0; k < 2 * S::kSteps; k += 4) {
        const uint4 x = *reinterpret_cast<const uint4 *>(src + 2 * k);
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
      return fminf(fmaxf(ldexpf(p.scale_log2, exponent_of(p, 0, u.kvh) - up), FLT_MIN), FLT_MAX);
    };
    if (S::kQueryRegs) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float of_row = take_row(nt, q + (S::kQueryRegs ? nt * 2 * S::kSteps : 0));
        c[S::kQueryRegs ? 2 * nt : 0] = __shfl_sync(~0u, of_row, 8 * t);
        c[S::kQueryRegs ? 2 * nt + 1 : 0] = __shfl_sync(~0u, of_row, 8 * t + 4);
        if (t == 0) scales[8 * nt + g] = of_row;
      }
    } else {
#pragma unroll 1
      for (int nt = 0; nt < NT; ++nt) {
        uint32_t w[2 * S::kSteps];
        const float of_row = take_row(nt, w);
#pragma unroll
        for (int k = 0; k < S::kSteps; ++k)
          asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(queries + ((nt * S::kSteps + k) * 32 + lane) * 8), "r"(w[2 * k]), "r"(w[2 * k + 1]) : "memory");
        if (t == 0) scales[8 * nt + g] = of_row;
      }
    }
    __syncwarp();
    auto scale_of = [&](int nt, int e) { return S::kQueryRegs ? c[S::kQueryRegs ? 2 * nt + e : 0] : scales[8 * nt + 2 * t + e]; };
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
    for (int slice = u.slice0 + (alone ? 0 : warp); slice < u.slice0 + u.nslices; slice += alone ? 1 : W) {
      const uint32_t keys = ring + stage * S::kStage;
      {
        const bool here = bar_try(bars + 8 * stage, phase);
        if (!__all_sync(~0u, here) && alive && !wait_slow(bars + 8 * stage, phase)) {
          alive = false;               // nothing more is copied, and the results are void
          if (lane == 0) atomicExch(p.status, 1u);
        }
      }
      {
        const int before = stage ? stage - 1 : S::kStages - 1;
        if (alive) feed.next(ring + before * S::kStage, bars + 8 * before, warp);
      }
      if (++stage == S::kStages) {
        stage = 0;
        phase ^= 1;
      }
      const int key0 = slice * S::kKeys;
      if (key0 < u.lo || key0 + S::kKeys > u.hi) {
        // values that no row sees are unwritten or another's: their weight is 0, but 0
        // times a NaN is not
        for (int k = lane; k < S::kKeys * (D / 16); k += 32) {
          const int at = k / (D / 16);
          if (key0 + at < u.lo || key0 + at >= u.hi)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(keys + at / 16 * (2 * S::kHalf) + S::kHalf + at % 16 * D + k % (D / 16) * 16), "r"(0) : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
      }

      // ---------------------------------------------------------- S^T = K Q^T
      float s[NT][S::kSubs][4], odd[NT][4];      // odd: a second chain of products (NT == 1, one of 16 keys)
      constexpr bool kTwo = NT == 1 && S::kSubs == 1;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          odd[nt][e] = 0.f;
#pragma unroll
          for (int h = 0; h < S::kSubs; ++h) s[nt][h][e] = 0.f;
        }
#pragma unroll
      for (int h = 0; h < S::kSubs; ++h)
#pragma unroll
        for (int d = 0; d < D / 64; ++d) {
          const uint32_t at = keys + h * 2 * S::kHalf + key_of<D>(g) * D + (D == 128 ? (2 * t + d) ^ g : t ^ (key_of<D>(g) >> 1 & 3)) * 16;
          uint32_t x[4], y[4];
          load4(at, x);
          load4(at + 8 * D, y);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t a[4] = {widen_low(x[k]), widen_low(y[k]), widen_high(x[k]), widen_high(y[k])};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              uint32_t b[2];
              if (S::kQueryRegs)
                b[0] = q[S::kQueryRegs ? 2 * (nt * S::kSteps + 4 * d + k) : 0], b[1] = q[S::kQueryRegs ? 2 * (nt * S::kSteps + 4 * d + k) + 1 : 0];
              else
                load2(queries + ((nt * S::kSteps + 4 * d + k) * 32 + lane) * 8, b);
              mma(kTwo && k % 2 ? odd[nt] : s[nt][h], a, b[0], b[1]);
            }
          }
        }
      if (kTwo) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[0][0][e] += odd[0][e];
      }

      // ---------------------------------------------------------- softmax
      if (key0 < max_lo || key0 + S::kKeys > min_hi) {
        const int key = key0 + key_of<D>(g);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            int lo, hi;
            seen_by(nt, e, lo, hi);
#pragma unroll
            for (int h = 0; h < S::kSubs; ++h) {
              if (key + 16 * h < lo || key + 16 * h >= hi) s[nt][h][e] = -INFINITY;
              if (key + 16 * h + 8 < lo || key + 16 * h + 8 >= hi) s[nt][h][2 + e] = -INFINITY;
            }
          }
        }
      }
      // the base follows the largest score when that has grown by more than 2^8
      float x[NT][S::kSubs][4], most = -INFINITY;
      auto exponents = [&] {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float by[2] = {scale_of(nt, 0), scale_of(nt, 1)};
#pragma unroll
          for (int h = 0; h < S::kSubs; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              x[nt][h][e] = fmaf(s[nt][h][e] - m[nt][e & 1], by[e & 1], kShift);
              most = fmaxf(most, x[nt][h][e]);
            }
        }
      };
      exponents();
      if (__any_sync(~0u, most > kShift + kGrow)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float by[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = fmaxf(s[nt][0][e], s[nt][0][2 + e]);
#pragma unroll
            for (int h = 1; h < S::kSubs; ++h) top = fmaxf(top, fmaxf(s[nt][h][e], s[nt][h][2 + e]));
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
        exponents();
      }
      uint32_t w[NT][S::kSubs][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int h = 0; h < S::kSubs; ++h) {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[nt][h][e] = exp2_approx(x[nt][h][e]);
          l[nt][0] += x[nt][h][0] + x[nt][h][2];
          l[nt][1] += x[nt][h][1] + x[nt][h][3];
          w[nt][h][0] = transposed(pack_f16(x[nt][h][0], x[nt][h][1]));
          w[nt][h][1] = transposed(pack_f16(x[nt][h][2], x[nt][h][3]));
        }
      }

      // ---------------------------------------------------------- O^T += V^T P^T
#pragma unroll
      for (int h = 0; h < S::kSubs; ++h) {
        uint32_t v[4][DP / 4];         // of the keys of columns 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int at = key_of<D>(2 * t + (j & 1)) + 8 * (j >> 1);
          const uint32_t row = keys + (2 * h + 1) * S::kHalf + at * D;
          if (D == 128)
            load4(row + (g ^ (at & 7)) * 16, v[j]);
          else
            load2(row + (g / 2 ^ (at >> 1 & 3)) * 16 + (g & 1) * 8, v[j]);
        }
#pragma unroll
        for (int k = 0; k < DP / 4; ++k) {
          const uint32_t p0 = __byte_perm(v[0][k], v[1][k], 0x5140), p1 = __byte_perm(v[0][k], v[1][k], 0x7362);
          const uint32_t p2 = __byte_perm(v[2][k], v[3][k], 0x5140), p3 = __byte_perm(v[2][k], v[3][k], 0x7362);
          const uint32_t a[4] = {widen_low(p0), widen_high(p0), widen_low(p2), widen_high(p2)};
          const uint32_t b[4] = {widen_low(p1), widen_high(p1), widen_low(p3), widen_high(p3)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma(o[nt][2 * k], a, w[nt][h][0], w[nt][h][1]);
            mma(o[nt][2 * k + 1], b, w[nt][h][0], w[nt][h][1]);
          }
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
      }
    const bool split = u.nsplit > 1;
    const int64_t part = u.part_row + int64_t(u.split) * u.rows;
    const float unscaled = power_of_two(exponent_of(p, 1, u.kvh));
    auto token_of = [&](int r) { return (u.row0 + r) * p.group_inverse >> 16; };
    auto lse_of = [&](int r) { return p.lse + int64_t(u.tok0 + token_of(r)) * p.q_heads + u.kvh * p.group + u.row0 + r - token_of(r) * p.group; };
    auto out_of = [&](int r) {
      return static_cast<uint16_t *>(p.out) + (u.tok0 + token_of(r)) * p.out_stride[0] + (u.kvh * p.group + u.row0 + r - token_of(r) * p.group) * p.out_stride[1];
    };
    auto rounded = [&](float x, float y) { return p.bf16 ? pack_bf16(x, y) : pack_f16(x, y); };
    if (alone) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = 8 * nt + 2 * t + e;
          if (r >= u.rows) continue;
          if (split) {
            float4 *to = reinterpret_cast<float4 *>(p.part_o + (part + r) * D + DP * g);
#pragma unroll
            for (int k = 0; k < S::kSteps; k += 2) __stcg(to + k / 2, make_float4(o[nt][k][e], o[nt][k][2 + e], o[nt][k + 1][e], o[nt][k + 1][2 + e]));
            if (g == 0) __stcg(p.part_ml + part + r, make_float4(m[nt][e], l[nt][e], scale_of(nt, e), 0.f));
          } else {
            const float inv = reciprocal(l[nt][e]) * unscaled;
            uint4 *to = reinterpret_cast<uint4 *>(out_of(r) + DP * g);
#pragma unroll
            for (int k = 0; k < S::kSteps; k += 4)
              to[k / 4] = make_uint4(rounded(o[nt][k][e] * inv, o[nt][k][2 + e] * inv), rounded(o[nt][k + 1][e] * inv, o[nt][k + 1][2 + e] * inv),
                                     rounded(o[nt][k + 2][e] * inv, o[nt][k + 2][2 + e] * inv), rounded(o[nt][k + 3][e] * inv, o[nt][k + 3][2 + e] * inv));
            if (g == 0 && p.lse) *lse_of(r) = log_sum(m[nt][e], scale_of(nt, e), l[nt][e]);
          }
        }
      }
      __syncwarp();        // queries and scales have been read
      continue;
    }
    if (g == 0) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) sums[warp * NT * 8 + 8 * nt + 2 * t + e] = make_float2(m[nt][e], l[nt][e]);
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
    if (threadIdx.x < u.rows) {
      const int r = threadIdx.x;
      const float2 all = joined(r, scales[r]);
      if (split) {
        __stcg(p.part_ml + part + r, make_float4(all.x, all.y, scales[r], 0.f));
      } else if (p.lse) {
        *lse_of(r) = log_sum(all.x, scales[r], all.y);
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
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
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int from = 0; from < S::kRounds; ++from) {
        if (nt || from) __syncthreads();
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int k = 2 * from;
          const uint32_t to = join + ((warp * 8 + 2 * t + e) * 8 + (g ^ t << 1)) * 16;
          asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(o[nt][k][e]), "f"(o[nt][k][2 + e]), "f"(o[nt][k + 1][e]), "f"(o[nt][k + 1][2 + e]) : "memory");
        }
        __syncthreads();
        if (threadIdx.x < 64 && 8 * nt + threadIdx.x / 8 < u.rows) {
          const int of_tile = threadIdx.x / 8, r = 8 * nt + of_tile, of = threadIdx.x % 8;
          float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < W; ++w) {
            float4 x;
            const uint32_t at = join + ((w * 8 + of_tile) * 8 + (of ^ (of_tile >> 1) << 1)) * 16;
            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(at) : "memory");
            sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
          }
          const int component = DP * of + 4 * from;
          if (split) {
            __stcg(reinterpret_cast<float4 *>(p.part_o + (part + r) * D + component), sum);
          } else {
            *reinterpret_cast<uint2 *>(out_of(r) + component) = make_uint2(rounded(sum.x, sum.y), rounded(sum.z, sum.w));
          }
        }
      }
    }
    __syncthreads();      // sums have been read
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // copies in flight land before the CTA ends, also when their user gave up
  if (!alive) {
    const uint64_t t0 = now_ns();
    for (int k = 0; k < S::kStages; ++k)
      for (uint32_t parity = 0; parity < 2; ++parity)
        while (now_ns() - t0 < 100000000ull && !bar_try(bars + 8 * k, parity)) {
        }
  }
}

struct JoinParams {
  const Joined *rows;
  const int *exponents;
  const unsigned *status;
  const float *part_o;
  const float4 *part_ml;
  void *out;
  float *lse;
  int64_t out_stride[2];
  int q_heads, kv_heads, group, bf16;
};

// The parts of one row an item, in their order: a thread has 4 components of every
// kGroups-th part.  Launched while the kernel before it ends, and waits for that.
template <int D> __global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ JoinParams p) {
  constexpr int kLanes = D / 4, kGroups = 128 / kLanes;
  __shared__ float4 sums[128];
  __shared__ float totals[kGroups], tops[4];
  const int4 u = __ldg(reinterpret_cast<const int4 *>(p.rows + blockIdx.x));       // of the plan: not written by any kernel
  const int head = __ldg(&p.rows[blockIdx.x].head), tid = threadIdx.x, group = tid / kLanes, step = u.y, nsplit = u.z;
  const float unscaled = power_of_two(p.exponents ? min(max(__ldg(p.exponents + p.kv_heads + head / p.group), EMMY_MIN_EXPONENT), EMMY_MAX_EXPONENT) : 0);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (__ldcg(p.status)) return;
  const float4 *const ml = p.part_ml + u.x;
  const float c = __ldcg(ml).z;
  float top = kNoMax, total = 0.f;
  for (int k = tid; k < nsplit; k += 128) top = fmaxf(top, __ldcg(ml + int64_t(k) * step).x);
  for (int k = 16; k; k /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, k));
  if (tid % 32 == 0) tops[tid / 32] = top;
  __syncthreads();
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  const float4 *const src = reinterpret_cast<const float4 *>(p.part_o + int64_t(u.x) * D) + tid % kLanes;
#pragma unroll 8
  for (int k = group; k < nsplit; k += kGroups) {
    const float4 of = __ldcg(ml + int64_t(k) * step), x = __ldcg(src + int64_t(k) * step * kLanes);
    const float by = weight(of.x, top, c);
    total += by * of.y;
    sum.x += by * x.x, sum.y += by * x.y, sum.z += by * x.z, sum.w += by * x.w;
  }
  sums[tid] = sum;
  if (tid % kLanes == 0) totals[group] = total;
  __syncthreads();
  if (group) return;
  for (int k = 1; k < kGroups; ++k) {
    const float4 x = sums[k * kLanes + tid];
    sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
  }
  total = 0.f;
#pragma unroll
  for (int k = 0; k < kGroups; ++k) total += totals[k];
  const float inv = reciprocal(total) * unscaled;
  uint16_t *to = static_cast<uint16_t *>(p.out) + u.w * p.out_stride[0] + head * p.out_stride[1] + 4 * tid;
  *reinterpret_cast<uint2 *>(to) = p.bf16 ? make_uint2(pack_bf16(sum.x * inv, sum.y * inv), pack_bf16(sum.z * inv, sum.w * inv))
                                          : make_uint2(pack_f16(sum.x * inv, sum.y * inv), pack_f16(sum.z * inv, sum.w * inv));
  if (tid == 0 && p.lse) p.lse[int64_t(u.w) * p.q_heads + head] = log_sum(top, c, total);
}

struct ReadParams {
  const Job *jobs;
  const unsigned *status;
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
  if (__ldcg(p.status)) return;
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
  const int ps = a->page_size;
  if (ps < 8 || (ps < kBlock ? (ps & (ps - 1)) != 0 : ps % kBlock != 0))
    return fail("emmy_quantised_attention: page_size %ld (8, 16, 32, 64 or a multiple of 128)", ps);
  if (a->pages < (reads ? 1 : 0)) return fail("emmy_quantised_attention: a cache of %ld pages", a->pages);
  if (a->table_width < 0 || int64_t(a->table_width) * a->page_size < plan->max_kv)
    return fail("emmy_quantised_attention: a table of %ld pages a sequence does not hold %ld tokens", a->table_width, plan->max_kv);
  const Scratch scratch = scratch_of(*plan);
  if (!a->q || !a->out || (reads && (!a->k_cache || !a->v_cache || !a->table)) || !a->plan_words || (scratch.end && !a->scratch))
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
  unsigned *const status = reinterpret_cast<unsigned *>(words + plan->at.status);
  const uint64_t status_at = reinterpret_cast<uint64_t>(status);
  char *scratch_at = reinterpret_cast<char *>(a->scratch);
  // key * inverse >> shift is key / page_size for keys up to 2^30: 2^shift / page_size
  // rounded up is too large by less than 1, which key times that, under 2^shift, forgives
  int log = 0;
  while ((int64_t(1) << log) < a->page_size) ++log;
  const int shift = 30 + log;
  const uint32_t inverse = static_cast<uint32_t>(((uint64_t(1) << shift) + a->page_size - 1) / a->page_size);

  if (plan->at.ctas) {
    Params p;
    memset(&p, 0, sizeof p);
    p.box = a->page_size % 16 ? 8 : 16;
    if (plan->reads) {
      const uint64_t dims[4] = {uint64_t(d), uint64_t(a->page_size), uint64_t(plan->kv_heads), uint64_t(a->pages)};
      const uint32_t box[4] = {uint32_t(d), uint32_t(p.box), 1, 1};
      for (int i = 0; i < 2; ++i) {
        const int64_t *st = i ? a->v_cache_stride : a->k_cache_stride;
        uint64_t steps[3];
        const int order[3] = {1, 2, 0};
        for (int k = 0; k < 3; ++k) steps[k] = extent[order[k]] == 1 ? 16 : st[order[k]];      // (a stride of one entry is never used)
        if (int e = emmy_tensormap_encode(i ? &p.v : &p.k, 0, 4, i ? a->v_cache : a->k_cache, dims, steps, box, d == 128 ? 3 : 2)) return e;
      }
    }
    p.status = status;
    p.first = words + 4;
    p.pieces = reinterpret_cast<const Piece *>(words + plan->at.pieces);
    p.table = reinterpret_cast<const int *>(a->table);
    p.exponents = reinterpret_cast<const int *>(args->exponents);
    p.q = reinterpret_cast<const void *>(a->q);
    p.out = reinterpret_cast<void *>(a->out);
    p.lse = reinterpret_cast<float *>(a->lse);
    p.part_o = reinterpret_cast<float *>(scratch_at);
    p.part_ml = reinterpret_cast<float4 *>(p.part_o + plan->part_rows * d);
    p.table_stride = a->table_stride;
    for (int i = 0; i < 2; ++i) p.q_stride[i] = a->q_stride[i], p.out_stride[i] = a->out_stride[i];
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
    const int e = d == 128 ? (plan->tiles == 1 ? launch<128, 1>(p, n, s) : launch<128, 2>(p, n, s))
                           : (plan->tiles == 1 ? launch<64, 1>(p, n, s) : launch<64, 2>(p, n, s));
    if (e) return e;
    if (plan->n_joined) {
      JoinParams join{};
      join.rows = reinterpret_cast<const Joined *>(words + plan->at.joined);
      join.exponents = p.exponents;
      join.status = p.status;
      join.part_o = p.part_o;
      join.part_ml = p.part_ml;
      join.out = p.out;
      join.lse = p.lse;
      for (int i = 0; i < 2; ++i) join.out_stride[i] = p.out_stride[i];
      join.q_heads = p.q_heads;
      join.kv_heads = p.kv_heads;
      join.group = p.group;
      join.bf16 = p.bf16;
      cudaLaunchConfig_t config{};
      config.gridDim = dim3(plan->n_joined);
      config.blockDim = dim3(128);
      config.stream = s;
      cudaLaunchAttribute early;
      early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
      early.val.programmaticStreamSerializationAllowed = 1;
      config.attrs = &early;
      config.numAttrs = 1;
      if (const cudaError_t e = d == 128 ? cudaLaunchKernelEx(&config, join_kernel<128>, join) : cudaLaunchKernelEx(&config, join_kernel<64>, join))
        return cuda_fail("emmy_quantised_attention: launch", e);
    }
  }
  emmy_paged_attention_args b = *a;
  if (plan->middle) {
    b.plan_words = reinterpret_cast<uint64_t>(words + plan->at.middle);
    b.scratch = a->scratch + scratch.middle;
    if (int e = emmy_internal_paged_attention(plan->middle, &b, true, args->exponents, status_at, stream)) return e;
  }
  if (!plan->many) return 0;
  const int64_t page = int64_t(kBlock) * plan->kv_heads * d;
  b.page_size = kBlock;
  b.pages = static_cast<int32_t>(plan->workspace_pages);
  b.table_width = plan->table_width;
  b.table = reinterpret_cast<uint64_t>(words + plan->at.table);
  b.table_stride = plan->table_width;
  b.plan_words = reinterpret_cast<uint64_t>(words + plan->at.many);
  b.scratch = a->scratch + scratch.many;
  b.k_cache = a->scratch + scratch.workspace;
  b.v_cache = b.k_cache + plan->workspace_pages * page * 2;
  const int64_t strides[3] = {page, d, int64_t(kBlock) * d};
  for (int i = 0; i < 3; ++i) b.k_cache_stride[i] = b.v_cache_stride[i] = strides[i];
  if (plan->n_jobs) {
    ReadParams p{};
    p.jobs = reinterpret_cast<const Job *>(words + plan->at.jobs);
    p.status = status;
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
  return emmy_internal_paged_attention(plan->many, &b, false, 0, status_at, stream);
}

extern "C" EMMY_API int emmy_quantised_plan_status(emmy_quantised_plan_t plan, uint64_t plan_words, void *stream) {
  if (!plan || !plan_words) return fail("emmy_quantised_plan_status: bad argument");
  int status = 0;
  if (int e = emmy_memcpy_dtoh_async(&status, plan_words + 4 * uint64_t(plan->at.status), sizeof status, stream)) return e;
  if (int e = emmy_stream_sync(stream)) return e;
  if (status) return emmy_internal_fail(EMMY_EKERNEL, "emmy_quantised_attention: a wait ran out");
  if (plan->middle)
    if (int e = emmy_paged_plan_status(plan->middle, plan_words + 4 * uint64_t(plan->at.middle), stream)) return e;
  return plan->many ? emmy_paged_plan_status(plan->many, plan_words + 4 * uint64_t(plan->at.many), stream) : 0;
}
