// emmy_paged_attention.cu -- attention of ragged chunks of new tokens, from one
// token a sequence upwards, over a paged key/value cache.
//
//   s_j = scale q.k_j,  o = sum_j e^(s_j - m) v_j / l,  l = sum_j e^(s_j - m)
//
// in one pass over the keys with a running maximum and sum.  The G query heads
// of a key head are stacked with the tokens (row = token * G + head of the
// group), so a key tile is read once for all of them, whatever G is.
//
// One persistent CTA an SM walks its list of units (emmy_paged.h).  Its roles:
//   warps 0-3, 4-7  softmax of stream 0 and 1, one thread a row;
//   warps 10, 11    issue the tensor-core products of stream 0 and 1;
//   warps 8, 9      load key tiles, and value and query tiles; keys and values,
//                   page by page, into one ring.
// A unit with two query tiles gives one to each stream and both see every key
// tile; a unit with one query tile (decode) gives it to both streams, which
// take the key tiles in turn and are joined at the end.  Either way one
// stream's softmax runs while the tensor cores work for the other.
//
// The few rows of a decoding unit (32 or less) would leave three of a stream's
// four warps idle and one with 128 exponentials a row, 1,200 cycles, more than
// the tile takes to arrive.  Their queries are loaded four times, into the rows
// of each warp: every warp then has all scores of all rows, and takes a quarter
// of the keys, with a maximum and a sum of its own.  The products with a quarter's
// values write that warp's rows only: weights of 0 in the other rows would come to
// the same, but for values that are infinite.  The eight results are joined in
// shared memory, where the second query tile would be.
//
// Tensor memory: S_t at column 128 t, P_t over it (two 16-bit weights a
// column), O_t at 256 + 128 t.  S = Q K^T and O += P V are 128 x 128 x D and
// 128 x D x 128 tcgen05.mma chains; both accumulate in 32 bits.  P is rounded
// to the type of V, which the product needs; the sum l is taken before that.
//
// What bounds it.  Decoding: memory; a pair of tiles costs a CTA 1.37 us with 128
// components, 0.73 with 64 (6.1 to 7.0 TB/s at length), and a unit's end 2 to 3.5.
// Chunks: a stream's tile is a chain of softmax (load and maximum 360 cycles,
// exponentials 1,340), P V and Q K^T (1,100), 3,030 cycles for both streams where
// the tensor cores alone take 2,048 and the exponential unit as much: 1,180 to
// 1,280 TFLOP/s at units of 64 and 128 tiles, 8 prompts of 4,096 tokens with 32 + 8
// heads of 128 in 0.99 ms replayed from a graph (1,105 TFLOP/s of what causal attention
// needs) and 1.08 ms called again and again, where the power limit lowers the clock.
//
// Every wait is bounded; one that runs out sets the plan's status word, and
// from then on its CTA issues nothing more, and later calls do nothing.
#include "emmy_paged.h"

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <climits>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>

int emmy_internal_fail(int code, const char *msg);   // emmy_runtime.cpp

namespace {

using emmy_paged::kTile;
using emmy_paged::Unit;

// Registers a thread: at launch, then those of the softmax warps, which hold a
// row of scores, and of the others; the shares add up to what was launched.
// BITS8: a cache of 8-bit floats, which four more warps widen.
template <bool BITS8> struct Warps {
  static constexpr int kThreads = BITS8 ? 512 : 384;
  static constexpr int kLaunchRegs = BITS8 ? 128 : 168, kSoftmaxRegs = BITS8 ? 200 : 216, kOtherRegs = BITS8 ? 56 : 72;
  static_assert(256 * kSoftmaxRegs + (kThreads - 256) * kOtherRegs <= kThreads * kLaunchRegs, "register split");
};
constexpr int kSoftmaxWarps = 8, kKeyWarp = 8, kMmaWarp = 10, kWideningWarp = 12;
constexpr int kSmem = 227 * 1024;
constexpr float kNoMax = -FLT_MAX;      // exponent base of a row that has seen no key
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct alignas(64) Params {
  CUtensorMap q, q32, k, v;            // q32: the rows of one warp
  const Unit *units;
  const int *cta_first;
  const int *table;
  unsigned *counters, *status;
  unsigned *batch_status;              // of the plan that this one is a part of; its own where it is none
  float *part_o;
  float2 *part_ml;
  void *out;
  float *lse;
  int64_t table_stride, out_stride[2];
  int q_heads, group, group_inverse, per_tile, box, causal, window, aligned32;
  int tiles_a_page;                    // of pages of a tile or more
  float scale_log2, scale_power;       // c, and the power of two next to it
  const int *exponents;                // of an 8-bit cache's keys and values, [2][kv_heads]; null: 0
  int kv_heads;
};

template <int D, bool BITS8> struct Shape {
  static constexpr int kTileBytes = kTile * D * 2;       // 16 KiB or more: the joining needs them
  static constexpr int kStages = BITS8 ? (D == 128 ? 4 : 8) : D == 128 ? 5 : 12;      // key and value tiles in flight
  // after two query tiles (BITS8, where no unit is wide: one, and 16 KiB for the joining)
  static constexpr int kRing = kTileBytes + (BITS8 ? 16384 : kTileBytes);
  // BITS8: the tiles as they arrive, of 8-bit floats; the others are widened
  static constexpr int kRawStages = BITS8 ? (D == 128 ? 3 : 8) : 0, kRaw = kRing + kStages * kTileBytes;
  static constexpr int kBars = kRaw + kRawStages * (kTileBytes / 2);
  static constexpr int kWords = kBars + (2 * kStages + 14 + 2 * kRawStages + (BITS8 ? 1 : 0)) * 8, kPowers = kWords + 32 + kTile * 8;
  static constexpr int kEnd = kPowers + (BITS8 ? 2 * kTile : 0);
  // tiles that are copied ahead, and bytes of an element there
  static constexpr int kCopied = BITS8 ? kRawStages : kStages, kElement = BITS8 ? 1 : 2;
  // A loader waits for a stage by one bit of its phase, which two fills earlier has as well.
  // It comes to a place of the ring at most 3 after its last (load_role), for which it saw
  // the fill `kCopied` before that released, and stages are released in the ring's order: from
  // 3 stages on that covers the fill 2 kCopied before the place.
  static_assert(kCopied >= 3, "a stage's phase would be ambiguous");
  static_assert(kEnd + 1024 <= kSmem, "shared memory");
};

// ---------------------------------------------------------------- PTX
__device__ __forceinline__ uint32_t smem_addr(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void bar_init(uint32_t bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
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
// the same without the pause that a failed try takes
__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
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

// What a role needs to give up: the CTA's flag (any role may set it) and the
// plan's status word, with that of the plan which it is a part of.
struct Guard {
  uint32_t dead;          // shared-memory address
  const Params &p;
  // false once a wait of this CTA ran out (2 s); the caller then issues nothing more
  __device__ __forceinline__ bool slow(uint32_t bar, uint32_t parity, int code) const {
    const uint64_t t0 = now_ns();
    for (;;) {
      if (bar_try(bar, parity)) return true;
      int gave_up;
      asm volatile("ld.volatile.shared.b32 %0, [%1];" : "=r"(gave_up) : "r"(dead) : "memory");
      if (gave_up) return false;
      if (now_ns() - t0 > 2000000000ull) {
        asm volatile("st.volatile.shared.b32 [%0], 1;" ::"r"(dead) : "memory");
        atomicExch(p.status, code);
        atomicExch(p.batch_status, code);
        return false;
      }
    }
  }
  // one answer for the warp
  __device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, int code) const {
    const bool ok = bar_try(bar, parity);
    return __all_sync(~0u, ok) || __all_sync(~0u, slow(bar, parity, code));
  }
};

__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
// true for one lane of a converged warp.  Compared with `lane == 0` the compiler
// knows that one lane at most is active, and passes a tensor instruction's
// operands without a loop over the lanes.
__device__ __forceinline__ bool elected() {
  uint32_t yes;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
  return yes;
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// a and b: low words of the operands' descriptors, `high` the high word of both
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t high, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(high), "r"(idesc), "r"(static_cast<uint32_t>(acc))
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t high, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(high), "r"(idesc), "r"(static_cast<uint32_t>(acc))
      : "memory");
}
// the same, into the rows of warp `w` (lanes 32 w to 32 w + 31 of D) only
__device__ __forceinline__ void mma_ts_rows(uint32_t d, uint32_t a, uint32_t b, uint32_t high, uint32_t idesc, bool acc, int w) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, {%6, %7, %8, %9}, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(high), "r"(idesc), "r"(static_cast<uint32_t>(acc)), "r"(w == 0 ? 0u : ~0u), "r"(w == 1 ? 0u : ~0u),
      "r"(w == 2 ? 0u : ~0u), "r"(w == 3 ? 0u : ~0u)
      : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at));
}
__device__ __forceinline__ void tmem_ld16(uint32_t at, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at));
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// the registers of a load are valid only after this: they pass through it so
// that no use of them can move above it
template <int N> __device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[N], int from = 0, int to = N) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = from; i < to; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(uint32_t x, uint32_t y, uint32_t z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(__uint_as_float(x)), "f"(__uint_as_float(y)), "f"(__uint_as_float(z)));
  return r;
}
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float &x, float &y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// 2^x of a pair on the multiply-add pipe, for x <= 128: n = x rounded, a quintic in
// x - n on [-1/2, 1/2] (minimising the largest relative error: 2.2e-7 evaluated in 32
// bits, what the exponential unit has too), times 2^n, exactly 0 from -127 down.  NaN
// stays.  A cubic's 7.5e-5 would do for the weights, which are rounded to 16 bits, but
// shows in their sum: the lse of rows of few keys came out up to 7e-5 off.
__device__ __forceinline__ uint64_t exp2_pair(uint64_t x) {
  float a, b;
  unpair(x, a, b);
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(a));
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(b));
  x = pair(a, b);
  const uint64_t t = add2(x, pair(12582912.f, 12582912.f));     // 1.5 * 2^23: n in the low bits
  const uint64_t f = fma2(add2(t, pair(-12582912.f, -12582912.f)), pair(-1.f, -1.f), x);
  uint64_t p = fma2(pair(0.0013276472454890609f, 0.0013276472454890609f), f, pair(0.0096755409613251686f, 0.0096755409613251686f));
  p = fma2(p, f, pair(0.055507130920886993f, 0.055507130920886993f));
  p = fma2(p, f, pair(0.24022120237350464f, 0.24022120237350464f));
  p = fma2(p, f, pair(0.69314694404602051f, 0.69314694404602051f));
  p = fma2(p, f, pair(1.f, 1.f));
  unpair(t, a, b);
  return mul2(p, pair(__uint_as_float((__float_as_uint(a) << 23) + 0x3f800000u), __uint_as_float((__float_as_uint(b) << 23) + 0x3f800000u)));
}
template <bool BF16> __device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  if (BF16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Shared-memory operand descriptor: 128-byte swizzle, leading and stride byte
// offsets in 16-byte units.  Keys and queries are K-major (rows of 64
// components, 8-row groups 1024 bytes apart); values are MN-major (64 columns
// of one key a row, the next 64 columns 16 KiB further).
constexpr uint32_t kOperandHigh = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t operand(uint32_t addr, uint32_t lead) {
  // a reduction's result is known to be the same in every lane, so that it and
  // the steps along it stay in uniform registers, which the products read
  return __reduce_or_sync(~0u, ((addr >> 4) & 0x3fff) | ((lead >> 4) << 16));
}
template <bool BF16> __host__ __device__ constexpr uint32_t instruction(int n, bool b_mn_major) {
  return (1u << 4) | (uint32_t(BF16) << 7) | (uint32_t(BF16) << 10) | (uint32_t(b_mn_major) << 16) | (uint32_t(n >> 3) << 17) |
         (uint32_t(kTile >> 4) << 24);
}

// ---------------------------------------------------------------- roles
template <int D, bool SPREAD, bool BITS8> struct Smem {
  using S = Shape<D, BITS8>;
  uint32_t base;       // 1024-byte aligned
  __device__ uint32_t query(int t) const { return base + t * S::kTileBytes; }
  __device__ uint32_t stage(int s) const { return base + S::kRing + s * S::kTileBytes; }
  __device__ uint32_t bar(int i) const { return base + S::kBars + 8 * i; }
  __device__ uint32_t full(int s) const { return bar(s); }
  __device__ uint32_t empty(int s) const { return bar(S::kStages + s); }
  __device__ uint32_t q_full() const { return bar(2 * S::kStages); }
  __device__ uint32_t q_empty() const { return bar(2 * S::kStages + 1); }
  __device__ uint32_t s_full(int t) const { return bar(2 * S::kStages + 2 + t); }
  // the weights of a tile's first and last 64 keys
  __device__ uint32_t p_ready(int t, int half) const { return bar(2 * S::kStages + 4 + 2 * t + half); }
  __device__ uint32_t final(int t) const { return bar(2 * S::kStages + 8 + t); }
  __device__ uint32_t drain(int t) const { return bar(2 * S::kStages + 10 + t); }
  // wide units: stream t may issue
  __device__ uint32_t turn(int t) const { return bar(2 * S::kStages + 12 + t); }
  // where queries are known to have been copied, and by which power of two a row of
  // them was multiplied, of even and odd units
  __device__ uint32_t q_copied() const { return BITS8 ? bar(2 * S::kStages + 14 + 2 * S::kRawStages) : q_full(); }
  __device__ volatile int8_t *powers(int odd) const { return static_cast<volatile int8_t *>(__cvta_shared_to_generic(base + S::kPowers)) + odd * kTile; }
  // where tiles are copied to, and their barriers
  __device__ uint32_t copied(int s) const { return BITS8 ? base + S::kRaw + s * (S::kTileBytes / 2) : stage(s); }
  __device__ uint32_t copied_full(int s) const { return BITS8 ? bar(2 * S::kStages + 14 + s) : full(s); }
  __device__ uint32_t copied_empty(int s) const { return BITS8 ? bar(2 * S::kStages + 14 + S::kRawStages + s) : empty(s); }
  __device__ volatile int *words() const { return static_cast<volatile int *>(__cvta_shared_to_generic(base + S::kWords)); }
  __device__ float2 *ml() const { return static_cast<float2 *>(__cvta_shared_to_generic(base + S::kWords + 32)); }
};
// words(): 0 dead, 1 tensor memory address, 2 + t "last to arrive" of stream t

template <int STAGES> struct Ring {
  int stage = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int n = 1) {     // n <= STAGES
    stage += n;
    if (stage >= STAGES) {
      stage -= STAGES;
      phase ^= 1;
    }
  }
};

// row / group of a tile's rows (both under 2^8) as a product
__device__ __forceinline__ int token_of(const Params &p, int row) { return row * p.group_inverse >> 16; }

// Read anew where it is used (from L1, which keeps it): a unit kept in registers
// across the loop over its key tiles would cost the softmax warps 16 of them.
__device__ __forceinline__ Unit read_unit(const Params &p, int i) {
  Unit u;
  const Unit *at = p.units + i;
  asm volatile("ld.global.nc.L1::evict_last.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(u.seq), "=r"(u.kvh), "=r"(u.tok0), "=r"(u.ntok) : "l"(at));
  asm volatile("ld.global.nc.L1::evict_last.v4.b32 {%0, %1, %2, %3}, [%4+16];" : "=r"(u.pos0), "=r"(u.tile0), "=r"(u.ntiles), "=r"(u.lo) : "l"(at));
  asm volatile("ld.global.nc.L1::evict_last.v4.b32 {%0, %1, %2, %3}, [%4+32];" : "=r"(u.hi), "=r"(u.kv_len), "=r"(u.wide), "=r"(u.item) : "l"(at));
  asm volatile("ld.global.nc.L1::evict_last.v4.b32 {%0, %1, %2, %3}, [%4+48];" : "=r"(u.split), "=r"(u.nsplit), "=r"(u.part_row), "=r"(u.pad) : "l"(at));
  return u;
}

// A unit of at most 32 rows: each warp of a stream has all of them and a quarter
// of the keys.  A plan without such units runs a kernel without their code
// (!SPREAD), which in the wide units' kernel costs them 3 to 4 % though they never
// come to it: 1,030 against 1,005 us on 8 prompts of 4,096, 165 against 158 on the
// windowed chunks.
template <int D, bool SPREAD, bool BITS8> __device__ __forceinline__ bool spread(const Params &p, const Smem<D, SPREAD, BITS8> &, const Unit &u) {
  return SPREAD && emmy_paged::is_spread(u.wide, u.ntiles, u.ntok, p.group);
}

// Query tiles: one 128-row tile for each stream of a wide unit, one for both of
// a narrow one, each a box of group x tokens_per_tile rows; the rows of a spread
// unit four times.
template <int D, bool SPREAD, bool BITS8>
__device__ __forceinline__ void load_queries(const Params &p, const Smem<D, SPREAD, BITS8> &sm, const Unit &u) {
  if (spread(p, sm, u)) {
    bar_expect(sm.q_copied(), 4 * p.group * (32 / p.group) * 128 * (D / 64));
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int h = 0; h < D / 64; ++h)
        load_box(sm.query(0) + h * (kTile * 128) + w * (32 * 128), &p.q32, sm.q_copied(), 64 * h, 0, u.kvh, u.tok0);
  } else {
    const int tiles = u.wide ? 2 : 1;
    bar_expect(sm.q_copied(), tiles * p.group * p.per_tile * 128 * (D / 64));
    for (int t = 0; t < tiles; ++t)
#pragma unroll
      for (int h = 0; h < D / 64; ++h)
        load_box(sm.query(t) + h * (kTile * 128), &p.q, sm.q_copied(), 64 * h, 0, u.kvh, u.tok0 + t * p.per_tile);
  }
}

// Key tiles, or (VALUES) value and query tiles.  Lane b of the warp copies box b
// of a tile: a page, or 128 tokens of one.  Boxes without a key that the item
// sees are left out; what the stage then holds in their place is masked (keys)
// or cleared (values).  The order of the tiles in the ring is that of their use:
// the first keys (one tile, or one for each stream), then values of tile n and
// keys of tile n + ahead; a loader's next place is at most 3 on, in a unit (2) and from
// one to the next alike: the last keys lie 3 before a unit's end, the first values 2
// after its start.  One warp for both took 2,400 cycles a tile pair, more
// than a pair of 64-component heads takes to arrive.
template <bool VALUES, int D, bool SPREAD, bool BITS8>
__device__ void load_role(const Params &p, const Smem<D, SPREAD, BITS8> &sm, const Guard &g, int first, int last) {
  constexpr int S = Shape<D, BITS8>::kCopied, kElement = Shape<D, BITS8>::kElement;
  const int lane = threadIdx.x % 32, boxes = kTile / p.box;
  const CUtensorMap *map = VALUES ? &p.v : &p.k;
  Ring<S> ring;
  uint32_t issued = 0, parity = 0;       // of each stage: the last copy into it
  uint32_t q_phase = 0, queries_out = 1;      // out: the last load's phase of q_full
  bool alive = true;
  for (int i = first; i < last && alive; ++i) {
    const Unit u = read_unit(p, i);
    if (!u.ntiles) continue;
    if (i + 1 < last) asm volatile("prefetch.global.L1 [%0];" ::"l"(p.units + i + 1));
    const int ahead = u.wide ? 1 : 2;
    const int *row = p.table + u.seq * p.table_stride;
    struct Box { int page, token; };       // INT_MIN: no box of this lane's
    auto box_of = [&](int n) {
      const int tile = u.tile0 + n, key = tile * kTile + lane * p.box;
      const bool wanted = n < u.ntiles && lane < boxes && key < u.hi && key + p.box > u.lo;
      // pages of less than a tile, or of whole tiles
      const int index = boxes > 1 ? tile * boxes + lane : p.tiles_a_page == 1 ? tile : tile / p.tiles_a_page;
      return Box{wanted ? max(-1, __ldg(row + index)) : INT_MIN, boxes > 1 ? 0 : (tile - index * p.tiles_a_page) * kTile};
    };
    Box b0 = box_of(0), b1 = box_of(1), b2 = box_of(2);
    // The queries go when the last unit's have been used, values meanwhile: only a
    // full ring waits for them.  (What spread units join in the second tile's place is
    // never in their way: a CTA's wide units come before its others.)
    bool queries_due = VALUES;
    auto queries = [&](bool now) {
      if (!now) {
        if (!__all_sync(~0u, bar_test(sm.q_empty(), q_phase ^ 1))) return;
      } else {
        alive = g.wait(sm.q_empty(), q_phase ^ 1, 5);
        if (!alive) return;
      }
      if (elected()) load_queries(p, sm, u);
      __syncwarp();
      queries_due = false;
      queries_out = q_phase;
    };
    int at = 0;                            // places of the ring behind this unit's first
    for (int n = 0; n < u.ntiles; ++n) {
      const int place = VALUES ? n + min(u.ntiles, n + ahead) : n < ahead ? n : 2 * n - ahead + 1;
      ring.next(place - at);
      at = place;
      const Box b3 = box_of(n + 3);
      if (VALUES && queries_due) {
        // whichever comes first: the queries' place or this tile's
        const uint64_t t0 = now_ns();
        for (;;) {
          queries(false);
          const bool room = bar_test(sm.copied_empty(ring.stage), ring.phase ^ 1);
          if (!queries_due || __any_sync(~0u, room || now_ns() - t0 > 1000000000ull)) break;
        }
      }
      alive = alive && g.wait(sm.copied_empty(ring.stage), ring.phase ^ 1, 1);
      if (!alive) break;
      const bool wanted = b0.page != INT_MIN;
      const uint32_t bar = sm.copied_full(ring.stage);
      const int count = __popc(__ballot_sync(~0u, wanted));
      if (elected()) bar_expect(bar, count * p.box * D * kElement);
      __syncwarp();
      if (wanted) {
        if (BITS8) {
          load_box(sm.copied(ring.stage) + lane * p.box * D, map, bar, 0, b0.token, u.kvh, b0.page);
        } else {
          const uint32_t dst = sm.stage(ring.stage) + lane * p.box * 128;
#pragma unroll
          for (int h = 0; h < D / 64; ++h) load_box(dst + h * (kTile * 128), map, bar, 64 * h, b0.token, u.kvh, b0.page);
        }
      }
      issued |= 1u << ring.stage;
      parity = (parity & ~(1u << ring.stage)) | ring.phase << ring.stage;
      b0 = b1;
      b1 = b2;
      b2 = b3;
    }
    if (VALUES) {
      if (alive && queries_due) queries(true);
      if (alive) q_phase ^= 1;
    }
    ring.next(2 * u.ntiles - at);
  }
  // copies in flight land before the CTA ends, also when their users gave up
  const uint64_t t0 = now_ns();
  if (!alive)
    for (int k = 0; k < S; ++k)
      while ((issued >> k & 1) && !bar_try(sm.copied_full(k), parity >> k & 1) && now_ns() - t0 < 100000000ull) {
      }
  if (VALUES)
    while (!bar_try(sm.q_copied(), queries_out) && now_ns() - t0 < 100000000ull) {
    }
}

__device__ __forceinline__ void load16(uint32_t at, uint32_t *r) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void store16(uint32_t at, const uint32_t *r) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
__device__ __forceinline__ uint32_t widened(uint32_t word, bool upper) {
  uint32_t r;
  if (upper)
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(word));
  else
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(word));
  return r;
}

// BITS8: 32 rows a warp, and 32 keys of each tile.
//
// Tiles go from where they arrive to f16 tiles for the products, in the ring's order;
// every 8-bit float is an f16.  A lane has 8 components of every second or fourth of
// its warp's keys, so that 16 lanes read 128 bytes in a row and 8 write a row's pieces,
// whose order is the 128-byte swizzle's.
//
// Queries (BF16: of bfloat16) become f16 where they lie, a row a lane, times the power of
// two that brings the row's largest to 2^14..2^15: exact for components down to 2^-29
// of it, and within 2^-40 of it below.  The softmax takes it back.
template <bool BF16, int D, bool SPREAD>
__device__ void widen_role(const Params &p, const Smem<D, SPREAD, true> &sm, const Guard &g, int first, int last) {
  using S = Shape<D, true>;
  constexpr int kOfRow = D / 8, kAtOnce = 32 / kOfRow;       // lanes of a row, rows at once
  const int warp = threadIdx.x / 32 - kWideningWarp, lane = threadIdx.x % 32;
  const int key = 32 * warp + lane / kOfRow, piece = lane % kOfRow;
  const uint32_t from = key * D + piece * 8, to = (piece / 8) * (kTile * 128) + key * 128 + ((piece % 8) ^ (key & 7)) * 16;
  Ring<S::kRawStages> raw;
  Ring<S::kStages> ring;
  uint32_t q_phase = 0;
  bool alive = true;
  auto tile = [&] {
    // (both asked at once: one after the other is 130 of a tile's 900 cycles)
    const bool here = bar_try(sm.copied_full(raw.stage), raw.phase) & bar_try(sm.empty(ring.stage), ring.phase ^ 1);
    alive = alive && (__all_sync(~0u, here) || (g.wait(sm.copied_full(raw.stage), raw.phase, 6) && g.wait(sm.empty(ring.stage), ring.phase ^ 1, 7)));
    if (alive) {
      const uint32_t src = sm.copied(raw.stage) + from, dst = sm.stage(ring.stage) + to;
#pragma unroll
      for (int k0 = 0; k0 < 32 / kAtOnce; k0 += 8) {
        uint32_t in[8][2];         // (reads under way together)
#pragma unroll
        for (int k = 0; k < 8; ++k)
          asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(in[k][0]), "=r"(in[k][1]) : "r"(src + (k0 + k) * kAtOnce * D) : "memory");
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t out[4] = {widened(in[k][0], false), widened(in[k][0], true), widened(in[k][1], false), widened(in[k][1], true)};
          store16((dst ^ ((k0 + k) * kAtOnce & 7) * 16) + (k0 + k) * kAtOnce * 128, out);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        bar_arrive(sm.full(ring.stage));
        bar_arrive(sm.copied_empty(raw.stage));
      }
    }
    raw.next();
    ring.next();
  };
  auto queries = [&](const Unit &u) {
    alive = alive && g.wait(sm.q_copied(), q_phase, 8);
    const int row = 32 * warp + lane, rows = u.ntok * p.group;
    if (alive && (spread(p, sm, u) ? lane < rows : row < rows)) {
      const uint32_t at = sm.query(0) + row * 128;
      auto both = [&](uint32_t x) {
        if (BF16) return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
        return __half22float2(*reinterpret_cast<__half2 *>(&x));
      };
      float top = 0.f;
#pragma unroll 4
      for (int k = 0; k < D / 8; ++k) {
        uint32_t in[4];
        load16(at + k / 8 * (kTile * 128) + ((k % 8) ^ (row & 7)) * 16, in);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = both(in[e]);
          top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      }
      const int up = top == 0.f ? 0 : min(14 - (int(__float_as_uint(top) >> 23) - 127), 120);
      const float by = __uint_as_float(uint32_t(up + 127) << 23);
#pragma unroll 4
      for (int k = 0; k < D / 8; ++k) {
        const uint32_t where = at + k / 8 * (kTile * 128) + ((k % 8) ^ (row & 7)) * 16;
        uint32_t x[4];
        load16(where, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = both(x[e]);
          x[e] = pack16<false>(f.x * by, f.y * by);
        }
        store16(where, x);
      }
      sm.powers(q_phase)[row] = static_cast<int8_t>(up);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0 && alive) bar_arrive(sm.q_full());
    q_phase ^= 1;
  };
  for (int i = first; i < last; ++i) {
    const Unit u = read_unit(p, i);
    if (!u.ntiles) continue;
    // the queries' place may be in use until the unit before is through with its keys
    for (int n = 0; n < min(2, u.ntiles); ++n) tile();
    queries(u);
    for (int n = 0; n < u.ntiles; ++n) {
      tile();
      if (n + 2 < u.ntiles) tile();
    }
  }
}

// 2^exponent of a head's keys (0) or values (1)
__device__ __forceinline__ int exponent_of(const Params &p, int which, int head) {
  return p.exponents ? min(max(__ldg(p.exponents + which * p.kv_heads + head), EMMY_MIN_EXPONENT), EMMY_MAX_EXPONENT) : 0;
}
template <bool BITS8> __device__ __forceinline__ float unscaled(const Params &p, const Unit &u) {
  return BITS8 ? __uint_as_float(uint32_t(exponent_of(p, 1, u.kvh) + 127) << 23) : 1.f;
}

// The products of stream t.  In a wide unit the streams issue in turn, so that
// one's products run while the other's softmax does; left alone they fall into
// step and wait for the exponentials and for the tensor cores together.  Both
// streams' warps walk the whole ring: a stage is free when both have arrived, the
// one that uses it by the completion of its products, the other at once.
template <bool BF16, int D, bool SPREAD, bool BITS8>
__device__ void mma_role(const Params &p, const Smem<D, SPREAD, BITS8> &sm, const Guard &g, int first, int last, uint32_t tmem, int t) {
  const int lane = threadIdx.x % 32;
  constexpr uint32_t kQk = instruction<BF16>(kTile, false), kPv = instruction<BF16>(D, true);
  const uint32_t s_at = tmem + kTile * t, o_at = tmem + 2 * kTile + kTile * t;
  Ring<Shape<D, BITS8>::kStages> ring;
  uint32_t q_phase = 0, p_phase = 0, turn_phase = t ^ 1;
  bool alive = true;
  auto wait = [&](uint32_t bar, uint32_t parity) { alive = alive && g.wait(bar, parity, 2); };
  auto issue_qk = [&](uint32_t a, uint32_t b, int stage) {   // S_t = Q K^T
    if (alive && elected()) {
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const int off = (k % 4) * 2 + (k / 4) * (kTile * 128 / 16);
        mma_ss(s_at, a + off, b + off, kOperandHigh, kQk, k > 0);
      }
      commit(sm.s_full(t));
      commit(sm.empty(stage));
    }
  };
  // O_t (+)= P_t V over 64 keys; quarters: 32 keys into the rows of one warp each
  auto issue_pv = [&](uint32_t b, int half, bool acc, bool quarters) {
    if (!alive || !elected()) return;
    if (quarters) {
#pragma unroll
      for (int k = 4 * half; k < 4 * half + 4; ++k)
        mma_ts_rows(o_at, s_at + 8 * k, b + k * (16 * 128 / 16), kOperandHigh, kPv, acc || k % 2, k / 2);
    } else {
#pragma unroll
      for (int k = 4 * half; k < 4 * half + 4; ++k)
        mma_ts(o_at, s_at + 8 * k, b + k * (16 * 128 / 16), kOperandHigh, kPv, acc || k > 0);
    }
  };
  auto take_turn = [&](bool wide) {
    if (!wide) return;
    wait(sm.turn(t), turn_phase);
    turn_phase ^= 1;
  };
  auto give_turn = [&](bool wide) {
    if (wide && alive && elected()) bar_arrive(sm.turn(t ^ 1));
  };
  auto pass_by = [&](int stage) {
    if (alive && lane == 0) bar_arrive(sm.empty(stage));
  };
  auto clear_values = [&](const Unit &u, int tile, int stage) {
    // values of keys that no token of the item sees are unwritten or another's:
    // their weight is 0, but 0 times an infinity is not.  Both warps of a wide
    // unit do it, each before its own products.
    const int key0 = (u.tile0 + tile) * kTile;
    const int above = min(kTile, max(0, u.hi - key0)), below = min(kTile, max(0, u.lo - key0));
    if (above == kTile && below == 0) return;
    constexpr int kChunks = D / 8;        // of 16 bytes a key
    for (int i = lane; i < (below + kTile - above) * kChunks; i += 32) {
      int key = i / kChunks;
      key = key < below ? key : key - below + above;
      const int chunk = i % kChunks;
      const uint32_t at = sm.stage(stage) + (chunk / 8) * (kTile * 128) + key * 128 + (chunk % 8) * 16;
      asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
  };
  for (int i = first; i < last; ++i) {
    const Unit u = read_unit(p, i);
    if (!u.ntiles) continue;
    const int ahead = u.wide ? 1 : 2;
    const bool quarters = spread(p, sm, u);
    const uint32_t q_op = operand(sm.query(u.wide ? t : 0), 16);
    wait(sm.q_full(), q_phase);
    q_phase ^= 1;
    auto done_with_queries = [&](bool products) {
      if (alive && elected()) {
        if (products)
          commit(sm.q_empty());
        else
          bar_arrive(sm.q_empty());
      }
    };
    for (int n = 0; n < min(ahead, u.ntiles); ++n) {
      wait(sm.full(ring.stage), ring.phase);
      if (u.wide || n == t) {
        take_turn(u.wide);
        fence_after();
        issue_qk(q_op, operand(sm.stage(ring.stage), 16), ring.stage);
        give_turn(u.wide);
        if (n + ahead >= u.ntiles) done_with_queries(true);
      } else {
        pass_by(ring.stage);
      }
      ring.next();
    }
    if (!u.wide && t >= u.ntiles) done_with_queries(false);
    for (int n = 0; n < u.ntiles; ++n) {
      const bool mine = u.wide || n % 2 == t, more = n + ahead < u.ntiles;
      const int v_stage = ring.stage;
      wait(sm.full(v_stage), ring.phase);
      ring.next();
      const int k_stage = ring.stage;
      if (mine) {
        if (alive) clear_values(u, n, v_stage);
        if (more) {
          wait(sm.full(k_stage), ring.phase);
          ring.next();
        }
        const uint32_t v_op = operand(sm.stage(v_stage), kTile * 128), k_op = operand(sm.stage(k_stage), 16);
        take_turn(u.wide);
        wait(sm.p_ready(t, 0), p_phase);
        fence_after();
        issue_pv(v_op, 0, n >= ahead, quarters);
        wait(sm.p_ready(t, 1), p_phase);
        p_phase ^= 1;
        fence_after();
        issue_pv(v_op, 1, quarters ? n >= ahead : true, quarters);
        if (more) issue_qk(q_op, k_op, k_stage);
        give_turn(u.wide);
        if (more) {
          if (n + 2 * ahead >= u.ntiles) done_with_queries(true);
        }
        if (alive && elected()) {
          if (!more) commit(sm.final(t));
          commit(sm.empty(v_stage));
        }
      } else {
        pass_by(v_stage);
        if (more) {
          wait(sm.full(k_stage), ring.phase);
          ring.next();
          pass_by(k_stage);
        }
      }
    }
  }
  // nothing of this thread's is in flight when the CTA gives up its memory
  if (elected()) commit(sm.drain(t));
  const uint64_t t0 = now_ns();
  while (!bar_try(sm.drain(t), 0) && now_ns() - t0 < 100000000ull) {
  }
}

__device__ __forceinline__ void group_sync(int id, int threads) {
  asm volatile("barrier.cta.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// 32 bytes of a row; at once where the address is on that grid.  A lane's rows
// lie apart, so that each store is a line of its own: fewer and larger ones are
// what counts (16-byte stores took 4 us a unit of 256 rows).
__device__ __forceinline__ void store32(void *at, const uint32_t *w, bool aligned32) {
  if (aligned32) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4 *>(at)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    reinterpret_cast<uint4 *>(at)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

// Reciprocal of a row's sum: 0 for a row that saw no key, NaN stays.
__device__ __forceinline__ float reciprocal(float l) { return l > 0.f ? __frcp_rn(l) : l; }
__device__ __forceinline__ float log_sum(float m, float l) { return l > 0.f ? (m + log2f(l)) * kLn2 : (l == 0.f ? -INFINITY : l); }

// The parts of `rows` rows, joined in their order: weights 2^(m - top), eight
// lanes a row and four rows a warp at once, so that 16 loads are in flight.
template <int D, bool BF16, bool BITS8> __device__ void join_parts(const Params &p, const Unit &u, int rows, int row0, int first_tok, int wid, int lane) {
  constexpr int kPieces = D / 32;           // of 4 components a lane
  const int64_t stride = int64_t(u.ntok) * p.group;
  for (int r = wid * 4 + lane / 8; r < rows; r += 16) {
    const int64_t at = u.part_row + row0 + r;
    float top = kNoMax, total = 0.f, acc[kPieces][4] = {};
#pragma unroll 4
    for (int s = 0; s < u.nsplit; ++s) top = fmaxf(top, __ldcg(p.part_ml + at + s * stride).x);
#pragma unroll 4
    for (int s = 0; s < u.nsplit; ++s) {
      const float2 ml = __ldcg(p.part_ml + at + s * stride);
      const float by = exp2_approx(ml.x - top);
      total += by * ml.y;
      const float4 *src = reinterpret_cast<const float4 *>(p.part_o + (at + s * stride) * D) + lane % 8;
#pragma unroll
      for (int k = 0; k < kPieces; ++k) {
        const float4 v = __ldcg(src + 8 * k);
        acc[k][0] += by * v.x, acc[k][1] += by * v.y, acc[k][2] += by * v.z, acc[k][3] += by * v.w;
      }
    }
    const float inv = reciprocal(total) * unscaled<BITS8>(p, u);
    const int64_t token = u.tok0 + first_tok + token_of(p, r);
    const int head = u.kvh * p.group + r - token_of(p, r) * p.group;
    uint2 *dst = reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.out) + token * p.out_stride[0] + head * p.out_stride[1]) + lane % 8;
#pragma unroll
    for (int k = 0; k < kPieces; ++k)
      dst[8 * k] = make_uint2(pack16<BF16>(acc[k][0] * inv, acc[k][1] * inv), pack16<BF16>(acc[k][2] * inv, acc[k][3] * inv));
    if (lane % 8 == 0 && p.lse) p.lse[token * p.q_heads + head] = log_sum(top, total);
  }
}

template <bool BF16, int D, bool SPREAD, bool BITS8>
__device__ void softmax_role(const Params &p, const Smem<D, SPREAD, BITS8> &sm, const Guard &g, int first, int last, uint32_t tmem) {
  // exponents may run 8 over the base before it moves; 16-bit floats of 5
  // exponent bits get a base 6 lower, so that small weights keep their bits
  // BITS8: all products are of f16, whatever the queries and results are
  constexpr bool kBrain = BF16 && !BITS8;
  constexpr float kShift = kBrain ? 0.f : 6.f, kGrow = 8.f;
  // with 64 components every fourth pair's exponentials off the exponential unit: 4
  // prompts of 4,096 tokens, 32 + 8 heads, 374 us against 387 with every eighth and 392
  // with none; 8 chunks of 1 to 511 over 12,288, 32 + 4 heads, 163 us against 166 with
  // every eighth.  With 128 components the tensor cores set the power: cycles saved
  // (3,030 -> 2,820 a tile pair) come back as a lower clock, nothing is gained
  constexpr int kPolyEvery = D == 128 ? kTile : 4;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, t = warp / 4, wid = warp % 4;
  const int row = threadIdx.x % kTile;
  const uint32_t lanes = tmem + (uint32_t(wid * 32) << 16);
  const uint32_t s_at = lanes + kTile * t, o_at = lanes + 2 * kTile + kTile * t;
  float c = p.scale_log2, c_power = p.scale_power;     // (BITS8: of a row)
  // a base of this size is off by 2^5 at most (the sums take that) or 1 (weights of 5 exponent bits)
  constexpr float kLarge = kBrain ? 0x1p29f : 0x1p24f;
  uint32_t s_phase = 0, f_phase = 0;
  [[maybe_unused]] int odd = 0;        // of the units with tiles
  bool alive = true;
  // this stream's tile of queries: its first token in the unit, and its rows
  const int row_token = token_of(p, row), row_head = row - row_token * p.group, lane_token = token_of(p, lane);
  auto first_token = [&](const Unit &u) { return u.wide ? t * p.per_tile : 0; };
  auto stream_rows = [&](const Unit &u) { return min(u.ntok - first_token(u), p.per_tile) * p.group; };
  // the keys that this thread's row sees; rows after the last take its place
  auto seen_by_row = [&](const Unit &u, int &lo, int &hi) {
    const int token = spread(p, sm, u) ? lane_token : row_token;
    const int pos = u.pos0 + first_token(u) + min(token, min(u.ntok - first_token(u), p.per_tile) - 1);
    hi = p.causal ? min(u.kv_len, pos + 1) : u.kv_len;
    lo = p.window ? max(0, pos - p.window + 1) : 0;
  };
  auto weights_stored = [&](int half) {
    tmem_st_wait();
    fence_before();
    __syncwarp();
    if (lane == 0) bar_arrive(sm.p_ready(t, half));
  };
  for (int i = first; i < last; ++i) {
    int step, key0, end;           // first key of a tile, and past the last
    int min_hi, max_lo;            // every row of the warp sees the keys between
    bool warp_active, quarter;     // quarter: of the keys
    {
      const Unit u = read_unit(p, i);
      quarter = spread(p, sm, u);
      warp_active = quarter || wid * 32 < stream_rows(u);
      int lo, hi;
      seen_by_row(u, lo, hi);
      min_hi = __reduce_min_sync(~0u, hi);
      max_lo = __reduce_max_sync(~0u, lo);
      step = u.wide ? kTile : 2 * kTile;
      key0 = (u.tile0 + (u.wide ? 0 : t)) * kTile;
      end = (u.tile0 + u.ntiles) * kTile;
    }
    // A base stands away from the product of score and c that it was rounded from, and
    // the multiply-add of the exponents, exact until its end, raises 2 to that: nothing
    // to a small base, 0 or infinity to a large one.  A row whose base is kLarge or more
    // multiplies by the power of two next to c instead, which is exact.  What that does
    // to scores a rounding apart is within the rounding of scores as large in 32 bits;
    // from 2^29 up different ones are 32 and more apart, and only the largest counts.
    if (BITS8) c = p.scale_log2;
    float m = kNoMax, l = 0.f, by_c = c;
    bool begun = false;
    // the base follows the row's maximum when that grows by more than 2^8: the
    // running sum and output (idle, the last product is complete) come down to it
    auto rebase = [&](float top) {
      const float best = __fmul_rn(top, by_c);
      const bool need = best - m > kShift + kGrow;      // (a large m + 14 would be rounded)
      if (!__any_sync(~0u, need)) return;
      float by = 1.f;
      if (need) {
        const float scaled = __fmul_rn(top, c), was = by_c;
        const bool large = fabsf(scaled) >= kLarge;
        by_c = large ? c_power : c;
        const float to = large ? __fmul_rn(top, by_c) : scaled - kShift;
        by = exp2_approx(was == by_c ? m - to : m * (c / was) - (large ? scaled : to));
        m = to;
      }
      l *= by;
      if (!begun) return;
      const uint64_t by2 = pair(by, by);
#pragma unroll 1
      for (int k = 0; k < D; k += 16) {
        uint32_t o[16];
        tmem_ld16(o_at + k, o);
        tmem_ld_wait(o);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          float e, f;
          unpair(mul2(pair(__uint_as_float(o[2 * q]), __uint_as_float(o[2 * q + 1])), by2), e, f);
          o[2 * q] = __float_as_uint(e);
          o[2 * q + 1] = __float_as_uint(f);
        }
        tmem_st16(o_at + k, o);
      }
    };
    for (; key0 < end; key0 += step) {
      alive = alive && g.wait(sm.s_full(t), s_phase, 3);
      s_phase ^= 1;
      if (BITS8 && !begun) {
        const int power = exponent_of(p, 0, read_unit(p, i).kvh) - sm.powers(odd)[row];
        auto of_row = [&](float x) { return fminf(fmaxf(ldexpf(x, power), FLT_MIN), FLT_MAX); };
        by_c = c = of_row(p.scale_log2);
        c_power = of_row(p.scale_power);
      }
      if (quarter && alive) {
        fence_after();
        uint32_t s[32], w[16];
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        tmem_ld32(s_at + 32 * wid, s);
        tmem_ld_wait(s);
        const int base = key0 + 32 * wid;
        if (base < max_lo || base + 32 > min_hi) {
          int lo, hi;
          seen_by_row(read_unit(p, i), lo, hi);
          const int from = lo - base;
          const unsigned span = max(0, hi - lo);
#pragma unroll
          for (int k = 0; k < 32; ++k)
            if (unsigned(k - from) >= span) s[k] = __float_as_uint(-INFINITY);
        }
#pragma unroll
        for (int k = 0; k < 32; k += 8)
#pragma unroll
          for (int q = 0; q < 4; ++q) top[q] = max3(__float_as_uint(top[q]), s[k + q], s[k + 4 + q]);
        rebase(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
        const uint64_t c2 = pair(by_c, by_c), base2 = pair(-m, -m);
        uint64_t part[2] = {0, 0};
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          float e, f;
          unpair(fma2(pair(__uint_as_float(s[2 * q]), __uint_as_float(s[2 * q + 1])), c2, base2), e, f);
          e = exp2_approx(e);
          f = exp2_approx(f);
          part[q % 2] = add2(part[q % 2], pair(e, f));
          w[q] = pack16<kBrain>(e, f);
        }
        tmem_st16(s_at + 16 * wid, w);
        weights_stored(0);
        if (lane == 0) bar_arrive(sm.p_ready(t, 1));
        float even, odd;
        unpair(add2(part[0], part[1]), even, odd);
        l += even + odd;
      } else if (warp_active && alive) {
        fence_after();
        if (key0 < max_lo || key0 + kTile > min_hi) {
          // some row of the warp does not see the whole tile: the scores are
          // masked where they lie, so that the way below has no branches
          int lo, hi;
          seen_by_row(read_unit(p, i), lo, hi);
          const int from = lo - key0;
          const unsigned span = max(0, hi - lo);
#pragma unroll 1
          for (int column = 0; column < kTile; column += 16) {
            uint32_t v[16];
            tmem_ld16(s_at + column, v);
            tmem_ld_wait(v);
#pragma unroll
            for (int k = 0; k < 16; ++k)
              if (unsigned(column + k - from) >= span) v[k] = __float_as_uint(-INFINITY);
            tmem_st16(s_at + column, v);
          }
          tmem_st_wait();
        }
        // the row's scores stay in registers
        uint32_t s[kTile];
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        auto take_in = [&](int from) {
#pragma unroll
          for (int k = from; k < from + 64; k += 8)
#pragma unroll
            for (int q = 0; q < 4; ++q) top[q] = max3(__float_as_uint(top[q]), s[k + q], s[k + 4 + q]);
        };
        tmem_ld32(s_at, s);
        tmem_ld32(s_at + 32, s + 32);
        tmem_ld_wait(s, 0, 64);
        tmem_ld32(s_at + 64, s + 64);
        tmem_ld32(s_at + 96, s + 96);
        take_in(0);
        tmem_ld_wait(s, 64, 128);
        take_in(64);
        rebase(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
        const uint64_t c2 = pair(by_c, by_c);
        const uint64_t base2 = pair(-m, -m);
        uint64_t part[4] = {0, 0, 0, 0};
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          // a branch that is always taken keeps the last chunk's exponentials
          // from being scheduled before the first half is handed on
          if (h == 3 && !p.group) break;
          uint32_t w[16];
#pragma unroll
          for (int q = 0; q < 16; ++q) {
            uint64_t x = fma2(pair(__uint_as_float(s[32 * h + 2 * q]), __uint_as_float(s[32 * h + 2 * q + 1])), c2, base2);
            float e, f;
            if (q % kPolyEvery == kPolyEvery - 1) {
              x = exp2_pair(x);
              unpair(x, e, f);
            } else {
              unpair(x, e, f);
              e = exp2_approx(e);
              f = exp2_approx(f);
              x = pair(e, f);
            }
            part[q % 4] = add2(part[q % 4], x);
            w[q] = pack16<kBrain>(e, f);
          }
          if (h == 2) weights_stored(0);      // of the first 64 keys
          tmem_st16(s_at + 16 * h, w);
        }
        weights_stored(1);
        float even, odd;
        unpair(add2(add2(part[0], part[1]), add2(part[2], part[3])), even, odd);
        l += even + odd;
      } else {
        __syncwarp();
        if (lane == 0) {
          bar_arrive(sm.p_ready(t, 0));
          bar_arrive(sm.p_ready(t, 1));
        }
      }
      begun = true;
    }

    // ------------------------------------------------------------ the unit's end
    const Unit u = read_unit(p, i);
    if (BITS8 && u.ntiles) odd ^= 1;
    const int rows = stream_rows(u), row0 = first_token(u) * p.group;
    const bool joined = !u.wide && u.ntiles > 1;      // stream 1 saw keys too
    if (begun) {
      alive = alive && g.wait(sm.final(t), f_phase, 4);
      f_phase ^= 1;
      fence_after();
    }
    if (by_c != c) m *= c / by_c;        // from here on every row's base is one of c
    float by0 = 1.f, by1 = 0.f;
    if (joined) {
      if (t == 1) sm.ml()[row] = make_float2(m, l);
      fence_before();
      group_sync(3, 256);           // stream 1's output is complete as well
      if (t == 0) {
        const float2 other = sm.ml()[row];
        const float top = fmaxf(m, other.x);
        by0 = exp2_approx(m - top);
        by1 = exp2_approx(other.x - top);
        l = l * by0 + other.y * by1;
        m = top;
      }
    }
    if (t == 0 || u.wide) {
      fence_after();
      const bool split = u.nsplit > 1;
      const int64_t split_row = u.part_row + int64_t(u.split) * u.ntok * p.group + row0;
      if (quarter) {
        // the four warps' results come down to one base and meet in shared memory,
        // as many columns at a time as fit for 8, 16 or 32 rows:
        // [warp][row][pieces of 16 bytes], the pieces of a row in an order of its
        // own so that neither side meets in a bank
        const uint32_t scratch = sm.query(1);
        asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(scratch + row * 8), "f"(m), "f"(l) : "memory");
        group_sync(1, kTile);
        float ms[4], ls[4], top = kNoMax, total = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(ms[w]), "=f"(ls[w]) : "r"(scratch + (32 * w + lane) * 8) : "memory");
          top = fmaxf(top, ms[w]);
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) total += exp2_approx(ms[w] - top) * ls[w];
        const float scale = exp2_approx(m - top) * (split ? 1.f : reciprocal(total) * unscaled<BITS8>(p, u));
        const uint64_t f0 = pair(by0 * scale, by0 * scale), f1 = pair(by1 * scale, by1 * scale);
        group_sync(1, kTile);
        const int fit = rows <= 8 ? 7 : rows <= 16 ? 6 : 5;           // log2 of the columns
        const int shift = min(fit, D == 128 ? 7 : 6) - 2, pieces = 1 << shift;
        const uint32_t mine = scratch + ((wid << (10 - fit)) + lane) * (pieces * 16);
#pragma unroll 1
        for (int first_column = 0; first_column < D; first_column += 4 * pieces) {
          if (first_column) group_sync(1, kTile);
#pragma unroll 1
          for (int k = 0; k < 4 * pieces; k += 32) {
            uint32_t o[32], o1[32];
            tmem_ld32(o_at + first_column + k, o);
            if (joined) tmem_ld32(o_at + kTile + first_column + k, o1);
            tmem_ld_wait(o);
            tmem_ld_wait(o1);
            if (lane < rows) {
#pragma unroll
              for (int q = 0; q < 32; q += 4) {
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; r += 2) {
                  uint64_t x = mul2(pair(__uint_as_float(o[q + r]), __uint_as_float(o[q + r + 1])), f0);
                  if (joined) x = fma2(pair(__uint_as_float(o1[q + r]), __uint_as_float(o1[q + r + 1])), f1, x);
                  unpair(x, v[r], v[r + 1]);
                }
                asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(mine + ((k + q) / 4 ^ (lane & 7)) * 16), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]) : "memory");
              }
            }
            __syncwarp();
          }
          group_sync(1, kTile);
          for (int item = row; item < rows << shift; item += kTile) {
            const int r = item >> shift, piece = item & (pieces - 1);
            float sum[4] = {};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              float v[4];
              const uint32_t at = scratch + (((w << (10 - fit)) + r) * pieces + (piece ^ (r & 7))) * 16;
              asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(at) : "memory");
#pragma unroll
              for (int e = 0; e < 4; ++e) sum[e] += v[e];
            }
            if (!alive) continue;
            if (split) {
              __stcg(reinterpret_cast<float4 *>(p.part_o + (split_row + r) * D + first_column) + piece, make_float4(sum[0], sum[1], sum[2], sum[3]));
            } else {
              const int token = token_of(p, r);
              uint16_t *to = static_cast<uint16_t *>(p.out) + int64_t(u.tok0 + token) * p.out_stride[0] +
                             (u.kvh * p.group + r - token * p.group) * p.out_stride[1] + first_column;
              reinterpret_cast<uint2 *>(to)[piece] = make_uint2(pack16<BF16>(sum[0], sum[1]), pack16<BF16>(sum[2], sum[3]));
            }
          }
        }
        group_sync(1, kTile);
        if (wid == 0 && lane < rows && alive) {
          if (split)
            __stcg(p.part_ml + split_row + lane, make_float2(top, total));
          else if (p.lse)
            p.lse[int64_t(u.tok0 + lane_token) * p.q_heads + u.kvh * p.group + lane - lane_token * p.group] = log_sum(top, total);
        }
      } else if (warp_active && alive) {
        const bool mine = row < rows;
        const int64_t out_token = u.tok0 + first_token(u) + row_token, part = split_row + row;
        const int head = u.kvh * p.group + row_head;
        const float inv = split ? 1.f : reciprocal(l) * unscaled<BITS8>(p, u);
        const uint64_t f0 = pair(by0 * inv, by0 * inv), f1 = pair(by1 * inv, by1 * inv);
        char *to = split ? reinterpret_cast<char *>(p.part_o + part * D)
                         : static_cast<char *>(p.out) + 2 * (out_token * p.out_stride[0] + head * p.out_stride[1]);
#pragma unroll 1
        for (int k = 0; k < D; k += 32) {
          uint32_t o[32];
          if (begun) {
            tmem_ld32(o_at + k, o);
            tmem_ld_wait(o);
          } else {
#pragma unroll
            for (int q = 0; q < 32; ++q) o[q] = 0;
          }
#pragma unroll
          for (int q = 0; q < 32; q += 2) {
            float x, y;
            unpair(mul2(pair(__uint_as_float(o[q]), __uint_as_float(o[q + 1])), f0), x, y);
            o[q] = __float_as_uint(x);
            o[q + 1] = __float_as_uint(y);
          }
          if (joined) {
            uint32_t o1[32];
            tmem_ld32(o_at + kTile + k, o1);
            tmem_ld_wait(o1);
#pragma unroll
            for (int q = 0; q < 32; q += 2) {
              float x, y;
              unpair(fma2(pair(__uint_as_float(o1[q]), __uint_as_float(o1[q + 1])), f1,
                          pair(__uint_as_float(o[q]), __uint_as_float(o[q + 1]))), x, y);
              o[q] = __float_as_uint(x);
              o[q + 1] = __float_as_uint(y);
            }
          }
          if (mine && split) {
#pragma unroll
            for (int q = 0; q < 32; q += 8) store32(to + 4 * (k + q), o + q, true);
          } else if (mine) {
#pragma unroll
            for (int q = 0; q < 32; q += 16) {
              uint32_t w[8];
#pragma unroll
              for (int r = 0; r < 8; ++r)
                w[r] = pack16<BF16>(__uint_as_float(o[q + 2 * r]), __uint_as_float(o[q + 2 * r + 1]));
              store32(to + 2 * (k + q), w, p.aligned32);
            }
          }
        }
        if (mine && split) __stcg(p.part_ml + part, make_float2(m, l));
        if (mine && !split && p.lse) p.lse[out_token * p.q_heads + head] = log_sum(m, l);
      }
      fence_before();
      if (split) {
        // the stream that arrives last joins the parts
        __threadfence();
        group_sync(1 + t, kTile);
        if (row == 0) {
          unsigned *counter = p.counters + 2 * u.item + t;
          const bool is_last = alive && atomicAdd(counter, 1u) == unsigned(u.nsplit - 1);
          if (is_last) *counter = 0;
          __threadfence();
          sm.words()[2 + t] = is_last;
        }
        group_sync(1 + t, kTile);
        if (sm.words()[2 + t]) join_parts<D, BF16, BITS8>(p, u, rows, row0, first_token(u), wid, lane);
      }
    }
    if (joined) group_sync(3, 256);       // stream 1's output and sums have been read
  }
}

template <int D, bool BF16, bool SPREAD, bool BITS8>
__global__ void __launch_bounds__(Warps<BITS8>::kThreads, 1) paged_attention_kernel(const __grid_constant__ Params p) {
  using S = Shape<D, BITS8>;
  extern __shared__ char raw[];
  Smem<D, SPREAD, BITS8> sm;
  sm.base = (smem_addr(raw) + 1023) & ~1023u;
  const int warp = threadIdx.x / 32;
  // the first unit is on its way while the CTA sets itself up
  const unsigned status = threadIdx.x == 0 ? __ldcg(p.status) | __ldcg(p.batch_status) : 0;
  const int first = __ldg(p.cta_first + blockIdx.x), last = __ldg(p.cta_first + blockIdx.x + 1);
  asm volatile("prefetch.global.L1 [%0];" ::"l"(p.units + first));
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      bar_init(sm.full(s), BITS8 ? 4 : 1);
      bar_init(sm.empty(s), 2);
    }
    for (int s = 0; s < S::kRawStages; ++s) {
      bar_init(sm.copied_full(s), 1);
      bar_init(sm.copied_empty(s), 4);
    }
    if (BITS8) bar_init(sm.q_copied(), 1);
    bar_init(sm.q_full(), BITS8 ? 4 : 1);
    bar_init(sm.q_empty(), 2);
    for (int t = 0; t < 2; ++t) {
      bar_init(sm.s_full(t), 1);
      bar_init(sm.p_ready(t, 0), 4);
      bar_init(sm.p_ready(t, 1), 4);
      bar_init(sm.final(t), 1);
      bar_init(sm.drain(t), 1);
      bar_init(sm.turn(t), 1);
    }
    sm.words()[0] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(const_cast<int *>(sm.words() + 1))) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  // an earlier call that gave up left counters and parts as they were: nothing is started over them
  const bool gave_up = __syncthreads_or(status);
  fence_after();
  const uint32_t tmem = __reduce_or_sync(~0u, sm.words()[1]);
  if (gave_up) {
    if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    return;
  }
  const Guard g{sm.base + S::kWords, p};
  if (warp < kSoftmaxWarps) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Warps<BITS8>::kSoftmaxRegs));
    softmax_role<BF16>(p, sm, g, first, last, tmem);
    // an end of their own: code shared with the other warps would have to do
    // with their registers
    __syncwarp();
    fence_before();
    asm volatile("barrier.cta.sync 0;" ::: "memory");
    return;
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Warps<BITS8>::kOtherRegs));
    if (BITS8 && warp >= kWideningWarp) {
      if constexpr (BITS8) widen_role<BF16>(p, sm, g, first, last);
    } else if (warp >= kMmaWarp)
      mma_role<BF16 && !BITS8>(p, sm, g, first, last, tmem, warp - kMmaWarp);
    else if (warp == kKeyWarp)
      load_role<false>(p, sm, g, first, last);
    else
      load_role<true>(p, sm, g, first, last);
  }
  __syncwarp();
  fence_before();
  asm volatile("barrier.cta.sync 0;" ::: "memory");
  if (warp == kMmaWarp) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
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

// A stride in bytes; that of an extent of 1 is never used, whatever it says.
uint64_t step(int64_t stride, int64_t extent, int element = 2) { return extent == 1 ? 16 : static_cast<uint64_t>(stride) * element; }
bool bad_stride(int64_t stride, int64_t extent, int grid = 8) {
  return extent != 1 && (stride <= 0 || stride % grid || stride >= (int64_t(1) << 38));
}

template <int D, bool BF16, bool SPREAD, bool BITS8> int launch(const Params &p, int ctas, cudaStream_t s) {
  static std::atomic<uint64_t> ready{0};     // a bit for each device
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return cuda_fail("emmy_paged_attention: cudaGetDevice", e);
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (dev > 63 || !(ready.load() & bit)) {
    if (cudaError_t e = cudaFuncSetAttribute(paged_attention_kernel<D, BF16, SPREAD, BITS8>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem))
      return cuda_fail("emmy_paged_attention: shared memory", e);
    // the softmax warps wait for the registers of the split: they must exist
    cudaFuncAttributes attr;
    if (cudaError_t e = cudaFuncGetAttributes(&attr, paged_attention_kernel<D, BF16, SPREAD, BITS8>))
      return cuda_fail("emmy_paged_attention: attributes", e);
    if (attr.numRegs != Warps<BITS8>::kLaunchRegs)
      return fail("emmy_paged_attention: built with %ld registers, not %ld", attr.numRegs, Warps<BITS8>::kLaunchRegs);
    if (dev <= 63) ready.fetch_or(bit);
  }
  paged_attention_kernel<D, BF16, SPREAD, BITS8><<<ctas, Warps<BITS8>::kThreads, kSmem, s>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : cuda_fail("emmy_paged_attention: launch", e);
}

// bits8: the caches hold 8-bit floats, with `exponents`; batch_status: of the plan that
// this one is a part of, or 0
int run(emmy_paged_plan_t plan, const emmy_paged_attention_args *a, bool bits8, uint64_t exponents, uint64_t batch_status, void *stream) {
  if (!plan || !a) return fail("emmy_paged_attention: bad argument");
  if (bits8 && !plan->narrow) return fail("emmy_paged_attention: a plan with wide units");
  if (a->dtype != 6 && a->dtype != 9) return fail("emmy_paged_attention: dtype %ld (f16 or bf16)", a->dtype);
  if (!(a->scale > 0.f) || !std::isfinite(a->scale * kLog2e)) return fail("emmy_paged_attention: scale must be positive and finite");
  if (plan->tokens == 0) return 0;
  const int ps = a->page_size;
  const bool reads = plan->tiled || plan->spread;     // some unit sees a key
  if (ps < 8 || (ps < kTile ? (ps & (ps - 1)) != 0 : ps % kTile != 0))
    return fail("emmy_paged_attention: page_size %ld (8, 16, 32, 64 or a multiple of 128)", ps);
  if (a->pages < (reads ? 1 : 0)) return fail("emmy_paged_attention: a cache of %ld pages", a->pages);
  if (a->table_width < 0 || int64_t(a->table_width) * ps < plan->max_kv)
    return fail("emmy_paged_attention: a table of %ld pages a sequence does not hold %ld tokens", a->table_width, plan->max_kv);
  if (!a->q || !a->out || (reads && (!a->k_cache || !a->v_cache || !a->table)) || !a->plan_words || (plan->part_rows && !a->scratch))
    return fail("emmy_paged_attention: null address");
  if ((a->q | a->out | a->k_cache | a->v_cache | a->plan_words) % 16 || a->scratch % 32 || (a->table | a->lse) % 4)
    return fail("emmy_paged_attention: address not a multiple of 16 bytes (scratch: 32)");
  const int group = plan->q_heads / plan->kv_heads, d = plan->head_dim;
  const int64_t extent[3] = {a->pages, ps, plan->kv_heads};
  for (int i = 0; i < 3 && reads; ++i)
    if (bad_stride(a->k_cache_stride[i], extent[i], bits8 ? 16 : 8) || bad_stride(a->v_cache_stride[i], extent[i], bits8 ? 16 : 8))
      return fail("emmy_paged_attention: cache stride %ld not a positive multiple of %ld elements", i, bits8 ? 16 : 8);
  const int64_t rows[2] = {plan->tokens, plan->q_heads};
  for (int i = 0; i < 2; ++i)
    if (bad_stride(a->q_stride[i], rows[i]) || bad_stride(a->out_stride[i], rows[i]))
      return fail("emmy_paged_attention: q or out stride %ld not a positive multiple of 8 elements", i);
  Params p;
  memset(&p, 0, sizeof p);
  const uint32_t box = ps < kTile ? ps : kTile;
  const int per_tile = kTile / group;
  const uint64_t q_dims[4] = {uint64_t(d), uint64_t(group), uint64_t(plan->kv_heads), uint64_t(plan->tokens)};
  const uint64_t q_steps[3] = {step(a->q_stride[1], plan->q_heads), group * step(a->q_stride[1], plan->q_heads), step(a->q_stride[0], plan->tokens)};
  const uint32_t q_box[4] = {64, uint32_t(group), 1, uint32_t(per_tile)};
  const uint32_t q32_box[4] = {64, uint32_t(group), 1, uint32_t(group <= 32 ? 32 / group : 1)};
  // (each map costs the caller half a microsecond: only those that a unit uses)
  if (plan->tiled)
    if (int e = emmy_tensormap_encode(&p.q, a->dtype, 4, a->q, q_dims, q_steps, q_box, 3)) return e;
  if (plan->spread)
    if (int e = emmy_tensormap_encode(&p.q32, a->dtype, 4, a->q, q_dims, q_steps, q32_box, 3)) return e;
  const uint64_t dims[4] = {uint64_t(d), uint64_t(ps), uint64_t(plan->kv_heads), uint64_t(a->pages)};
  const uint32_t kv_box[4] = {bits8 ? uint32_t(d) : 64, box, 1, 1};
  const int element = bits8 ? 1 : 2;
  for (int i = 0; i < 2 && reads; ++i) {
    const int64_t *st = i ? a->v_cache_stride : a->k_cache_stride;
    const uint64_t steps[3] = {step(st[1], ps, element), step(st[2], plan->kv_heads, element), step(st[0], a->pages, element)};
    // (8-bit tiles, type 0 and without a swizzle, are read and written on by threads)
    if (int e = emmy_tensormap_encode(i ? &p.v : &p.k, bits8 ? 0 : a->dtype, 4, i ? a->v_cache : a->k_cache, dims, steps, kv_box, bits8 ? 0 : 3)) return e;
  }
  int *words = reinterpret_cast<int *>(a->plan_words);
  p.status = reinterpret_cast<unsigned *>(words);
  p.batch_status = batch_status ? reinterpret_cast<unsigned *>(batch_status) : p.status;
  p.cta_first = words + 4;
  p.counters = reinterpret_cast<unsigned *>(words + plan->at.counters);
  p.units = reinterpret_cast<const Unit *>(words + plan->at.units);
  p.table = reinterpret_cast<const int *>(a->table);
  p.table_stride = a->table_stride;
  p.part_o = reinterpret_cast<float *>(a->scratch);
  p.part_ml = reinterpret_cast<float2 *>(p.part_o + plan->part_rows * d);
  p.out = reinterpret_cast<void *>(a->out);
  p.out_stride[0] = a->out_stride[0];
  p.out_stride[1] = a->out_stride[1];
  p.lse = reinterpret_cast<float *>(a->lse);
  p.q_heads = plan->q_heads;
  p.group = group;
  p.group_inverse = (65536 + group - 1) / group;
  p.per_tile = per_tile;
  p.tiles_a_page = ps < kTile ? 1 : ps / kTile;
  p.box = box;
  p.aligned32 = (a->out % 32 == 0) && (rows[0] == 1 || a->out_stride[0] % 16 == 0) && (rows[1] == 1 || a->out_stride[1] % 16 == 0);
  p.causal = plan->causal;
  p.window = plan->window;
  p.scale_log2 = a->scale * kLog2e;
  int exponent = 0;
  const float mantissa = std::frexp(p.scale_log2, &exponent);      // 1/2 to 1
  p.scale_power = std::ldexp(1.f, std::min(127, mantissa * mantissa < 0.5f ? exponent - 1 : exponent));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  p.exponents = reinterpret_cast<const int *>(exponents);
  p.kv_heads = plan->kv_heads;
  const int n = plan->at.ctas;
  if (bits8) {
    if (d == 128) return a->dtype == 9 ? launch<128, true, true, true>(p, n, s) : launch<128, false, true, true>(p, n, s);
    return a->dtype == 9 ? launch<64, true, true, true>(p, n, s) : launch<64, false, true, true>(p, n, s);
  }
  if (plan->spread) {
    if (d == 128) return a->dtype == 9 ? launch<128, true, true, false>(p, n, s) : launch<128, false, true, false>(p, n, s);
    return a->dtype == 9 ? launch<64, true, true, false>(p, n, s) : launch<64, false, true, false>(p, n, s);
  }
  if (d == 128) return a->dtype == 9 ? launch<128, true, false, false>(p, n, s) : launch<128, false, false, false>(p, n, s);
  return a->dtype == 9 ? launch<64, true, false, false>(p, n, s) : launch<64, false, false, false>(p, n, s);
}

}  // namespace

extern "C" EMMY_API int emmy_paged_attention(emmy_paged_plan_t plan, const emmy_paged_attention_args *a, void *stream) {
  return run(plan, a, false, 0, 0, stream);
}

int emmy_internal_paged_attention(emmy_paged_plan_t plan, const emmy_paged_attention_args *a, bool bits8, uint64_t exponents, uint64_t batch_status,
                                  void *stream) {
  return run(plan, a, bits8, exponents, batch_status, stream);
}

extern "C" EMMY_API int emmy_paged_plan_status(emmy_paged_plan_t plan, uint64_t plan_words, void *stream) {
  if (!plan || !plan_words) return fail("emmy_paged_plan_status: bad argument");
  int status = 0;
  if (int e = emmy_memcpy_dtoh_async(&status, plan_words, sizeof status, stream)) return e;
  if (int e = emmy_stream_sync(stream)) return e;
  if (!status) return 0;
  char buf[128];
  snprintf(buf, sizeof buf, "emmy_paged_attention: a wait ran out (code %d)", status);
  return emmy_internal_fail(EMMY_EKERNEL, buf);
}
