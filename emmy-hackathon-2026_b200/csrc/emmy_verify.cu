// emmy_verify.cu -- drafted tokens against the target's probabilities.
//
// Draft x of probability q(x) is kept while u q(x) < p(x); the token after those kept
// is drawn from max(p - q, 0) at the first draft that is not, from p after the last:
// the first j with p_0 + .. + p_j > v (the whole sum).  Then every token is distributed
// as the target's.
//
// One pass over one row of p and one of q a sequence, which is the floor: 8 bytes an
// element of the vocabulary.  A cluster of up to 8 CTAs has a sequence; each warp sums
// a segment of the vocabulary, every CTA adds the segments' sums of its cluster in their
// order (distributed shared memory), and the CTA with the segment in which v falls goes
// through that segment again, a thread a few elements.  Nothing is kept between calls.
//
// Products, differences and sums are in 64 bits.  Products and differences of 32-bit
// numbers are exact or off by 2^-53.  A sum of numbers that are not negative is off by
// 2^-53 of it for each addition on an element's way: those of its lane one after the
// other (64 of 131,071 elements over 8 CTAs, 512 over one) and 30 or so of lanes, segments
// and threads.  So a token is another one than with exact sums only if v comes within twice
// that of a border: 2^-45 there, 2^-42 over one CTA, more as the vocabulary grows.  (Sums
// one after the other in 64 bits are off by up to 2^-36 of as many.)  Sums in 32 bits of
// 131,071 elements would move borders by 1e-6 and one token in a hundred.  At the rate of
// the memory an SM has 3 elements a cycle, for which the conversions and additions in 64
// bits suffice.
#include "../../include/emmy_b200.h"

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <climits>
#include <cstdint>
#include <cstdio>

namespace cg = cooperative_groups;

int emmy_internal_fail(int code, const char *msg);   // emmy_runtime.cpp
int emmy_internal_sms(int *sms);                     // emmy_rotate_append.cu

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kMostCtas = 8;
static_assert(kMostCtas * kWarps <= 64, "two segments a lane");
constexpr int kEach = 8;             // elements of a thread where the token lies
constexpr int kBatch = 16;           // elements of a thread that are loaded together, of both rows

__device__ __forceinline__ double wide(float x) { return double(x); }
__device__ __forceinline__ double wide(__half x) { return double(__half2float(x)); }
__device__ __forceinline__ double wide(__nv_bfloat16 x) { return double(__bfloat162float(x)); }

// blockIdx.x: sequence x CTAs of its cluster + CTA.
template <typename T> __global__ void __launch_bounds__(kThreads, 4) verify_kernel(const __grid_constant__ emmy_verify_args a) {
  __shared__ double sums[kWarps], warp_sums[kWarps];
  __shared__ int kept_shared, segment_shared, positive_shared[kWarps], token_shared[kWarps];
  __shared__ double target_shared, before_shared;
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = cluster.num_blocks(), rank = cluster.block_rank(), seq = blockIdx.x / ctas;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int *const first = reinterpret_cast<const int *>(a.first);
  const int begin = first[seq], end = first[seq + 1];
  const int64_t draft0 = int64_t(begin) - seq;      // of the sequence's drafts: every earlier sequence has one row more
  const bool valid = begin >= 0 && end > begin && end <= a.rows && draft0 >= 0 && int64_t(end) - 1 - seq <= a.drafts;
  if (!valid) {                                     // (alike in all of a cluster's threads)
    if (rank == 0 && tid == 0) reinterpret_cast<int *>(a.accepted)[seq] = -1;
    return;
  }
  const int n = end - begin - 1;
  const int *const drafted = reinterpret_cast<const int *>(a.drafted) + draft0;
  const T *const target = reinterpret_cast<const T *>(a.target), *const proposal = reinterpret_cast<const T *>(a.proposal);

  // ---------------------------------------------------------------- drafts kept
  if (tid == 0) kept_shared = n;
  __syncthreads();
  for (int i = tid; i < n; i += kThreads) {
    const int x = drafted[i];
    bool keep = false;
    if (x >= 0 && x < a.vocabulary) {
      const double p = wide(target[(begin + i) * a.target_stride + x]);
      const double q = proposal ? wide(proposal[(draft0 + i) * a.proposal_stride + x]) : 1.0;
      keep = double(reinterpret_cast<const float *>(a.uniforms)[draft0 + i]) * q < p;
    }
    if (!keep) atomicMin(&kept_shared, i);
  }
  __syncthreads();
  const int kept = kept_shared;
  int *const tokens = reinterpret_cast<int *>(a.tokens) + begin;
  if (rank == 0) {
    if (tid == 0) reinterpret_cast<int *>(a.accepted)[seq] = kept;
    for (int i = tid; i <= n; i += kThreads)
      if (i != kept) tokens[i] = i < kept ? drafted[i] : -1;
  }

  // ---------------------------------------------------------------- the next token
  const T *const p_row = target + (begin + kept) * a.target_stride;
  const T *q_row = kept < n && proposal ? proposal + (draft0 + kept) * a.proposal_stride : nullptr;
  int without = kept < n && !proposal ? drafted[kept] : -1;      // certain drafts: q is 1 there
  const int segments = ctas * kWarps, length = (a.vocabulary + segments - 1) / segments;
  auto segment_begin = [&](int s) { return min(a.vocabulary, s * length); };
  auto mass = [&](int j) {
    double d = wide(p_row[j]);
    if (q_row) d -= wide(q_row[j]);
    return d > 0.0 && j != without ? d : 0.0;
  };
  for (int pass = 0;; ++pass) {
    {
      const int s = rank * kWarps + warp, to = segment_begin(s + 1);
      double sum = 0.0;
      int j = segment_begin(s) + lane;
      if (q_row) {
        for (; j + 32 * (kBatch / 2 - 1) < to; j += 32 * (kBatch / 2)) {
          T x[kBatch / 2], y[kBatch / 2];
#pragma unroll
          for (int k = 0; k < kBatch / 2; ++k) x[k] = p_row[j + 32 * k];
#pragma unroll
          for (int k = 0; k < kBatch / 2; ++k) y[k] = q_row[j + 32 * k];
#pragma unroll
          for (int k = 0; k < kBatch / 2; ++k) {
            const double d = wide(x[k]) - wide(y[k]);
            sum += d > 0.0 ? d : 0.0;
          }
        }
      } else {
        for (; j + 32 * (kBatch - 1) < to; j += 32 * kBatch) {
          T x[kBatch];
#pragma unroll
          for (int k = 0; k < kBatch; ++k) x[k] = p_row[j + 32 * k];
#pragma unroll
          for (int k = 0; k < kBatch; ++k) {
            const double d = wide(x[k]);
            sum += d > 0.0 && j + 32 * k != without ? d : 0.0;
          }
        }
      }
      for (; j < to; j += 32) sum += mass(j);
      for (int k = 16; k; k /= 2) sum += __shfl_xor_sync(~0u, sum, k);
      if (lane == 0) sums[warp] = sum;
    }
    cluster.sync();
    if (warp == 0) {
      // a lane has two segments next to one another
      double mine[2], upto;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int s = 2 * lane + k;
        mine[k] = s < segments ? cluster.map_shared_rank(sums, s / kWarps)[s % kWarps] : 0.0;
      }
      upto = mine[0] + mine[1];
      for (int k = 1; k < 32; k *= 2) {
        const double x = __shfl_up_sync(~0u, upto, k);
        if (lane >= k) upto += x;
      }
      const double total = __shfl_sync(~0u, upto, 31), goal = double(reinterpret_cast<const float *>(a.finals)[seq]) * total;
      double before = __shfl_up_sync(~0u, upto, 1);
      if (lane == 0) before = 0.0;
      // the first segment whose end is past the goal; else the last that has anything
      const bool first_past = mine[0] > 0.0 && before + mine[0] > goal, past = first_past || (mine[1] > 0.0 && upto > goal);
      const unsigned all_past = __ballot_sync(~0u, past), any = __ballot_sync(~0u, mine[0] > 0.0 || mine[1] > 0.0);
      const int owner = all_past ? __ffs(all_past) - 1 : 31 - __clz(any);      // (-1: none)
      if (lane == max(owner, 0)) {
        const bool second = all_past ? !first_past : mine[1] > 0.0;
        segment_shared = total > 0.0 && owner >= 0 ? 2 * lane + second : -1;
        target_shared = goal;
        before_shared = second ? before + mine[0] : before;
      }
    }
    __syncthreads();
    cluster.barrier_arrive();          // the sums have been read
    const int at = segment_shared;
    if (at < 0 && pass == 0 && (q_row || without >= 0)) {      // nothing is left of p: p itself
      q_row = nullptr;
      without = -1;
      cluster.barrier_wait();
      continue;
    }
    if (at < 0) {
      if (rank == 0 && tid == 0) tokens[kept] = -1;
    } else if (at / kWarps == rank) {
      // the segment once more, some elements next to one another a thread at a time, and
      // the threads' sums in their order
      const int to = segment_begin(at + 1);
      const double goal = target_shared;
      double before = before_shared;
      int last = -1;
      for (int from = segment_begin(at);; from += kThreads * kEach) {
        double d[kEach], sum = 0.0;
        int positive = -1, token = INT_MAX;
        const int mine = from + tid * kEach;
#pragma unroll
        for (int k = 0; k < kEach; ++k) d[k] = mine + k < to ? mass(mine + k) : 0.0;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
          sum += d[k];
          if (d[k] > 0.0) positive = mine + k;
        }
        double upto = sum;
        for (int k = 1; k < 32; k *= 2) {
          const double x = __shfl_up_sync(~0u, upto, k);
          if (lane >= k) upto += x;
        }
        if (lane == 31) warp_sums[warp] = upto;
        positive = __reduce_max_sync(~0u, positive);
        if (lane == 0) positive_shared[warp] = positive;
        __syncthreads();
        double reached = before + (upto - sum);
        for (int w = 0; w < kWarps; ++w) {
          if (w < warp) reached += warp_sums[w];
          before += warp_sums[w];
          last = max(last, positive_shared[w]);
        }
        // the first element past the goal
#pragma unroll
        for (int k = kEach - 1; k >= 0; --k) {
          double s = reached;
#pragma unroll
          for (int e = 0; e <= k; ++e) s += d[e];
          if (d[k] > 0.0 && s > goal) token = mine + k;
        }
        token = __reduce_min_sync(~0u, token);
        if (lane == 0) token_shared[warp] = token;
        __syncthreads();
        for (int w = 0; w < kWarps; ++w) token = min(token, token_shared[w]);
        const bool end = from >= to - kThreads * kEach;
        if (token != INT_MAX || end) {
          // (none: the goal is the end, or within a rounding of it)
          if (tid == 0) tokens[kept] = token != INT_MAX ? token : last;
          break;
        }
      }
    }
    break;
  }
  cluster.barrier_wait();              // a CTA's shared memory lasts while others read it
}

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

template <typename T> int launch(const emmy_verify_args &a, cudaStream_t s) {
  // CTAs of a cluster: as many as have 4,096 elements each, fewer where the sequences
  // fill the GPU's 4 CTAs an SM without
  int ctas = 1, sms = 0;
  if (const int e = emmy_internal_sms(&sms)) return cuda_fail("emmy_verify: device", static_cast<cudaError_t>(e));
  while (ctas < kMostCtas && a.vocabulary > 4096 * ctas && int64_t(a.sequences) * 2 * ctas <= 4 * sms) ctas *= 2;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(a.sequences) * ctas);
  config.blockDim = dim3(kThreads);
  config.stream = s;
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = ctas;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  config.attrs = &cluster;
  config.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&config, verify_kernel<T>, a);
  return e == cudaSuccess ? 0 : cuda_fail("emmy_verify: launch", e);
}

}  // namespace

extern "C" EMMY_API int emmy_verify(const emmy_verify_args *a, void *stream) {
  if (!a) return fail("emmy_verify: bad argument");
  if (a->dtype != 6 && a->dtype != 7 && a->dtype != 9) return fail("emmy_verify: dtype %ld (f16, f32 or bf16)", a->dtype);
  if (a->sequences < 0 || a->sequences > (1 << 24) || a->rows < 0 || a->drafts < 0 || a->rows > (1 << 30) || a->drafts > a->rows)
    return fail("emmy_verify: bad count of sequences, rows or drafts");
  if (a->vocabulary < 1 || a->vocabulary > (1 << 28)) return fail("emmy_verify: a vocabulary of %ld (1 to 2^28)", a->vocabulary);
  if (a->sequences == 0) return 0;
  if (!a->target || !a->first || !a->finals || !a->accepted || !a->tokens || (a->drafts && (!a->drafted || !a->uniforms)))
    return fail("emmy_verify: null address");
  const int size = a->dtype == 7 ? 4 : 2;
  if ((a->target | a->proposal) % size || (a->first | a->finals | a->accepted | a->tokens | a->drafted | a->uniforms) % 4)
    return fail("emmy_verify: address not a multiple of its element's size");
  if ((a->rows > 1 && a->target_stride < 0) || (a->drafts > 1 && a->proposal && a->proposal_stride < 0))
    return fail("emmy_verify: a stride is negative");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->dtype == 6) return launch<__half>(*a, s);
  if (a->dtype == 7) return launch<float>(*a, s);
  return launch<__nv_bfloat16>(*a, s);
}
