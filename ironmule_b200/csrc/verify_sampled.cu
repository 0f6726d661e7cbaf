// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Draft i of a sequence is kept iff every earlier one was and u_i q_i(d_i) < p_i(d_i); without a draft distribution (n-gram
// drafts) iff u_i < p_i(d_i). At the first refusal the next token is drawn from max(p - q, 0) (without a distribution:
// from p without d_i), after all drafts from p: the smallest token whose cumulative weight exceeds u times the total.
// Everything after the loads is float64: products of two float32 are exact in it, so are differences but for the last
// bit, and sums over a vocabulary are off by 1e-13 of themselves, where float32 sums would draw another token in a
// percent of the draws.
//
// Bound: HBM, one row of p and one of q a sequence; for few sequences, the chain of dependent steps (the drafts, their
// probabilities, a row's sum, the token). A sequence is a cluster of up to 16 blocks, each with a run of the vocabulary.
// Every block decides on the drafts for itself (a few gathers), sums its run and tells the others its total through
// distributed shared memory; the warp that holds the target then looks for the token in its own part.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace im {

namespace cg = cooperative_groups;

constexpr int VS_THREADS = 512;
constexpr int VS_WARPS = VS_THREADS / 32;
constexpr int VS_CLUSTER = 16;

struct VerifyArgs {
  const void* p;
  const void* q;
  long long p_ld, q_ld;
  const int* drafts;
  long long drafts_ld;
  const int* n_drafts;
  const float* u;
  long long u_ld;
  long long K, V;
  int* out_tokens;
  int* out_count;
};

__device__ __forceinline__ double vs_value(float v) { return v; }
__device__ __forceinline__ double vs_value(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ double vs_value(__half v) { return __half2float(v); }

// A probability, or 0 where it is none.
template <typename T>
__device__ __forceinline__ double vs_prob(T v) {
  const double d = vs_value(v);
  return d > 0.0 && d < __longlong_as_double(0x7ff0000000000000ll) ? d : 0.0;
}

__device__ __forceinline__ double vs_warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Cluster = sequence: rank r takes tokens [r span, (r + 1) span), a warp a part of them, read 32 at a time.
template <typename T>
__global__ void __launch_bounds__(VS_THREADS, 2) verify_sampled_kernel(VerifyArgs a) {
  __shared__ int first;
  __shared__ double sums[VS_WARPS];
  __shared__ double totals[2][VS_CLUSTER];  // of the cluster's blocks, by attempt; written by them
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = cluster.num_blocks(), rank = cluster.block_rank();
  pdl_wait();
  pdl_trigger();
  const long long b = blockIdx.x / ranks;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const T* p0 = (const T*)a.p + b * (a.K + 1) * a.p_ld;
  const T* q0 = (const T*)a.q + b * a.K * a.q_ld;
  const int* drafts = a.drafts + b * a.drafts_ld;
  const float* u = a.u + b * a.u_ld;
  int n = (int)a.K;
  if (a.n_drafts) n = min(max(a.n_drafts[b], 0), (int)a.K);
  const double u_last = u[a.K];
  if (t == 0) first = n;
  __syncthreads();
  for (int i = t; i < n; i += VS_THREADS) {
    const long long d = drafts[i];
    const bool inside = d >= 0 && d < a.V;
    const double p = inside ? vs_prob(p0[i * a.p_ld + d]) : 0.0;
    const double q = !a.q ? 1.0 : inside ? vs_prob(q0[i * a.q_ld + d]) : 0.0;
    if (!((double)u[i] * q < p)) atomicMin(&first, i);
  }
  __syncthreads();
  const int kept = first;
  const T* p = p0 + kept * a.p_ld;
  const T* q = a.q && kept < n ? q0 + kept * a.q_ld : nullptr;
  const int without = !a.q && kept < n ? drafts[kept] : -1;
  const int part = (int)((a.V + ranks * VS_WARPS * 32 - 1) / (ranks * VS_WARPS * 32)) * 32;  // tokens of a warp
  const int V = (int)a.V;
  const long long begin = (long long)(rank * VS_WARPS + warp) * part;
  const int lo = (int)min(begin, a.V), hi = min(lo + part, V);
  bool whole = kept == n;
  auto weight = [&](int v, bool all) {
    double w = vs_prob(p[v]);
    if (!all) {
      if (q) w = fmax(w - vs_prob(q[v]), 0.0);
      if (v == without) w = 0.0;
    }
    return w;
  };
  double target = 0.0, before = 0.0;
  int owner = -1;  // the block whose run the target falls into: the first that passes it, or the last with any weight
  for (int attempt = 0; attempt < 2; attempt++) {
    double sum = 0.0;
#pragma unroll 8
    for (int v = lo + lane; v < hi; v += 32) sum += weight(v, whole);
    sum = vs_warp_sum(sum);
    if (lane == 0) sums[warp] = sum;
    __syncthreads();
    if (warp == 0) {
      double s = lane < VS_WARPS ? sums[lane] : 0.0;
      s = vs_warp_sum(s);
      if (lane < ranks) *cluster.map_shared_rank(&totals[attempt][rank], lane) = s;
    }
    cluster.sync();
    double total = 0.0;
    for (int r = 0; r < ranks; r++) total += totals[attempt][r];
    if (!(total > 0.0) && !whole) {  // nothing is left beside q: the token comes from p
      whole = true;
      continue;
    }
    target = u_last * total;
    double at = 0.0;
    for (int r = 0; r < ranks; r++) {
      const double s = totals[attempt][r];
      if (s > 0.0) {
        owner = r, before = at;
        if (at + s > target) break;
      }
      at += s;
    }
    break;
  }
  if (rank != max(owner, 0)) return;
  // within the block, then the warp, the same
  int mine = -1;
  double at = before;
  for (int w = 0; w < VS_WARPS; w++) {
    const double s = sums[w];
    if (s > 0.0) {
      mine = w, before = at;
      if (at + s > target) break;
    }
    at += s;
  }
  if (warp != max(mine, 0)) return;
  int token = 0;  // of a row without any weight
  if (mine >= 0) {
    // each lane takes a run of the part in order; the lane that the target falls into walks its run
    const int each = part / 32, v0 = min(lo + lane * each, hi), v1 = min(v0 + each, hi);
    double sum = 0.0;
#pragma unroll 4
    for (int v = v0; v < v1; v++) sum += weight(v, whole);
    double incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    const unsigned any = __ballot_sync(0xffffffffu, sum > 0.0);
    const unsigned pass = __ballot_sync(0xffffffffu, sum > 0.0 && before + incl > target);
    const int holder = pass ? __ffs(pass) - 1 : 31 - __clz(any);
    if (lane == holder) {
      double run = before + incl - sum;
      for (int v = v0; v < v1; v++) {
        const double w = weight(v, whole);
        run += w;
        if (w > 0.0) {
          token = v;
          if (run > target) break;
        }
      }
    }
    token = __shfl_sync(0xffffffffu, token, holder);
  }
  int* out = a.out_tokens + b * (a.K + 1);
  for (int i = lane; i <= a.K; i += 32) out[i] = i < kept ? drafts[i] : i == kept ? token : -1;
  if (lane == 0) a.out_count[b] = kept + 1;
}

template <typename T>
int launch_verify_sampled(const VerifyArgs& a, int64_t B, cudaStream_t st) {
  // blocks a sequence: enough to fill the device's two blocks an SM, of at least 2048 tokens
  int ranks = 1;
  while (ranks < VS_CLUSTER && B * ranks * 2 <= 296 && a.V >= ranks * 2 * 2048) ranks *= 2;
  if (ranks > 8) {
    const cudaError_t e =
        cudaFuncSetAttribute(verify_sampled_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) {
      set_error("verify_sampled_kernel: %s", cudaGetErrorString(e));
      return IM_CUDA_ERROR;
    }
  }
  return launch_cluster("verify_sampled_kernel", verify_sampled_kernel<T>, dim3((unsigned)(B * ranks)),
                        dim3(VS_THREADS), ranks, 0, st, a);
}

}  // namespace im

using namespace im;

extern "C" int im_verify_sampled(const void* target, int64_t target_ld, const void* draft, int64_t draft_ld, int dtype,
                                 const int32_t* drafts, int64_t drafts_ld, const int32_t* n_drafts,
                                 const float* uniforms, int64_t uniforms_ld, int64_t B, int64_t K, int64_t V,
                                 int32_t* out_tokens, int32_t* out_count, void* stream) {
  clear_error();
  IM_REQUIRE(B >= 0 && K >= 0 && V >= 1 && target_ld >= V && (!draft || draft_ld >= V) && drafts_ld >= 0 &&
                 uniforms_ld >= 0,
             IM_INVALID, "im_verify_sampled: bad sizes");
  IM_REQUIRE(dtype >= IM_BF16 && dtype <= IM_F32, IM_INVALID, "im_verify_sampled: type %d", dtype);
  if (B == 0) return IM_OK;
  IM_REQUIRE(target && uniforms && out_tokens && out_count && (drafts || K == 0), IM_INVALID,
             "im_verify_sampled: null pointer");
  IM_REQUIRE(B < (1 << 16) && K <= 4096 && V < (1ll << 31) - 65536, IM_UNSUPPORTED,
             "im_verify_sampled: %lld sequences, %lld drafts, %lld tokens (up to 65535, 4096, 2^31 - 65537)", (long long)B,
             (long long)K, (long long)V);
  const int size = dtype == IM_F32 ? 4 : 2;
  IM_REQUIRE(aligned(target, size) && aligned(draft, size) && aligned(drafts, 4) && aligned(n_drafts, 4) &&
                 aligned(uniforms, 4) && aligned(out_tokens, 4) && aligned(out_count, 4),
             IM_INVALID, "im_verify_sampled: misaligned pointer");
  VerifyArgs a = {target, K ? draft : nullptr, target_ld, draft_ld, drafts, drafts_ld, n_drafts, uniforms,
                  uniforms_ld, K, V, out_tokens, out_count};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == IM_BF16) return launch_verify_sampled<__nv_bfloat16>(a, B, st);
  if (dtype == IM_F16) return launch_verify_sampled<__half>(a, B, st);
  return launch_verify_sampled<float>(a, B, st);
}
