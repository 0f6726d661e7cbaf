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
// distributed shared memory; the warp that holds the target then looks for the token in its own part. Four drafts of 151936
// float32 values take 10 us, 32 sequences of them 18.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <utility>

#include "common.cuh"

namespace im {

namespace cg = cooperative_groups;

constexpr int VS_THREADS = 512;
constexpr int VS_WARPS = VS_THREADS / 32;
constexpr int VS_CLUSTER = 16;
constexpr int VS_LEFT = 2048;  // weights looked through at a time for the token

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

__device__ __forceinline__ float vs_value(float v) { return v; }
__device__ __forceinline__ float vs_value(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float vs_value(__half v) { return __half2float(v); }

// A probability, or 0 where it is none.
__device__ __forceinline__ float vs_clean(float v) { return v > 0.f && v < INFINITY ? v : 0.f; }
template <typename T>
__device__ __forceinline__ float vs_prob(T v) {
  return vs_clean(vs_value(v));
}

// What is left of p beside q: exact in float64 but for the last bit.
__device__ __forceinline__ double vs_left(float p, float q) { return p > q ? (double)p - (double)q : 0.0; }

__device__ __forceinline__ double vs_warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Cluster = sequence: rank r takes tokens [r span, (r + 1) span), a warp a part of them, read 32 at a time.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) VsVec {
  T v[VEC];
};

template <typename T, bool WIDE>
__global__ void __launch_bounds__(VS_THREADS, 2) verify_sampled_kernel(VerifyArgs a) {
  __shared__ int first;
  __shared__ double sums[VS_WARPS];
  __shared__ double totals[2][VS_CLUSTER];  // of the cluster's blocks, by attempt; written by them
  extern __shared__ double left[];          // the weights of the part that holds the token
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = cluster.num_blocks(), rank = cluster.block_rank();
  // a block may be written to once it is known to run: all arrive here, and wait for the others before the first remote
  // store, with the gathers and sums between
  auto started = cluster.barrier_arrive();
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
    const float p = inside ? vs_prob(p0[i * a.p_ld + d]) : 0.f;
    const float q = !a.q ? 1.f : inside ? vs_prob(q0[i * a.q_ld + d]) : 0.f;
    if (!((double)u[i] * (double)q < (double)p)) atomicMin(&first, i);
  }
  __syncthreads();
  const int kept = first;
  const T* p = p0 + kept * a.p_ld;
  const T* q = a.q && kept < n ? q0 + kept * a.q_ld : nullptr;
  const int without = !a.q && kept < n ? drafts[kept] : -1;
  constexpr int VEC = WIDE ? 16 / (int)sizeof(T) : 1, STEP = 32 * VEC;
  const int part = (int)((a.V + ranks * VS_WARPS * STEP - 1) / (ranks * VS_WARPS * STEP)) * STEP;  // tokens of a warp
  const long long begin = (long long)(rank * VS_WARPS + warp) * part;
  const int lo = (int)min(begin, a.V), hi = (int)min((long long)lo + part, a.V);
  bool whole = kept == n;
  double target = 0.0, before = 0.0;
  int owner = -1;  // the block whose run the target falls into: the first that passes it, or the last with any weight
  for (int attempt = 0; attempt < 2; attempt++) {
    const bool beside = !whole && q != nullptr;
    double sum = 0.0;
    constexpr int BATCH = !WIDE ? 8 : sizeof(T) == 4 ? 4 : 2;  // loads in flight a lane, of p and of q each
    for (int v0 = lo; v0 < hi; v0 += STEP * BATCH) {
      VsVec<T, VEC> pv[BATCH], qv[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; i++) {
        const int v = v0 + i * STEP + lane * VEC;
        if (v < hi) {
          pv[i] = *(const VsVec<T, VEC>*)(p + v);
          if (beside) qv[i] = *(const VsVec<T, VEC>*)(q + v);
        }
      }
#pragma unroll
      for (int i = 0; i < BATCH; i++) {
        const int v = v0 + i * STEP + lane * VEC;
        if (v < hi) {
#pragma unroll
          for (int e = 0; e < VEC; e++) {
            float x = vs_prob(pv[i].v[e]);
            if (beside) sum += vs_left(x, vs_prob(qv[i].v[e]));
            else sum += !whole && v + e == without ? 0.0 : (double)x;
          }
        }
      }
    }
    sum = vs_warp_sum(sum);
    if (lane == 0) sums[warp] = sum;
    __syncthreads();
    if (attempt == 0) cluster.barrier_wait(std::move(started));
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
    // the part's weights once more, all of them in flight; then each lane sums a run of them, and the lane whose run holds
    // the target walks it
    const bool beside = !whole && q != nullptr;
    bool found = false;
    for (int v0 = lo; v0 < hi && !found; v0 += VS_LEFT) {
      const int size = min(VS_LEFT, hi - v0);
      __syncwarp();
#pragma unroll 8
      for (int i = lane; i < size; i += 32) {
        const int v = v0 + i;
        const float x = vs_prob(p[v]);
        left[i] = beside ? vs_left(x, vs_prob(q[v])) : !whole && v == without ? 0.0 : (double)x;
      }
      __syncwarp();
      const int each = ((size + 31) / 32) | 1;  // odd: lanes' runs start in different banks
      const int i0 = min(size, lane * each), i1 = min(size, i0 + each);
      double sum = 0.0;
      for (int i = i0; i < i1; i++) sum += left[i];
      double incl = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
      }
      const unsigned any = __ballot_sync(0xffffffffu, sum > 0.0);
      const unsigned pass = __ballot_sync(0xffffffffu, sum > 0.0 && before + incl > target);
      if (any) {  // the first run that passes the target, else the last with any weight
        const int holder = pass ? __ffs(pass) - 1 : 31 - __clz(any);
        if (lane == holder) {
          double run = before + incl - sum;
          for (int i = i0; i < i1; i++) {
            run += left[i];
            if (left[i] > 0.0) {
              token = v0 + i;
              if (run > target) break;
            }
          }
        }
        token = __shfl_sync(0xffffffffu, token, holder);
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
      found = pass != 0;
    }
  }
  int* out = a.out_tokens + b * (a.K + 1);
  for (int i = lane; i <= a.K; i += 32) out[i] = i < kept ? drafts[i] : i == kept ? token : -1;
  if (lane == 0) a.out_count[b] = kept + 1;
}

template <typename T, bool WIDE>
int launch_verify_ranks(const VerifyArgs& a, int64_t B, int ranks, cudaStream_t st) {
  const int rc = configure<verify_sampled_kernel<T, WIDE>>("verify_sampled_kernel", 0, true);
  if (rc != IM_OK) return rc;
  return launch_cluster("verify_sampled_kernel", verify_sampled_kernel<T, WIDE>, dim3((unsigned)(B * ranks)),
                        dim3(VS_THREADS), ranks, VS_LEFT * sizeof(double), st, a);
}

template <typename T>
int launch_verify_sampled(const VerifyArgs& a, int64_t B, cudaStream_t st) {
  // blocks a sequence: enough to fill the device's two blocks an SM, of at least 2048 tokens
  int ranks = 1;
  while (ranks < VS_CLUSTER && B * ranks * 2 <= 296 && a.V >= ranks * 2 * 2048) ranks *= 2;
  // 16-byte loads where every row starts on 16 bytes and is whole
  const int n = 16 / sizeof(T);
  const bool wide = aligned(a.p, 16) && aligned(a.q, 16) && a.p_ld % n == 0 && a.q_ld % n == 0 && a.V % n == 0;
  return wide ? launch_verify_ranks<T, true>(a, B, ranks, st) : launch_verify_ranks<T, false>(a, B, ranks, st);
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
