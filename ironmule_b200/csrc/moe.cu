// Entry points of the products by expert: one grouped 4-bit product, and the gated MLP of two of them.
#include "common.cuh"
#include "moe.cuh"
#include "../../include/imspec.h"

namespace im {

// The checks that both entry points share; IM_OK when the sizes and the plan are usable.
static int moe_check(const char* who, int64_t M, int64_t E, int64_t top_k, const int32_t* pairs, const void* plan,
                     size_t plan_bytes) {
  IM_REQUIRE(M >= 0 && E >= 1 && top_k >= 1 && top_k <= E, IM_INVALID, "%s: bad sizes M=%lld E=%lld top_k=%lld", who,
             (long long)M, (long long)E, (long long)top_k);
  IM_REQUIRE(M <= MOE_MAX_ROWS && E <= MOE_MAX_EXPERTS && top_k <= MOE_MAX_TOP_K, IM_UNSUPPORTED,
             "%s: at most %lld rows, %d experts and %d places a row", who, (long long)MOE_MAX_ROWS, MOE_MAX_EXPERTS,
             MOE_MAX_TOP_K);
  if (M == 0) return IM_OK;
  IM_REQUIRE(pairs && plan && aligned(plan, 16), IM_INVALID, "%s: null or misaligned plan", who);
  const size_t need = moe_plan(M, E, top_k).bytes;
  IM_REQUIRE(plan_bytes >= need, IM_INVALID, "%s: plan of %zu bytes needed, %zu given", who, need, plan_bytes);
  return IM_OK;
}

static bool moe_nk_ok(int64_t N, int64_t K) {
  return N >= 1 && N <= (1 << 24) && K >= 64 && K % 64 == 0 && K <= (1 << 20);
}

static int moe_product(const MoePlan& p, const MoeProduct& a, cudaStream_t st) { return moe_mma_launch(p, a, st); }

}  // namespace im

using namespace im;

extern "C" size_t im_moe_packed_bytes(int64_t E, int64_t N, int64_t K) {
  if (E < 1 || E > MOE_MAX_EXPERTS || !moe_nk_ok(N, K)) return 0;
  return (size_t)E * im_qgemm_packed_bytes(N, K);
}

extern "C" int im_moe_pack_w4g64(const uint32_t* w, const uint16_t* scales, const uint16_t* biases, int64_t E,
                                 int64_t N, int64_t K, void* packed, void* stream) {
  clear_error();
  IM_REQUIRE(E >= 1 && E <= MOE_MAX_EXPERTS && moe_nk_ok(N, K), IM_INVALID,
             "im_moe_pack_w4g64: bad sizes E=%lld N=%lld K=%lld", (long long)E, (long long)N, (long long)K);
  IM_REQUIRE(w && scales && biases && packed, IM_INVALID, "im_moe_pack_w4g64: null pointer");
  const size_t bytes = im_qgemm_packed_bytes(N, K);
  for (int64_t e = 0; e < E; e++) {  // once per model load; rows of an expert are padded to whole tiles
    const int rc = im_qgemm_pack_w4g64(w + e * N * (K / 8), scales + e * N * (K / 64), biases + e * N * (K / 64), N, K,
                                       reinterpret_cast<char*>(packed) + e * bytes, stream);
    if (rc) return rc;
  }
  return IM_OK;
}

extern "C" int im_moe_grouped_qgemm(const void* packed, const uint16_t* x, uint16_t* y, int64_t M, int64_t E,
                                    int64_t top_k, int64_t N, int64_t K, int x_by_pair, const int32_t* pairs,
                                    const void* plan, size_t plan_bytes, void* stream) {
  clear_error();
  const int rc = moe_check("im_moe_grouped_qgemm", M, E, top_k, pairs, plan, plan_bytes);
  if (rc) return rc;
  IM_REQUIRE(moe_nk_ok(N, K), IM_INVALID, "im_moe_grouped_qgemm: bad sizes N=%lld K=%lld", (long long)N,
             (long long)K);
  if (M == 0) return IM_OK;
  IM_REQUIRE(packed && x && y, IM_INVALID, "im_moe_grouped_qgemm: null pointer");
  IM_REQUIRE(aligned(packed, 16) && aligned(x, 16) && aligned(y, 2), IM_INVALID,
             "im_moe_grouped_qgemm: packed and x must be 16-byte aligned");
  MoeProduct a = {};
  a.wp = reinterpret_cast<const unsigned char*>(packed);
  a.x = x;
  a.y = y;
  a.plan = reinterpret_cast<const int*>(plan);
  a.pairs = pairs;
  a.M = (int)M;
  a.E = (int)E;
  a.top_k = (int)top_k;
  a.N = (int)N;
  a.K = (int)K;
  a.src = x_by_pair ? MOE_BY_PAIR : MOE_BY_TOKEN;
  a.dst = MOE_BY_PAIR;
  a.epilogue = IM_EPI_STORE;
  return moe_product(moe_plan(M, E, top_k), a, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" size_t im_moe_mlp_workspace_bytes(int64_t M, int64_t E, int64_t top_k, int64_t H, int64_t I) {
  if (M < 0 || M > MOE_MAX_ROWS || E < 1 || E > MOE_MAX_EXPERTS || top_k < 1 || top_k > MOE_MAX_TOP_K || top_k > E ||
      H < 64 || H % 64 || I < 64 || I % 64)
    return 0;
  return (size_t)M * top_k * I * 2;
}

extern "C" int im_moe_mlp(const void* gate_up, const void* down, const uint16_t* x, uint16_t* y, int64_t M, int64_t E,
                          int64_t top_k, int64_t H, int64_t I, int activation, const int32_t* pairs, const void* plan,
                          size_t plan_bytes, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  const int rc = moe_check("im_moe_mlp", M, E, top_k, pairs, plan, plan_bytes);
  if (rc) return rc;
  IM_REQUIRE(moe_nk_ok(H, H) && moe_nk_ok(2 * I, I), IM_INVALID,
             "im_moe_mlp: hidden and intermediate sizes are multiples of 64 (H=%lld I=%lld)", (long long)H,
             (long long)I);
  IM_REQUIRE(activation == IM_EPI_SWIGLU || activation == IM_EPI_GEGLU, IM_INVALID, "im_moe_mlp: bad activation");
  if (M == 0) return IM_OK;
  IM_REQUIRE(gate_up && down && x && y, IM_INVALID, "im_moe_mlp: null pointer");
  IM_REQUIRE(aligned(gate_up, 16) && aligned(down, 16) && aligned(x, 16) && aligned(y, 2), IM_INVALID,
             "im_moe_mlp: weights and x must be 16-byte aligned");
  const size_t need = im_moe_mlp_workspace_bytes(M, E, top_k, H, I);
  IM_REQUIRE(workspace && aligned(workspace, 256) && workspace_bytes >= need, IM_INVALID,
             "im_moe_mlp: workspace of %zu bytes (256-aligned) needed, %zu given", need, workspace_bytes);
  const MoePlan p = moe_plan(M, E, top_k);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  // the gated activations lie in the order of the sorted pairs, so that an item's rows are contiguous
  MoeProduct a = {};
  a.wp = reinterpret_cast<const unsigned char*>(gate_up);
  a.x = x;
  a.y = reinterpret_cast<uint16_t*>(workspace);
  a.plan = reinterpret_cast<const int*>(plan);
  a.pairs = pairs;
  a.M = (int)M;
  a.E = (int)E;
  a.top_k = (int)top_k;
  a.N = (int)(2 * I);
  a.K = (int)H;
  a.src = MOE_BY_TOKEN;
  a.dst = MOE_SORTED;
  a.epilogue = activation;
  const int first = moe_product(p, a, st);
  if (first) return first;
  a.wp = reinterpret_cast<const unsigned char*>(down);
  a.x = reinterpret_cast<const uint16_t*>(workspace);
  a.y = y;
  a.N = (int)H;
  a.K = (int)I;
  a.src = MOE_SORTED;
  a.dst = MOE_BY_PAIR;
  a.epilogue = IM_EPI_STORE;
  // the first product waited for the routing before its CTAs let this launch begin
  a.early = 1;
  return moe_product(p, a, st);
}
