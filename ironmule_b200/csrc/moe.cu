// Entry points of the products by expert: one grouped 4-bit product, and the gated MLP of two of them.
#include <math.h>

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

// One thread per row of a block's group: its codes into the packed order, the largest |w| of the row (all values
// non-negative, so their bit patterns order as integers; a maximum does not depend on the order).
__global__ void __launch_bounds__(128)
moe_pack_kernel(const uint32_t* __restrict__ w, const uint16_t* __restrict__ sc, const uint16_t* __restrict__ bi, int N,
                int K, int blocks, unsigned char* __restrict__ out, unsigned* __restrict__ row_max) {
  const int G = K >> 6;
  const long long unit = blockIdx.x;  // (expert * blocks + block) * G + group
  const int grp = (int)(unit % G), block = (int)(unit / G % blocks);
  const long long expert = unit / G / blocks;
  const int r = block * 128 + threadIdx.x, tile = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t words[8] = {};
  uint16_t s = 0, b = 0;
  float top = 0.f;
  if (r < N) {
    const size_t row = (size_t)expert * N + r;
#pragma unroll
    for (int i = 0; i < 8; i++) words[i] = w[row * (K >> 3) + grp * 8 + i];
    s = sc[row * G + grp];
    b = bi[row * G + grp];
    top = fmaxf(fabsf(bf(b)), fabsf(fmaf(15.f, bf(s), bf(b))));
    if (!(top < INFINITY)) top = 0.f;  // (a broken group does not hide the scale of the others)
  }
  unsigned char* dst = out + unit * MOE_BLOCK_BYTES;
  uint4* d = reinterpret_cast<uint4*>(dst + tile * 1024 + lane * 16);
  d[0] = make_uint4(words[0], words[1], words[2], words[3]);
  d[32] = make_uint4(words[4], words[5], words[6], words[7]);
  uint16_t* sb = reinterpret_cast<uint16_t*>(dst + 4096 + tile * 128 + (lane & 7) * 16);
  sb[lane >> 3] = s;
  sb[4 + (lane >> 3)] = b;
  if (top > 0.f) atomicMax(row_max + (expert * blocks + block) * 128 + threadIdx.x, __float_as_uint(top));
}

// A warp per row: the row's 2-norm into the largest of its expert's half (over its finite groups, relative to its largest;
// a thousandth and 2^-16 of the largest per weight cover what rounding the weights to operands can add).
__global__ void __launch_bounds__(256)
moe_norm_kernel(const uint32_t* __restrict__ w, const uint16_t* __restrict__ sc, const uint16_t* __restrict__ bi,
                long long rows, int N, int K, int blocks, const float* __restrict__ row_max,
                unsigned* __restrict__ norm_max) {
  const int G = K >> 6, lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const long long expert = row / N;
  const int r = (int)(row % N);
  const float top = row_max[(expert * blocks + r / 128) * 128 + r % 128];
  if (!(top > 0.f)) return;
  const int e = min(max(ilogbf(top), -120), 120);
  const float inv = ldexpf(1.f, -e);
  float ss = 0.f;
  for (int g = lane; g < G; g += 32) {
    const float s = bf(sc[row * G + g]) * inv, b = bf(bi[row * G + g]) * inv;
    if (!(fmaxf(fabsf(b), fabsf(fmaf(15.f, s, b))) < INFINITY)) continue;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const uint32_t u = w[row * (K >> 3) + g * 8 + i];
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float v = fmaf((float)(u >> (4 * j) & 15u), s, b);
        ss = fmaf(v, v, ss);
      }
    }
  }
  ss = warp_sum(ss);
  const float norm = ldexpf(1.001f * sqrtf(ss) + 0x1p-16f * sqrtf((float)K), e);
  if (lane == 0) atomicMax(norm_max + 2 * expert + (r >> 4 & 1), __float_as_uint(norm));
}

static size_t moe_expert_bytes(int64_t N, int64_t K) { return (size_t)((N + 127) / 128) * (K / 64) * MOE_BLOCK_BYTES; }
static size_t moe_max_bytes(int64_t N) { return (size_t)((N + 127) / 128) * 512 + 8; }  // of an expert

}  // namespace im

using namespace im;

extern "C" size_t im_moe_packed_bytes(int64_t E, int64_t N, int64_t K) {
  if (E < 1 || E > MOE_MAX_EXPERTS || !moe_nk_ok(N, K)) return 0;
  return (size_t)E * (moe_expert_bytes(N, K) + moe_max_bytes(N));
}

extern "C" int im_moe_pack_w4g64(const uint32_t* w, const uint16_t* scales, const uint16_t* biases, int64_t E,
                                 int64_t N, int64_t K, void* packed, void* stream) {
  clear_error();
  IM_REQUIRE(E >= 1 && E <= MOE_MAX_EXPERTS && moe_nk_ok(N, K), IM_INVALID,
             "im_moe_pack_w4g64: bad sizes E=%lld N=%lld K=%lld", (long long)E, (long long)N, (long long)K);
  IM_REQUIRE(w && scales && biases && packed, IM_INVALID, "im_moe_pack_w4g64: null pointer");
  IM_REQUIRE(aligned(packed, 16) && aligned(w, 4) && aligned(scales, 2) && aligned(biases, 2), IM_INVALID,
             "im_moe_pack_w4g64: misaligned buffer");
  const int64_t blocks = (N + 127) / 128, units = E * blocks * (K / 64);
  IM_REQUIRE(units < (1ll << 31), IM_UNSUPPORTED, "im_moe_pack_w4g64: too many units");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  unsigned char* out = reinterpret_cast<unsigned char*>(packed);
  unsigned* row_max = reinterpret_cast<unsigned*>(out + (size_t)E * moe_expert_bytes(N, K));
  const cudaError_t e = cudaMemsetAsync(row_max, 0, (size_t)E * moe_max_bytes(N), st);
  if (e != cudaSuccess) {
    set_error("im_moe_pack_w4g64: %s", cudaGetErrorString(e));
    return IM_CUDA_ERROR;
  }
  moe_pack_kernel<<<(unsigned)units, 128, 0, st>>>(w, scales, biases, (int)N, (int)K, (int)blocks, out, row_max);
  const int rc = check_launch("moe_pack_kernel");
  if (rc) return rc;
  moe_norm_kernel<<<(unsigned)((E * N + 7) / 8), 256, 0, st>>>(w, scales, biases, E * N, (int)N, (int)K, (int)blocks,
                                                              reinterpret_cast<const float*>(row_max),
                                                              row_max + (size_t)E * blocks * 128);
  return check_launch("moe_norm_kernel");
}

extern "C" int im_moe_status(const void* plan) {
  clear_error();
  IM_REQUIRE(plan, IM_INVALID, "im_moe_status: null plan");
  int word = 0;
  // the products may run on a stream that the copy's own (the default) stream does not wait for
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpy(&word, reinterpret_cast<const int*>(plan) + 1, 4, cudaMemcpyDeviceToHost);
  if (e != cudaSuccess) {
    set_error("im_moe_status: %s", cudaGetErrorString(e));
    return IM_CUDA_ERROR;
  }
  return word;
}

extern "C" size_t im_moe_grouped_workspace_bytes(int64_t M, int64_t E, int64_t top_k, int64_t K) {
  if (M < 1 || M > MOE_MAX_ROWS || E < 1 || E > MOE_MAX_EXPERTS || top_k < 1 || top_k > MOE_MAX_TOP_K || top_k > E ||
      !moe_nk_ok(1, K))
    return 0;
  return moe_space(moe_plan(M, E, top_k), M * top_k, K, 0).total;
}

extern "C" int im_moe_grouped_qgemm(const void* packed, const uint16_t* x, uint16_t* y, int64_t M, int64_t E,
                                    int64_t top_k, int64_t N, int64_t K, int x_by_pair, const int32_t* pairs,
                                    void* plan, size_t plan_bytes, void* workspace, size_t workspace_bytes,
                                    void* stream) {
  clear_error();
  const int rc = moe_check("im_moe_grouped_qgemm", M, E, top_k, pairs, plan, plan_bytes);
  if (rc) return rc;
  IM_REQUIRE(moe_nk_ok(N, K), IM_INVALID, "im_moe_grouped_qgemm: bad sizes N=%lld K=%lld", (long long)N,
             (long long)K);
  if (M == 0) return IM_OK;
  IM_REQUIRE(packed && x && y, IM_INVALID, "im_moe_grouped_qgemm: null pointer");
  IM_REQUIRE(aligned(packed, 16) && aligned(x, 16) && aligned(y, 2), IM_INVALID,
             "im_moe_grouped_qgemm: packed and x must be 16-byte aligned");
  const size_t need = im_moe_grouped_workspace_bytes(M, E, top_k, K);
  IM_REQUIRE(workspace && aligned(workspace, 256) && workspace_bytes >= need, IM_INVALID,
             "im_moe_grouped_qgemm: workspace of %zu bytes (256-aligned) needed, %zu given", need, workspace_bytes);
  MoeProduct a = {};
  a.wp = reinterpret_cast<const unsigned char*>(packed);
  a.y = y;
  a.plan = reinterpret_cast<const int*>(plan);
  a.pairs = pairs;
  a.M = (int)M;
  a.E = (int)E;
  a.top_k = (int)top_k;
  a.N = (int)N;
  a.K = (int)K;
  a.epilogue = IM_EPI_STORE;
  const MoePlan p = moe_plan(M, E, top_k);
  const MoeSpace space = moe_space(p, M * top_k, K, 0);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int prep = moe_prep_launch(p, a, x, x_by_pair != 0, space, workspace, st);
  return prep ? prep : moe_product_launch(p, a, space, workspace, st);
}

extern "C" size_t im_moe_mlp_workspace_bytes(int64_t M, int64_t E, int64_t top_k, int64_t H, int64_t I) {
  if (M < 1 || M > MOE_MAX_ROWS || E < 1 || E > MOE_MAX_EXPERTS || top_k < 1 || top_k > MOE_MAX_TOP_K || top_k > E ||
      !moe_nk_ok(H, H) || !moe_nk_ok(2 * I, I))
    return 0;
  return moe_space(moe_plan(M, E, top_k), M * top_k, H, I).total;
}

extern "C" int im_moe_mlp(const void* gate_up, const void* down, const uint16_t* x, uint16_t* y, int64_t M, int64_t E,
                          int64_t top_k, int64_t H, int64_t I, int activation, const int32_t* pairs, void* plan,
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
  const MoeSpace space = moe_space(p, M * top_k, H, I);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  MoeProduct a = {};
  a.wp = reinterpret_cast<const unsigned char*>(gate_up);
  a.plan = reinterpret_cast<const int*>(plan);
  a.pairs = pairs;
  a.M = (int)M;
  a.E = (int)E;
  a.top_k = (int)top_k;
  a.N = (int)(2 * I);
  a.K = (int)H;
  a.epilogue = activation;
  int status = moe_prep_launch(p, a, x, 0, space, workspace, st);
  if (!status) status = moe_product_launch(p, a, space, workspace, st);
  if (status) return status;
  a.wp = reinterpret_cast<const unsigned char*>(down);
  a.y = y;
  a.N = (int)H;
  a.K = (int)I;
  a.epilogue = IM_EPI_STORE;
  a.second = true;
  return moe_product_launch(p, a, space, workspace, st);
}
