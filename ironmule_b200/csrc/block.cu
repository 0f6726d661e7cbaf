// The norms before and after a block, fused with its gate, the residual scale and the join of its places.
//
//   b  = sum_j w[m, j] y[m, j]                    (places in order; y[m] itself with one unweighted place)
//   b  = b / sqrt(mean(b^2) + eps) * w'           (post_norm given; w' = w, or 1 + w)
//   h' = residual_scale * h + gate * b
//   z  = h' / sqrt(mean(h'^2) + eps) * w'         (next_norm given)
//
// Everything is float32 in registers between one read of y and h and one write of h' and z; each output is rounded
// once, z from the float32 h'. out_sq is the sum of squares of the ROUNDED h' row (what a qGEMM with a fused RMSNorm
// prologue normalises). A place of weight 0 is left out, so what lies there (no expert chosen) does not matter.
// One CTA per row, 8 consecutive elements per thread and step; sums in a fixed order (thread, warp tree, warps in
// order), so a row's bits do not depend on the other rows. Bound by HBM for many rows, by two block reductions for few.
#include "common.cuh"
#include "../../include/imspec.h"

namespace im {

constexpr int BR_THREADS = 256;
constexpr int BR_MAX_PLACES = 32;
constexpr int BR_BATCH = 4;

struct BlockArgs {
  const uint16_t* y;
  const float* w;          // [M, places] or NULL
  const uint16_t* h;
  const uint16_t* post;
  const uint16_t* gate;
  const uint16_t* next;
  uint16_t* h_out;
  uint16_t* z;
  float* out_sq;
  long long gate_row, gate_col;
  float scale, eps;
  int places, H, gemma;
};

__device__ __forceinline__ float br_sum(float v, float* sh) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int w = 0; w < BR_THREADS / 32; w++) t += sh[w];
  return t;
}

// Eight consecutive bf16 values at p[i..i+8) of a row of H (VEC: 16-byte accesses; else element by element).
template <bool VEC>
__device__ __forceinline__ uint4 br_load(const uint16_t* p, int i, int H) {
  if constexpr (VEC) {
    return *reinterpret_cast<const uint4*>(p + i);
  } else {
    uint16_t e[8];
#pragma unroll
    for (int j = 0; j < 8; j++) e[j] = i + j < H ? p[i + j] : (uint16_t)0;
    return make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16, e[4] | (uint32_t)e[5] << 16,
                      e[6] | (uint32_t)e[7] << 16);
  }
}

// Eight floats rounded to bf16 (nearest even) in pairs.
__device__ __forceinline__ uint4 br_round(const float (&f)[8]) {
  uint32_t u[4];
#pragma unroll
  for (int j = 0; j < 4; j++) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u[j]) : "f"(f[2 * j + 1]), "f"(f[2 * j]));
  return make_uint4(u[0], u[1], u[2], u[3]);
}

template <bool VEC>
__device__ __forceinline__ void br_store(uint16_t* p, int i, int H, const uint4& u) {
  if constexpr (VEC) {
    *reinterpret_cast<uint4*>(p + i) = u;
  } else {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (i + j < H) p[i + j] = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
  }
}

__device__ __forceinline__ void br_floats(const uint4& u, float (&f)[8]) {
  f[0] = bf_lo(u.x); f[1] = bf_hi(u.x); f[2] = bf_lo(u.y); f[3] = bf_hi(u.y);
  f[4] = bf_lo(u.z); f[5] = bf_hi(u.z); f[6] = bf_lo(u.w); f[7] = bf_hi(u.w);
}

template <int VPT, bool VEC>
// Up to 2048 columns eight CTAs an SM: a prefill of 4096 rows x 8 places x 2048 takes 37 us, 42 at the four that the
// compiler's own register count allows.
__global__ void __launch_bounds__(BR_THREADS, VPT == 1 && VEC ? 8 : 1) block_residual_kernel(BlockArgs a) {
  __shared__ float sh[BR_THREADS / 32];
  pdl_wait();
  pdl_trigger();
  const size_t row = blockIdx.x;
  const uint16_t* y = a.y + row * a.places * a.H;
  float b[VPT][8];
  uint4 res[VPT];  // the residual, on its way while the places are summed
#pragma unroll
  for (int v = 0; v < VPT; v++) {
    const int i = (v * BR_THREADS + threadIdx.x) * 8;
    if (i < a.H) res[v] = br_load<VEC>(a.h + row * a.H, i, a.H);
  }
#pragma unroll
  for (int v = 0; v < VPT; v++) {
#pragma unroll
    for (int e = 0; e < 8; e++) b[v][e] = 0.f;
    const int i = (v * BR_THREADS + threadIdx.x) * 8;
    if (i < a.H) {
      if (!a.w) {
        br_floats(br_load<VEC>(y, i, a.H), b[v]);
      } else {
        const float* w = a.w + row * a.places;
        for (int j0 = 0; j0 < a.places; j0 += BR_BATCH) {  // a batch's loads leave together, whatever the weights
          uint4 u[BR_BATCH];
#pragma unroll
          for (int j = 0; j < BR_BATCH; j++)
            u[j] = j0 + j < a.places ? br_load<VEC>(y + (size_t)(j0 + j) * a.H, i, a.H) : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int j = 0; j < BR_BATCH; j++) {
            const float wj = j0 + j < a.places ? __ldg(w + j0 + j) : 0.f;
            if (wj == 0.f) continue;  // what lies there does not matter, NaN included
            float f[8];
            br_floats(u[j], f);
#pragma unroll
            for (int e = 0; e < 8; e++) b[v][e] = fmaf(wj, f[e], b[v][e]);
          }
        }
      }
    }
  }
  if (a.post) {
    float ss = 0.f;
#pragma unroll
    for (int v = 0; v < VPT; v++)
#pragma unroll
      for (int e = 0; e < 8; e++) ss = fmaf(b[v][e], b[v][e], ss);
    const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(br_sum(ss, sh), (float)a.H) + a.eps));
#pragma unroll
    for (int v = 0; v < VPT; v++) {
      const int i = (v * BR_THREADS + threadIdx.x) * 8;
      if (i < a.H) {
        float w[8];
        br_floats(br_load<VEC>(a.post, i, a.H), w);
#pragma unroll
        for (int e = 0; e < 8; e++) b[v][e] = b[v][e] * inv * (a.gemma ? 1.0f + w[e] : w[e]);
      }
    }
  }
  float ss = 0.f, sq = 0.f;
#pragma unroll
  for (int v = 0; v < VPT; v++) {
    const int i = (v * BR_THREADS + threadIdx.x) * 8;
    if (i < a.H) {
      float f[8];
      if (a.gate) {
        const uint16_t* g = a.gate + row * a.gate_row;
        if (a.gate_col) {
          br_floats(br_load<VEC>(g, i, a.H), f);
#pragma unroll
          for (int e = 0; e < 8; e++) b[v][e] *= f[e];
        } else {
          const float g0 = bf(g[0]);
#pragma unroll
          for (int e = 0; e < 8; e++) b[v][e] *= g0;
        }
      }
      br_floats(res[v], f);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        b[v][e] = fmaf(a.scale, f[e], b[v][e]);
        if (VEC || i + e < a.H) ss = fmaf(b[v][e], b[v][e], ss);
      }
      const uint4 o = br_round(b[v]);
      br_store<VEC>(a.h_out + row * a.H, i, a.H, o);
      if (a.out_sq) {
        br_floats(o, f);
#pragma unroll
        for (int e = 0; e < 8; e++)
          if (VEC || i + e < a.H) sq = fmaf(f[e], f[e], sq);
      }
    }
  }
  if (a.out_sq) {
    sq = br_sum(sq, sh);
    if (threadIdx.x == 0) a.out_sq[row] = sq;
  }
  if (a.next) {
    const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(br_sum(ss, sh), (float)a.H) + a.eps));
#pragma unroll
    for (int v = 0; v < VPT; v++) {
      const int i = (v * BR_THREADS + threadIdx.x) * 8;
      if (i < a.H) {
        float w[8];
        br_floats(br_load<VEC>(a.next, i, a.H), w);
#pragma unroll
        for (int e = 0; e < 8; e++) b[v][e] = b[v][e] * inv * (a.gemma ? 1.0f + w[e] : w[e]);
        br_store<VEC>(a.z + row * a.H, i, a.H, br_round(b[v]));
      }
    }
  }
}

template <int VPT>
static int br_launch(const BlockArgs& a, int64_t M, bool vec, cudaStream_t st) {
  return vec ? launch("block_residual_kernel", block_residual_kernel<VPT, true>, dim3((unsigned)M), dim3(BR_THREADS), 0,
                      st, a)
             : launch("block_residual_kernel", block_residual_kernel<VPT, false>, dim3((unsigned)M), dim3(BR_THREADS),
                      0, st, a);
}

}  // namespace im

using namespace im;

extern "C" int im_block_residual(const uint16_t* y, const float* weights, int64_t places, const uint16_t* h,
                                 const uint16_t* post_norm, const uint16_t* gate, int64_t gate_row_stride,
                                 int64_t gate_col_stride, float residual_scale, const uint16_t* next_norm, float eps,
                                 int gemma, int64_t M, int64_t H, uint16_t* h_out, uint16_t* z, float* out_sq,
                                 void* stream) {
  clear_error();
  IM_REQUIRE(M >= 0 && M <= 0x7fffffff && H >= 1 && places >= 1, IM_INVALID,
             "im_block_residual: bad sizes M=%lld H=%lld places=%lld", (long long)M, (long long)H, (long long)places);
  IM_REQUIRE(weights || places == 1, IM_INVALID, "im_block_residual: %lld places need weights", (long long)places);
  IM_REQUIRE(places <= BR_MAX_PLACES && H <= 16384, IM_UNSUPPORTED,
             "im_block_residual: at most %d places and 16384 columns (places=%lld H=%lld)", BR_MAX_PLACES,
             (long long)places, (long long)H);
  IM_REQUIRE(gate_col_stride == 0 || gate_col_stride == 1, IM_INVALID,
             "im_block_residual: gate column stride 0 or 1");
  if (M == 0) return IM_OK;
  IM_REQUIRE(y && h && h_out && (!next_norm || z), IM_INVALID, "im_block_residual: null pointer");
  IM_REQUIRE(aligned(y, 2) && aligned(h, 2) && aligned(h_out, 2) && aligned(z, 2) && aligned(weights, 4), IM_INVALID,
             "im_block_residual: misaligned buffer");
  BlockArgs a = {};
  a.y = y;
  a.w = weights;
  a.h = h;
  a.post = post_norm;
  a.gate = gate;
  a.next = next_norm;
  a.h_out = h_out;
  a.z = z;
  a.out_sq = out_sq;
  a.gate_row = gate_row_stride;
  a.gate_col = gate_col_stride;
  a.scale = residual_scale;
  a.eps = eps;
  a.places = (int)places;
  a.H = (int)H;
  a.gemma = gemma;
  const bool vec = H % 8 == 0 && aligned(y, 16) && aligned(h, 16) && aligned(h_out, 16) && aligned(post_norm, 16) &&
                   aligned(next_norm, 16) && aligned(z, 16) &&
                   (!gate || gate_col_stride == 0 || (aligned(gate, 16) && gate_row_stride % 8 == 0));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (H <= 2048) return br_launch<1>(a, M, vec, st);
  if (H <= 4096) return br_launch<2>(a, M, vec, st);
  if (H <= 8192) return br_launch<4>(a, M, vec, st);
  return br_launch<8>(a, M, vec, st);
}
