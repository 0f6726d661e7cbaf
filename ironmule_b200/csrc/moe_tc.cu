// Products by expert on the 5th-generation tensor cores: y[p] = W[e(p)] x[.] over packed 4-bit weights.
//
// D[128 outputs, N rows] = A[128, K] B[N, K]^T per tile: A is a 128-output block of one expert, B up to 128 gathered
// rows of it (one work item). Operands are fp16, accumulators float32 in tensor memory.
//
// Why fp16: w = scale * q + bias needs one rounding to become an operand. In bf16 (8 bits) that costs as much as the
// output's own rounding; in fp16 (11 bits) it is an eighth of it. The range is met by powers of two, which are exact:
//  * weights are scaled by the expert's largest |w| (found when they are packed), which lands in [2^7, 2^8);
//  * a row of x by its largest finite element, which lands in [2^9, 2^10) (moe_prep_kernel; bf16 values fit fp16);
//  * the gated activations h = act(g) u by a bound on the row: |g|, |u| <= |x|_2 sqrt(K) max |w|, so
//    |h| <= |x|_2^2 K max|w|^2, which lands below 2^15. No row can overflow, and typical rows stay well above
//    fp16's subnormals (the bound is loose by K or so, of 2^29).
// The factors return in float32 after the sum. A row with infinities or NaN gives those.
//
// A persistent grid (one CTA per SM) walks tiles; its warps are coupled by mbarriers only:
//  * warp 0 copies each 64-wide group of packed weights (4608 contiguous bytes) into a ring of 12;
//  * warps 14-21, two sets of 4, expand a group each: thread = output row, 64 codes -> 32 registers of fp16 pairs
//    (q exact, then one fused multiply-add) -> tensor memory, where the MMA reads A directly. Neither shared memory
//    nor its bandwidth carries expanded weights;
//  * warps 10-13 gather the item's rows, 16 bytes at a time (cp.async), into K-major 128-byte-swizzled B stages. The
//    k order within 8 follows the code expansion (k, k + 4 adjacent): the prep kernel and the gated epilogue write
//    their fp16 rows in that order;
//  * warp 1 issues 4 MMAs of K = 16 a group into one of two 128-column accumulators;
//  * warps 2-9, two sets of 4 for alternate 32 columns, read a finished accumulator (lane = output), scale it, apply
//    the gate, and store.
// Every column (row of x) is its own sum in K order, so a row's bits do not depend on the other rows.
//
// Every mbarrier wait is bounded (1 s): one that runs out sets the plan's error word and the CTA's abort flag, which
// every later wait honours; copies and MMAs in flight are drained before tensor memory is freed.
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"
#include "moe.cuh"
#include "tc.cuh"
#include "../../include/imspec.h"

namespace im {

constexpr int MT_N = MOE_TC_ROWS;       // rows of an item at most (MMA N)
constexpr int MT_S = 8;                 // A and B stages
constexpr int MT_W = 12;                // weight ring
constexpr int MT_B = MT_N * 128;        // bytes of a B stage
constexpr int MT_EPI = 8;               // epilogue warps
constexpr int MT_W_EPI = 2, MT_W_LOAD = MT_W_EPI + MT_EPI, MT_W_TRANS = MT_W_LOAD + 4;  // first warps of the roles
constexpr int MT_THREADS = (MT_W_TRANS + 8) * 32;
constexpr uint32_t MT_TMEM = 512;       // 2 accumulators of 128 columns, 8 A stages of 32
constexpr int MT_A0 = 256;
constexpr size_t MT_OFF_W = (size_t)MT_S * MT_B;
constexpr size_t MT_OFF_BAR = MT_OFF_W + (size_t)MT_W * MOE_BLOCK_BYTES;
// barriers: a stage's MMAs completed; a stage's A and B in place; weight ring; accumulators
constexpr int MT_DONE = 0, MT_FULL = MT_DONE + MT_S, MT_W_FULL = MT_FULL + MT_S, MT_W_EMPTY = MT_W_FULL + MT_W,
              MT_D_FULL = MT_W_EMPTY + MT_W, MT_D_EMPTY = MT_D_FULL + 2, MT_BARS = MT_D_EMPTY + 2;
constexpr size_t MT_OFF_META = (MT_OFF_BAR + MT_BARS * 8 + 16 + 15) / 16 * 16;  // an epilogue warp's columns
constexpr size_t MT_SMEM = 1024 + MT_OFF_META + (size_t)MT_EPI * 64 * 16;

struct TcArgs {
  MoeProduct p;
  const int4* items;
  unsigned* error;
  const __half* x16;     // rows of K, scaled
  const float* xscale;   // per row of x16: the factor it was divided by
  const float* xlog;     // per row: log2 |x|_2 (first product of a gated MLP)
  float* hscale;         // per sorted position: the factor h was divided by (written by the first product)
  const float* wmax;     // per expert: largest |w|
  size_t expert_bytes;
  int cols;              // 128-output blocks
};

__device__ __forceinline__ float mt_pow2(int e) { return __uint_as_float((uint32_t)(min(max(e, -126), 127) + 127) << 23); }

// The exponent that brings max (> 0) below 2^bits: max * 2^-e in [2^(bits-1), 2^bits); 0 for max = 0.
__device__ __forceinline__ int mt_exp(float max, int bits) {
  if (!(max > 0.f)) return 0;
  int e;
  frexpf(max, &e);
  e -= bits;
  return e < -120 ? -120 : (e > 120 ? 120 : e);
}

// Position of element k (0..7) of 8 in the operands' order.
__device__ __forceinline__ int mt_perm(int k) { return k < 4 ? 2 * k : 2 * (k - 4) + 1; }

// ---- rows of x -> scaled fp16 in operand order, one CTA per row --------------------------------------------
__global__ void __launch_bounds__(256)
moe_prep_kernel(const uint16_t* __restrict__ x, int K, __half* __restrict__ x16, float* __restrict__ xscale,
                float* __restrict__ xlog) {
  __shared__ float sh[2][8];
  pdl_wait();
  pdl_trigger();
  const size_t row = blockIdx.x;
  const uint4* src = reinterpret_cast<const uint4*>(x + row * K);
  const int n = K / 8;
  float top = 0.f;
  for (int i = threadIdx.x; i < n; i += 256) {
    const uint4 u = src[i];
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float a = fabsf(bf_lo(w[j])), b = fabsf(bf_hi(w[j]));
      if (a < INFINITY) top = fmaxf(top, a);
      if (b < INFINITY) top = fmaxf(top, b);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((threadIdx.x & 31) == 0) sh[0][threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; w++) top = fmaxf(top, sh[0][w]);
  const int e = mt_exp(top, 10);
  const float inv = mt_pow2(-e);
  float ss = 0.f;
  for (int i = threadIdx.x; i < n; i += 256) {
    const uint4 u = src[i];
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    float f[8];
    alignas(16) __half h[8];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      f[2 * j] = bf_lo(w[j]) * inv;
      f[2 * j + 1] = bf_hi(w[j]) * inv;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
      if (fabsf(f[j]) < INFINITY) ss = fmaf(f[j], f[j], ss);
      h[mt_perm(j)] = __float2half_rn(f[j]);
    }
    *reinterpret_cast<uint4*>(x16 + row * K + 8 * i) = *reinterpret_cast<const uint4*>(h);
  }
  ss = warp_sum(ss);
  if ((threadIdx.x & 31) == 0) sh[1][threadIdx.x >> 5] = ss;
  __syncthreads();
  if (threadIdx.x == 0) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < 8; w++) t += sh[1][w];
    xscale[row] = mt_pow2(e);
    xlog[row] = 0.5f * log2f(t) + (float)e;  // -inf for a zero row
  }
}

// ---- the products ----------------------------------------------------------------------------------------------
// fp16 pairs (k, k + 4) of a word's eight codes: scale * q + bias, one rounding.
__device__ __forceinline__ void mt_expand(uint32_t u, __half2 s, __half2 b, uint32_t* out) {
  const __half2 m1024 = __half2half2(__ushort_as_half(0xE400)), m64 = __half2half2(__ushort_as_half(0xD400)),
                r16 = __half2half2(__ushort_as_half(0x2C00));  // -1024, -64, 1/16
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const uint32_t v = u >> (8 * i);
    uint32_t lo = (v & 0x000F000Fu) | 0x64006400u, hi = (v & 0x00F000F0u) | 0x64006400u;  // 1024 + q, 1024 + 16 q
    const __half2 ql = __hadd2(*reinterpret_cast<__half2*>(&lo), m1024);
    const __half2 qh = __hfma2(*reinterpret_cast<__half2*>(&hi), r16, m64);
    const __half2 wl = __hfma2(ql, s, b), wh = __hfma2(qh, s, b);
    out[2 * i] = *reinterpret_cast<const uint32_t*>(&wl);
    out[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&wh);
  }
}

__device__ __forceinline__ float mt_gated(bool geglu, float g, float u) {
  if (!geglu) return __fdividef(g, 1.0f + __expf(-g)) * u;
  const float inner = 0.7978845608028654f * (g + 0.044715f * g * g * g);
  return 0.5f * g * (1.0f + tanhf(inner)) * u;
}

__device__ __forceinline__ void mt_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void mt_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

template <bool GLU>
__global__ void __launch_bounds__(MT_THREADS, 1) moe_tc_kernel(TcArgs a) {
  extern __shared__ unsigned char mt_raw[];
  const uint32_t raw = qt_smem(mt_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  unsigned char* sbase = mt_raw + (base - raw);
  const uint32_t bars = base + (uint32_t)MT_OFF_BAR;
  uint32_t* holder = reinterpret_cast<uint32_t*>(sbase + MT_OFF_BAR + MT_BARS * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(holder + 1);

  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int G = a.p.K >> 6;
  const int nout = GLU ? a.p.N >> 1 : a.p.N;

  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(qt_smem(holder)),
                 "r"(MT_TMEM));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (threadIdx.x == 0) {
    unsigned long long* b = reinterpret_cast<unsigned long long*>(sbase + MT_OFF_BAR);
    for (int s = 0; s < MT_S; s++) {
      qt_init(&b[MT_DONE + s], 1u);
      qt_init(&b[MT_FULL + s], 4u + 128u);  // four expansion warps, every gather thread
    }
    for (int s = 0; s < MT_W; s++) {
      qt_init(&b[MT_W_FULL + s], 1u);
      qt_init(&b[MT_W_EMPTY + s], 4u);
    }
    for (int s = 0; s < 2; s++) {
      qt_init(&b[MT_D_FULL + s], 1u);
      qt_init(&b[MT_D_EMPTY + s], MT_EPI);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *holder;
  // The routing's plan was finished before the launch that precedes this one (the prep kernel, or the first product)
  // let this one begin: the plan and the weights are read without waiting, rows and outputs only after pdl_wait().
  const int ntiles = a.p.plan[0] * a.cols;

  if (warp == 0) {
    // ---- weights -------------------------------------------------------------------------------------------
    if (lane == 0) {
      uint32_t s = 0, phase = 0;
      int k = 0;
      for (int tile = blockIdx.x; tile < ntiles; tile += gridDim.x) {
        const int expert = a.items[tile / a.cols].x;
        if (expert == a.p.E) continue;
        const unsigned char* src =
            a.p.wp + (size_t)expert * a.expert_bytes + (size_t)(tile % a.cols) * G * MOE_BLOCK_BYTES;
        for (int g = 0; g < G; g++, k++) {
          const uint32_t full = bars + 8 * (MT_W_FULL + s);
          if (!qt_wait_short(bars + 8 * (MT_W_EMPTY + s), phase ^ 1u, abort_flag, a.error)) goto weights_done;
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(full),
                       "r"((uint32_t)MOE_BLOCK_BYTES)
                       : "memory");
          asm volatile(
              "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                  base + (uint32_t)MT_OFF_W + s * MOE_BLOCK_BYTES),
              "l"(src), "r"((uint32_t)MOE_BLOCK_BYTES), "r"(full)
              : "memory");
          src += MOE_BLOCK_BYTES;
          if (++s == MT_W) s = 0, phase ^= 1u;
        }
      }
    weights_done:
      if (*abort_flag)  // copies still landing in this CTA's shared memory finish before it exits
        for (int j = k > MT_W ? k - MT_W : 0; j < k; j++)
          qt_drain(reinterpret_cast<unsigned long long*>(sbase + MT_OFF_BAR) + MT_W_FULL + j % MT_W,
                   (uint32_t)((j / MT_W) & 1));
    }
  } else if (warp == 1) {
    // ---- MMA issue -----------------------------------------------------------------------------------------
    // (the whole warp walks the loop, so that its addresses stay in uniform registers; one lane issues)
    const bool leader = qt_elect();
    uint32_t s = 0, phase = 0;
    int k = 0, t = 0;
    for (int tile = blockIdx.x; tile < ntiles; tile += gridDim.x) {
      const int4 item = a.items[tile / a.cols];
      if (item.x == a.p.E) continue;
      // f32 accumulate, f16 A and B, K-major, N = the item's rows in sixteens, M = 128
      const uint32_t idesc = (1u << 4) | ((uint32_t)((item.z + 15) / 16 * 2) << 17) | ((128u >> 4) << 24);
      const int buf = t & 1;
      if (!qt_wait_short(bars + 8 * (MT_D_EMPTY + buf), (uint32_t)((t / 2 + 1) & 1), abort_flag, a.error)) break;
      const uint32_t d = tmem + (uint32_t)(buf * MT_N);
      int g = 0;
      for (; g < G; g++, k++) {
        if (!qt_wait_short(bars + 8 * (MT_FULL + s), phase, abort_flag, a.error)) break;
        // the gathered rows were written through the generic proxy; the MMA reads them through the async one
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (leader) {
          const uint64_t bd = qt_desc(base + s * MT_B);
          const uint32_t ta = tmem + MT_A0 + 32 * s;
#pragma unroll
          for (int q = 0; q < 4; q++)
            asm volatile(
                "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
                "r"(ta + 8 * q), "l"(bd + 2 * q), "r"(idesc), "r"((uint32_t)(g + q > 0)));
          mt_commit(bars + 8 * (MT_DONE + s));
        }
        __syncwarp();
        if (++s == MT_S) s = 0, phase ^= 1u;
      }
      if (g < G) break;
      if (leader) mt_commit(bars + 8 * (MT_D_FULL + buf));
      __syncwarp();
      t++;
    }
    if (*abort_flag && k > 0)
      qt_drain(reinterpret_cast<unsigned long long*>(sbase + MT_OFF_BAR) + MT_DONE + (k - 1) % MT_S,
               (uint32_t)(((k - 1) / MT_S) & 1));
  } else if (warp < MT_W_LOAD) {
    // ---- epilogue: lane = output of the block, columns = the item's rows ---------------------------------------
    const int q = warp & 3, set = (warp - MT_W_EPI) >> 2;
    float4* meta = reinterpret_cast<float4*>(sbase + MT_OFF_META) + (warp - MT_W_EPI) * 64;
    const bool paired = (nout & 1) == 0 && (reinterpret_cast<uintptr_t>(a.p.y) & 3) == 0;
    pdl_wait();
    pdl_trigger();
    int t = 0;
    for (int tile = blockIdx.x; tile < ntiles; tile += gridDim.x) {
      const int4 item = a.items[tile / a.cols];
      const int col = tile % a.cols, rows = item.z;
      if (item.x == a.p.E) {  // places without an expert: zeros (a sorted output holds none of them)
        if (a.p.dst != MOE_SORTED) {
          const int f = col * 128 + q * 32 + lane;
          for (int j = set; j < rows; j += 2)
            if (f < nout) a.p.y[(size_t)a.p.pairs[item.y + j] * nout + f] = 0;
        }
        continue;
      }
      // this warp's columns 64 i + 32 set + lane: the factors of the accumulator and of h, the output row
      const float wmax = a.wmax[item.x];
      const float wscale = mt_pow2(mt_exp(wmax, 8));
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const int c = 64 * i + 32 * set + lane;
        if (c < rows) {
          const int pos = item.y + c, pair = a.p.pairs[pos];
          const int src = a.p.src == MOE_SORTED ? pos : (a.p.src == MOE_BY_PAIR ? pair : pair / a.p.top_k);
          float hs = 0.f;
          if constexpr (GLU) {
            const float bound = 2.f * a.xlog[src] + log2f((float)a.p.K) + 2.f * log2f(wmax);
            const int e = bound > -100.f ? (int)ceilf(fminf(bound, 135.f)) - 15 : -110;
            hs = mt_pow2(-e);
            if (col == 0 && q == 0) a.hscale[pos] = mt_pow2(e);
          }
          meta[32 * i + lane] =
              make_float4(a.xscale[src], hs, __int_as_float(a.p.dst == MOE_SORTED ? pos : pair), 0.f);
        }
      }
      __syncwarp();
      const int buf = t & 1;
      if (!qt_wait_short(bars + 8 * (MT_D_FULL + buf), (uint32_t)((t / 2) & 1), abort_flag, a.error)) break;
      t++;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
      for (int i = 0; 64 * i + 32 * set < rows; i++) {
        const int c0 = 64 * i + 32 * set, n = min(32, rows - c0);
        uint32_t v[32];
        const uint32_t ta = tmem + ((uint32_t)(32 * q) << 16) + (uint32_t)(buf * MT_N + c0);
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
            "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
            : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
              "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
              "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
              "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
            : "r"(ta));
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        const float4* m = meta + 32 * i;
        // Of two columns j, j + 1 each lane finishes one, with its partner lane's value of it (the partner: the other
        // half of a gated output, or the neighbouring output, so that two outputs leave in one store).
        const int other = GLU ? 16 : 1;
        const bool second = lane & other;
        const int f = GLU ? (col * 4 + q) * 16 + (lane & 15) : col * 128 + q * 32 + lane;
        if constexpr (GLU) {
          __half* h = reinterpret_cast<__half*>(a.p.y) + (f & ~7) + mt_perm(f & 7);
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float give = __uint_as_float(second ? v[j] : v[j + 1]);
            const float keep = __uint_as_float(second ? v[j + 1] : v[j]);
            const float got = __shfl_xor_sync(0xffffffffu, give, 16);
            const float4 mj = m[second ? j + 1 : j];
            const float x1 = mj.x * wscale;
            // lanes 0-15 hold gate features, 16-31 the matching up features
            const float g = (second ? got : keep) * x1, u = (second ? keep : got) * x1;
            const float o = mt_gated(a.p.epilogue == IM_EPI_GEGLU, g, u) * mj.y;
            if (j + (second ? 1 : 0) < n && f < nout)
              h[(size_t)__float_as_int(mj.z) * nout] = __float2half_rn(o);
          }
        } else if (paired) {
          uint16_t* y = a.p.y + (f & ~1);
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float give = __uint_as_float(second ? v[j] : v[j + 1]);
            const float keep = __uint_as_float(second ? v[j + 1] : v[j]);
            const float got = __shfl_xor_sync(0xffffffffu, give, 1);
            const float4 mj = m[second ? j + 1 : j];
            const float k1 = keep * wscale * mj.x, g1 = got * wscale * mj.x;
            uint32_t o;
            asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(o) : "f"(second ? k1 : g1), "f"(second ? g1 : k1));
            if (j + (second ? 1 : 0) < n && f < nout)
              *reinterpret_cast<uint32_t*>(y + (size_t)__float_as_int(mj.z) * nout) = o;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; j++) {
            const float4 mj = m[j];
            if (j < n && f < nout)
              a.p.y[(size_t)__float_as_int(mj.z) * nout + f] = to_bf(__uint_as_float(v[j]) * wscale * mj.x);
          }
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mt_arrive(bars + 8 * (MT_D_EMPTY + buf));
    }
  } else if (warp < MT_W_TRANS) {
    // ---- gather of B -------------------------------------------------------------------------------------------
    const int th = threadIdx.x - MT_W_LOAD * 32, c = th & 7, r0 = th >> 3;  // 16-byte chunk c of rows r0 + 16 i
    const uint32_t dst0 = base + (uint32_t)(r0 * 128 + ((c ^ (r0 & 7)) << 4));
    pdl_wait();
    uint32_t s = 0, phase = 1;
    for (int tile = blockIdx.x; tile < ntiles; tile += gridDim.x) {
      const int4 item = a.items[tile / a.cols];
      if (item.x == a.p.E) continue;
      const __half* src[MT_N / 16];
#pragma unroll
      for (int i = 0; i < MT_N / 16; i++) {
        const int r = min(r0 + 16 * i, item.z - 1);  // (rows past the item's repeat its last one: columns nobody reads)
        const int pos = item.y + r;
        int row = pos;
        if (a.p.src != MOE_SORTED) {
          row = a.p.pairs[pos];
          if (a.p.src == MOE_BY_TOKEN) row /= a.p.top_k;
        }
        src[i] = a.x16 + (size_t)row * a.p.K + 8 * c;
      }
      const int n16 = (item.z + 15) / 16;
      for (int g = 0; g < G; g++) {
        if (!qt_wait_short(bars + 8 * (MT_DONE + s), phase, abort_flag, a.error)) goto gather_done;
        const uint32_t dst = dst0 + s * MT_B;
#pragma unroll
        for (int i = 0; i < MT_N / 16; i++) {
          if (i < n16)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + (uint32_t)(i * 2048)), "l"(src[i])
                         : "memory");
          src[i] += 64;
        }
        // arrives once this thread's copies have landed
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bars + 8 * (MT_FULL + s)) : "memory");
        if (++s == MT_S) s = 0, phase ^= 1u;
      }
    }
  gather_done:
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    // ---- code expansion: set 0 takes the even steps of the CTA's sequence, set 1 the odd ones ---------------------
    const int set = (warp - MT_W_TRANS) >> 2, q = warp & 3;
    const uint32_t code_off = (uint32_t)(q * 1024 + lane * 16);
    const uint32_t sb_off = (uint32_t)(4096 + q * 128 + (lane & 7) * 16 + (lane >> 3) * 2);
    uint32_t s = set, phase = 1, sw = set, wphase = 0;
    int skip = set;  // steps of the next tile that lie before this set's next one
    for (int tile = blockIdx.x; tile < ntiles; tile += gridDim.x) {
      const int expert = a.items[tile / a.cols].x;
      if (expert == a.p.E) continue;
      const float inv = mt_pow2(-mt_exp(a.wmax[expert], 8));
      int g = skip;
      for (; g < G; g += 2) {
        if (!qt_wait_short(bars + 8 * (MT_W_FULL + sw), wphase, abort_flag, a.error)) goto expand_done;
        const unsigned char* w = sbase + MT_OFF_W + sw * MOE_BLOCK_BYTES;
        const uint4 c0 = *reinterpret_cast<const uint4*>(w + code_off);
        const uint4 c1 = *reinterpret_cast<const uint4*>(w + code_off + 512);
        const float sf = bf(*reinterpret_cast<const uint16_t*>(w + sb_off)) * inv;
        const float of = bf(*reinterpret_cast<const uint16_t*>(w + sb_off + 8)) * inv;
        const __half2 s2 = __float2half2_rn(sf), b2 = __float2half2_rn(of);
        uint32_t p[32];
        const uint32_t words[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
#pragma unroll
        for (int i = 0; i < 8; i++) mt_expand(words[i], s2, b2, p + 4 * i);
        __syncwarp();
        if (lane == 0) mt_arrive(bars + 8 * (MT_W_EMPTY + sw));
        if ((sw += 2) >= MT_W) sw -= MT_W, wphase ^= 1u;
        if (!qt_wait_short(bars + 8 * (MT_DONE + s), phase, abort_flag, a.error)) goto expand_done;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile(
            "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
            "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(
                tmem + ((uint32_t)(32 * q) << 16) + MT_A0 + 32 * s),
            "r"(p[0]), "r"(p[1]), "r"(p[2]), "r"(p[3]), "r"(p[4]), "r"(p[5]), "r"(p[6]), "r"(p[7]), "r"(p[8]),
            "r"(p[9]), "r"(p[10]), "r"(p[11]), "r"(p[12]), "r"(p[13]), "r"(p[14]), "r"(p[15]), "r"(p[16]),
            "r"(p[17]), "r"(p[18]), "r"(p[19]), "r"(p[20]), "r"(p[21]), "r"(p[22]), "r"(p[23]), "r"(p[24]),
            "r"(p[25]), "r"(p[26]), "r"(p[27]), "r"(p[28]), "r"(p[29]), "r"(p[30]), "r"(p[31])
            : "memory");
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mt_arrive(bars + 8 * (MT_FULL + s));
        if ((s += 2) >= MT_S) s -= MT_S, phase ^= 1u;
      }
      skip = g - G;
    }
  expand_done:;
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();  // every MMA of this CTA has completed (or been drained)
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(MT_TMEM));
  }
}

// Workspace of the tensor-core path: the scaled rows and their factors.
MoeTcSpace moe_tc_space(int64_t rows, int64_t K, int64_t pairs, int64_t I) {
  MoeTcSpace s;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t r = at;
    at += (bytes + 255) / 256 * 256;
    return r;
  };
  s.x16 = take((size_t)rows * K * 2);
  s.xscale = take((size_t)rows * 4);
  s.xlog = take((size_t)rows * 4);
  s.h16 = take((size_t)pairs * I * 2);
  s.hscale = take(I ? (size_t)pairs * 4 : 0);
  s.total = at;
  return s;
}

int moe_prep_launch(const uint16_t* x, int64_t rows, int64_t K, const MoeTcSpace& s, void* workspace,
                    cudaStream_t st) {
  char* ws = reinterpret_cast<char*>(workspace);
  return launch("moe_prep_kernel", moe_prep_kernel, dim3((unsigned)rows), dim3(256), 0, st, x, (int)K,
                reinterpret_cast<__half*>(ws + s.x16), reinterpret_cast<float*>(ws + s.xscale),
                reinterpret_cast<float*>(ws + s.xlog));
}

template <bool GLU>
static int mt_launch(const TcArgs& a, int64_t tiles, cudaStream_t st) {
  static int sms = 0;
  if (!sms) {
    int dev = 0, n = 0;
    cudaError_t e = cudaFuncSetAttribute(moe_tc_kernel<GLU>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)MT_SMEM);
    if (e == cudaSuccess) e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) {
      set_error("moe_tc_kernel: %s", cudaGetErrorString(e));
      return IM_CUDA_ERROR;
    }
    sms = n;
  }
  return launch("moe_tc_kernel", moe_tc_kernel<GLU>, dim3((unsigned)(tiles < sms ? tiles : sms)), dim3(MT_THREADS),
                MT_SMEM, st, a);
}

int moe_tc_launch(const MoePlan& p, const MoeProduct& prod, const MoeTcSpace& s, void* workspace, cudaStream_t st) {
  char* ws = reinterpret_cast<char*>(workspace);
  const bool second = prod.src == MOE_SORTED;
  TcArgs a = {};
  a.p = prod;
  a.items = reinterpret_cast<const int4*>(prod.plan + MOE_PLAN_HEADER);
  a.error = reinterpret_cast<unsigned*>(const_cast<int*>(prod.plan)) + 1;
  a.x16 = reinterpret_cast<const __half*>(ws + (second ? s.h16 : s.x16));
  a.xscale = reinterpret_cast<const float*>(ws + (second ? s.hscale : s.xscale));
  a.xlog = reinterpret_cast<const float*>(ws + s.xlog);
  a.hscale = reinterpret_cast<float*>(ws + s.hscale);
  const int G = prod.K / 64;
  a.cols = (prod.N + 127) / 128;
  a.expert_bytes = (size_t)a.cols * G * MOE_BLOCK_BYTES;
  a.wmax = reinterpret_cast<const float*>(prod.wp + (size_t)prod.E * a.expert_bytes);
  const int64_t tiles = p.max_items * a.cols;
  IM_REQUIRE(tiles < (1ll << 31), IM_UNSUPPORTED, "grouped product: too many tiles");
  if (prod.epilogue == IM_EPI_STORE) return mt_launch<false>(a, tiles, st);
  return mt_launch<true>(a, tiles, st);
}

}  // namespace im
