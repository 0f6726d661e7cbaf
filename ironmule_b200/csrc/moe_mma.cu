// Products by expert for few rows an expert: y[p] = W[e(p)] x[.] over packed 4-bit weights, on warp-level tensor-core MMA.
//
// An item is up to 8 NT rows of one expert. A CTA is 4 warps = the 4 tiles (128 outputs) of a packed block; each warp
// streams its tile's part of the block's groups through a register ring, expands the codes to exact bf16 (128 + q) and
// folds each group's affine in float32: tot += s acc + (b - 128 s) sum(x). The item's input rows are gathered by index
// into shared memory as MMA fragments, one K segment at a time.
//
// K is cut into segments by (N, K) alone and a row's sum is the segments' sums added in order, so a row's bits depend
// neither on the other rows nor on the rows per item. With few items (a decoded token: 8) one CTA takes one segment and
// the segments of a tile form a thread-block cluster that adds them through distributed shared memory; with many, a
// CTA walks all segments itself. Same bits.
//
// Bound by HBM (0.5625 B a weight of every chosen expert). Weights depend on the routing, so they cannot be fetched
// before the routing is known; the second product of a gated MLP knows it and fetches before its dependency wait.
#include "common.cuh"
#include "moe.cuh"
#include "../../include/imspec.h"

namespace im {

constexpr int MM_WARPS = 4;
constexpr int MM_THREADS = MM_WARPS * 32;
constexpr int MM_DEPTH = 3;          // units in flight per warp
constexpr int MM_SEG_GROUPS = 32;    // groups of a segment at most (shared memory)
constexpr int MM_MAX_CLUSTER = 8;    // the portable cluster size
constexpr int MM_WAVE = 148 * 4;     // CTAs of one wave

struct MmArgs {
  MoeProduct p;
  const int4* items;
  size_t expert_bytes;
  int tiles, segs, rg;
};

// K segments: the most that fill one wave with the eight items of a decoded token, at least 4 groups each, and few
// enough groups each for shared memory. A function of (N, K) only.
static int mm_segments(int ctas_x, int G) {
  int s = MM_WAVE / (8 * ctas_x);
  if (s > G / 4) s = G / 4;
  if (s > MM_MAX_CLUSTER) s = MM_MAX_CLUSTER;
  const int need = (G + MM_SEG_GROUPS - 1) / MM_SEG_GROUPS;
  return s < need ? need : s;
}

__device__ __forceinline__ void mm_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight codes (nibbles i and i + 4 of a pair) as exact bf16 128 + q.
__device__ __forceinline__ void mm_codes(uint32_t u, uint32_t* p) {
  p[0] = (u & 0x000F000Fu) | 0x43004300u;
  p[1] = ((u >> 4) & 0x000F000Fu) | 0x43004300u;
  p[2] = ((u >> 8) & 0x000F000Fu) | 0x43004300u;
  p[3] = ((u >> 12) & 0x000F000Fu) | 0x43004300u;
}

__device__ __forceinline__ void mm_prefetch_l2(const void* p, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

// Dynamic shared memory: fragments [rg][NT][32][2 x 16 B], group sums [rg][8 NT], segment sums [4 warps][8 NT][32].
struct MmSmem {
  size_t sx, part, total;
};
__host__ __device__ inline MmSmem mm_smem(int nt, int rg, bool split) {
  MmSmem m;
  m.sx = (size_t)rg * nt * 1024;
  m.part = m.sx + (size_t)rg * nt * 8 * 4;
  m.total = m.part + (split ? (size_t)MM_WARPS * 8 * nt * 32 * 4 : 0);
  return m;
}

// gate and up of one output feature, in float32, rounded once by the caller
__device__ __forceinline__ float mm_act(int epilogue, float g, float u) {
  if (epilogue == IM_EPI_SWIGLU) return g / (1.0f + expf(-g)) * u;
  const float inner = 0.7978845608028654f * (g + 0.044715f * g * g * g);
  return 0.5f * g * (1.0f + tanhf(inner)) * u;
}

// grid (CTA columns of 4 tiles, SPLIT ? segments : 1, items)
template <int NT, bool GLU, bool SPLIT>
__global__ void __launch_bounds__(MM_THREADS, NT == 1 ? 4 : 2) moe_mma_kernel(MmArgs a) {
  extern __shared__ __align__(16) unsigned char mm_raw[];
  __shared__ int src_s[8 * NT], dst_s[8 * NT];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int G = a.p.K >> 6;
  const int nout = GLU ? a.p.N >> 1 : a.p.N;
  if (!a.p.early) {
    pdl_wait();
    pdl_trigger();
  }
  if ((int)blockIdx.z >= a.p.plan[0]) return;  // (a whole cluster leaves)
  const int4 item = a.items[blockIdx.z];
  const int rows = item.z;
  const int tile = blockIdx.x * MM_WARPS + warp;
  const bool live = tile < a.tiles;

  if (item.x == a.p.E) {  // places without an expert: zeros (a sorted output holds none of them)
    if (a.p.early) {
      pdl_wait();
      pdl_trigger();
    }
    if (a.p.dst != MOE_SORTED && (!SPLIT || blockIdx.y == 0)) {
      const int f0 = blockIdx.x * MM_WARPS * (GLU ? 16 : 32), f1 = min(nout, f0 + MM_WARPS * (GLU ? 16 : 32));
      for (int i = threadIdx.x; i < rows * (f1 - f0); i += MM_THREADS)
        a.p.y[(size_t)a.p.pairs[item.y + i / (f1 - f0)] * nout + f0 + i % (f1 - f0)] = 0;
    }
    return;
  }

  const int seg0 = SPLIT ? blockIdx.y : 0, seg1 = SPLIT ? seg0 + 1 : a.segs;
  const unsigned char* wblock =
      a.p.wp + (size_t)item.x * a.expert_bytes + (size_t)blockIdx.x * G * MOE_BLOCK_BYTES;
  // this lane's 8 bytes (words 2t, 2t + 1 of the group) of rows g + 8 j: + 128 j; its scales and biases
  const int code_off = warp * 1024 + (t >> 1) * 512 + g * 16 + (t & 1) * 8, sb_off = 4096 + warp * 128 + g * 16;
  uint2 rc[MM_DEPTH][4];
  uint4 rsb[MM_DEPTH];
  auto fetch = [&](const unsigned char* p, uint2 (&c)[4], uint4& sb) {
#pragma unroll
    for (int j = 0; j < 4; j++) c[j] = ldg_stream_u2(p + code_off + 128 * j);
    sb = __ldg(reinterpret_cast<const uint4*>(p + sb_off));
  };
  // the first units of a segment into the register ring, the rest of it towards L2
  auto begin = [&](int seg) {
    const int cg0 = (int)((long long)G * seg / a.segs), ng = (int)((long long)G * (seg + 1) / a.segs) - cg0;
    const unsigned char* up = wblock + (size_t)cg0 * MOE_BLOCK_BYTES;
    if (threadIdx.x == 0 && ng > MM_DEPTH)
      mm_prefetch_l2(up + MM_DEPTH * MOE_BLOCK_BYTES, (uint32_t)(ng - MM_DEPTH) * MOE_BLOCK_BYTES);
    if (!live) return;
#pragma unroll
    for (int d = 0; d < MM_DEPTH; d++)
      if (d < ng) fetch(up + (size_t)d * MOE_BLOCK_BYTES, rc[d], rsb[d]);
  };
  begin(seg0);
  if (threadIdx.x < 8 * NT && (int)threadIdx.x < rows) {
    const int pos = item.y + threadIdx.x, pair = a.p.pairs[pos];
    src_s[threadIdx.x] = a.p.src == MOE_SORTED ? pos : (a.p.src == MOE_BY_PAIR ? pair : pair / a.p.top_k);
    dst_s[threadIdx.x] = a.p.dst == MOE_SORTED ? pos : pair;
  }
  if (a.p.early) {
    pdl_wait();
    pdl_trigger();
  }
  __syncthreads();

  const MmSmem lay = mm_smem(NT, a.rg, SPLIT);
  uint4 (*xf)[NT][32][2] = reinterpret_cast<uint4 (*)[NT][32][2]>(mm_raw);
  float (*sxs)[NT * 8] = reinterpret_cast<float (*)[NT * 8]>(mm_raw + lay.sx);
  float tot[2][NT][4], sum[2][NT][4];
#pragma unroll
  for (int tt = 0; tt < 2; tt++)
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int e = 0; e < 4; e++) sum[tt][nt][e] = 0.f;

#pragma unroll 1
  for (int seg = seg0; seg < seg1; seg++) {
    const int cg0 = (int)((long long)G * seg / a.segs), ng = (int)((long long)G * (seg + 1) / a.segs) - cg0;
    // ---- the rows' fragments and group sums of this segment: a thread takes (group, row, quarter) = 16 values
    for (int job = threadIdx.x; job < ng * NT * 32; job += MM_THREADS) {
      const int tq = job & 3, m = (job >> 2) % (NT * 8), gl = (job >> 2) / (NT * 8);
      uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
      float part = 0.f;
      if (m < rows) {
        const uint16_t* xp = a.p.x + (size_t)src_s[m] * a.p.K + (size_t)(cg0 + gl) * 64 + 16 * tq;
        lo = *reinterpret_cast<const uint4*>(xp);
        hi = *reinterpret_cast<const uint4*>(xp + 8);
        const uint32_t* l32 = reinterpret_cast<const uint32_t*>(&lo);
        const uint32_t* h32 = reinterpret_cast<const uint32_t*>(&hi);
#pragma unroll
        for (int e = 0; e < 4; e++) part += bf_lo(l32[e]) + bf_hi(l32[e]);
#pragma unroll
        for (int e = 0; e < 4; e++) part += bf_lo(h32[e]) + bf_hi(h32[e]);
      }
      uint4 f0, f1;
      f0.x = __byte_perm(lo.x, lo.z, 0x5410);
      f0.y = __byte_perm(lo.x, lo.z, 0x7632);
      f0.z = __byte_perm(lo.y, lo.w, 0x5410);
      f0.w = __byte_perm(lo.y, lo.w, 0x7632);
      f1.x = __byte_perm(hi.x, hi.z, 0x5410);
      f1.y = __byte_perm(hi.x, hi.z, 0x7632);
      f1.z = __byte_perm(hi.y, hi.w, 0x5410);
      f1.w = __byte_perm(hi.y, hi.w, 0x7632);
      xf[gl][m >> 3][(m & 7) * 4 + tq][0] = f0;
      xf[gl][m >> 3][(m & 7) * 4 + tq][1] = f1;
      part += __shfl_xor_sync(0xffffffffu, part, 1);
      part += __shfl_xor_sync(0xffffffffu, part, 2);
      if (tq == 0) sxs[gl][m] = part;
    }
    __syncthreads();

    // ---- this warp's tile over the segment
#pragma unroll
    for (int tt = 0; tt < 2; tt++)
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 4; e++) tot[tt][nt][e] = 0.f;
    const unsigned char* up = wblock + (size_t)cg0 * MOE_BLOCK_BYTES;
    auto unit = [&](const int gl, uint2 (&r)[4], uint4& rb) {
      const uint2 c[4] = {r[0], r[1], r[2], r[3]};
      const uint4 sb = rb;
      if (gl + MM_DEPTH < ng) fetch(up + (size_t)(gl + MM_DEPTH) * MOE_BLOCK_BYTES, r, rb);
      uint32_t px[NT][8];
      float sx[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        const uint4 f0 = xf[gl][nt][lane][0], f1 = xf[gl][nt][lane][1];
        px[nt][0] = f0.x; px[nt][1] = f0.y; px[nt][2] = f0.z; px[nt][3] = f0.w;
        px[nt][4] = f1.x; px[nt][5] = f1.y; px[nt][6] = f1.z; px[nt][7] = f1.w;
        const float2 s2 = *reinterpret_cast<const float2*>(&sxs[gl][nt * 8 + 2 * t]);
        sx[nt][0] = s2.x;
        sx[nt][1] = s2.y;
      }
      const float sv[4] = {bf_lo(sb.x), bf_hi(sb.x), bf_lo(sb.y), bf_hi(sb.y)};
      const float bv[4] = {bf_lo(sb.z), bf_hi(sb.z), bf_lo(sb.w), bf_hi(sb.w)};
      const uint32_t wd[2][4] = {{c[0].x, c[0].y, c[1].x, c[1].y}, {c[2].x, c[2].y, c[3].x, c[3].y}};
#pragma unroll
      for (int tt = 0; tt < 2; tt++) {
        uint32_t pa[8], pb[8];
        mm_codes(wd[tt][0], pa);
        mm_codes(wd[tt][1], pa + 4);
        mm_codes(wd[tt][2], pb);
        mm_codes(wd[tt][3], pb + 4);
        float acc[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 4; e++) acc[nt][e] = 0.f;
#pragma unroll
        for (int q = 0; q < 4; q++)
#pragma unroll
          for (int nt = 0; nt < NT; nt++)
            mm_mma(acc[nt], pa[2 * q], pb[2 * q], pa[2 * q + 1], pb[2 * q + 1], px[nt][2 * q], px[nt][2 * q + 1]);
        const float s0 = sv[2 * tt], s1 = sv[2 * tt + 1];
        const float b0 = fmaf(-128.f, s0, bv[2 * tt]), b1 = fmaf(-128.f, s1, bv[2 * tt + 1]);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          tot[tt][nt][0] = fmaf(b0, sx[nt][0], fmaf(s0, acc[nt][0], tot[tt][nt][0]));
          tot[tt][nt][1] = fmaf(b0, sx[nt][1], fmaf(s0, acc[nt][1], tot[tt][nt][1]));
          tot[tt][nt][2] = fmaf(b1, sx[nt][0], fmaf(s1, acc[nt][2], tot[tt][nt][2]));
          tot[tt][nt][3] = fmaf(b1, sx[nt][1], fmaf(s1, acc[nt][3], tot[tt][nt][3]));
        }
      }
    };
    if (live) {
#pragma unroll 1
      for (int gl0 = 0; gl0 < ng; gl0 += MM_DEPTH) {
#pragma unroll
        for (int d = 0; d < MM_DEPTH; d++) {
          if (gl0 + d >= ng) break;
          unit(gl0 + d, rc[d], rsb[d]);
        }
      }
    }
    if constexpr (!SPLIT) {
      if (seg + 1 < seg1) begin(seg + 1);
#pragma unroll
      for (int tt = 0; tt < 2; tt++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 4; e++) sum[tt][nt][e] += tot[tt][nt][e];
      __syncthreads();  // every warp has read the fragments
    }
  }

  bool finish = live;
  if constexpr (SPLIT) {
    // the segments' sums of a tile, added in order by the CTA of rank warp % segments
    constexpr int NV = 2 * NT * 4;
    float* mine = reinterpret_cast<float*>(mm_raw + lay.part) + warp * NV * 32;
#pragma unroll
    for (int tt = 0; tt < 2; tt++)
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 4; e++) mine[((tt * NT + nt) * 4 + e) * 32 + lane] = tot[tt][nt][e];
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    finish = live && (int)blockIdx.y == warp % a.segs;
    if (finish) {
      const uint32_t local = (uint32_t)__cvta_generic_to_shared(mine);
      for (int s = 0; s < a.segs; s++) {
        uint32_t peer;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(local), "r"(s));
#pragma unroll
        for (int v = 0; v < NV; v++) {
          float f;
          asm volatile("ld.shared::cluster.f32 %0, [%1];"
                       : "=f"(f)
                       : "r"(peer + (uint32_t)(v * 32 + lane) * 4u)
                       : "memory");
          sum[v / (NT * 4)][v / 4 % NT][v % 4] += f;
        }
      }
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  }
  if (finish) {
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int m = nt * 8 + 2 * t + (e & 1);
        if (m >= rows) continue;
        uint16_t* y = a.p.y + (size_t)dst_s[m] * nout;
        if constexpr (GLU) {  // tile rows 0-15 are gate features, 16-31 the matching up features
          const int f = tile * 16 + g + ((e >> 1) << 3);
          if (f < nout) y[f] = to_bf(mm_act(a.p.epilogue, sum[0][nt][e], sum[1][nt][e]));
        } else {
#pragma unroll
          for (int tt = 0; tt < 2; tt++) {
            const int r = tile * 32 + tt * 16 + g + ((e >> 1) << 3);
            if (r < nout) y[r] = to_bf(sum[tt][nt][e]);
          }
        }
      }
  }
  if constexpr (SPLIT)
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // no CTA leaves while a peer reads its sums
}

template <int NT, bool GLU, bool SPLIT>
static int mm_launch(const MmArgs& a, int ctas_x, int64_t items, cudaStream_t st) {
  const size_t smem = mm_smem(NT, a.rg, SPLIT).total;
  auto kernel = moe_mma_kernel<NT, GLU, SPLIT>;
  static bool configured = false;
  if (!configured) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)mm_smem(NT, MM_SEG_GROUPS, SPLIT).total);
    if (e == cudaSuccess && SPLIT) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) {
      set_error("moe_mma_kernel: %s", cudaGetErrorString(e));
      return IM_CUDA_ERROR;
    }
    configured = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas_x, SPLIT ? (unsigned)a.segs : 1u, (unsigned)items);
  cfg.blockDim = dim3(MM_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (launch_overlap()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    n++;
  }
  if (SPLIT) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = 1;
    attr[n].val.clusterDim.y = (unsigned)a.segs;
    attr[n].val.clusterDim.z = 1;
    n++;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e != cudaSuccess) {
    set_error("moe_mma_kernel: %s", cudaGetErrorString(e));
    return IM_CUDA_ERROR;
  }
  return IM_OK;
}

template <int NT>
static int mm_pick(const MmArgs& a, bool glu, bool split, int ctas_x, int64_t items, cudaStream_t st) {
  if (glu)
    return split ? mm_launch<NT, true, true>(a, ctas_x, items, st) : mm_launch<NT, true, false>(a, ctas_x, items, st);
  return split ? mm_launch<NT, false, true>(a, ctas_x, items, st) : mm_launch<NT, false, false>(a, ctas_x, items, st);
}

int moe_mma_launch(const MoePlan& p, const MoeProduct& prod, cudaStream_t st) {
  MmArgs a = {};
  a.p = prod;
  a.items = reinterpret_cast<const int4*>(prod.plan + MOE_PLAN_HEADER);
  const int G = prod.K / 64;
  a.tiles = (prod.N + 31) / 32;
  const int ctas_x = (a.tiles + MM_WARPS - 1) / MM_WARPS;
  a.expert_bytes = (size_t)ctas_x * G * MOE_BLOCK_BYTES;
  a.segs = mm_segments(ctas_x, G);
  a.rg = (G + a.segs - 1) / a.segs;
  // one segment per CTA while the grid still fits one wave of CTAs; beyond, a CTA walks its item's segments
  const bool split = a.segs > 1 && a.segs <= MM_MAX_CLUSTER && (int64_t)ctas_x * p.max_items <= MM_WAVE;
  const bool glu = prod.epilogue != IM_EPI_STORE;
  IM_REQUIRE(p.max_items <= 65535, IM_UNSUPPORTED, "grouped product: %lld work items exceed 65535",
             (long long)p.max_items);
  switch (p.item_rows) {
    case 8: return mm_pick<1>(a, glu, split, ctas_x, p.max_items, st);
    case 16: return mm_pick<2>(a, glu, split, ctas_x, p.max_items, st);
    default: return mm_pick<4>(a, glu, split, ctas_x, p.max_items, st);
  }
}

}  // namespace im
