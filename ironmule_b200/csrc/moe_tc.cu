// Products by expert on the 5th-generation tensor cores: y[p] = W[e(p)] x[.] over packed 4-bit weights.
//
// D[128 outputs, N rows] = A[128, K] B[N, K]^T per tile: A is a 128-output block of one expert, B up to 128 gathered
// rows of it (one work item). Operands are fp16, accumulators float32 in tensor memory.
//
// Why fp16: w = scale * q + bias needs one rounding to become an operand. In bf16 (8 bits) that costs as much as the
// output's own rounding; in fp16 (11 bits) it is an eighth of it. The range is met by powers of two, which are exact:
//  * a weight row is scaled by its largest |w| (found when it is packed), which lands in [2^-7, 2^-6): then a code in
//    the low bits of a half IS the subnormal q 2^-24 (or 16 q 2^-24), and one fused multiply-add with scale * 2^24
//    (2^20) makes the weight. What this range costs is below 2^-18 of the row's largest weight;
//  * a row of x by its largest finite element, which lands in [2^9, 2^10) (moe_prep_kernel; bf16 values fit fp16);
//  * the gated activations h = act(g) u by a bound on the row: |g| <= |x|_2 max |G_r|_2 over the rows of G (found when it
//    is packed), |u| likewise, so |h| <= |x|_2^2 max|G_r| max|U_r|, which lands below 2^15. No finite row can overflow.
//    The bound is loose by K or so (2^11 of fp16's normal range of 2^29 at K = 2048), by the square of what a few large
//    elements of x add to |x|_2, and by what the largest rows of G and U exceed the others: activations that lie 2^-40
//    below the bound are rounded as subnormals, and lost below that. Where G or U is zero throughout, so is h, and u and
//    g are left as they are.
// The factors return in float32 after the sum. A row with infinities or NaN gives those.
//
// A persistent grid (one CTA per SM) walks tiles; its warps are coupled by mbarriers only:
//  * warp 0 copies the packed weights, two 64-wide groups (9216 contiguous bytes) at a time, into a ring of 8 (one
//    warp starts a copy every 200 to 300 cycles, whatever its size: hence two groups a stage everywhere);
//  * warps 12-27, four sets of 4, expand a stage each: thread = output row, 64 codes -> 32 registers of fp16 pairs ->
//    tensor memory, where the MMA reads A directly. Neither shared memory nor its bandwidth carries expanded weights;
//  * warp 10 copies the item's rows of a stage, one contiguous copy: moe_prep_kernel lays each item's rows out as the
//    K-major 128-byte-swizzled tiles that the MMA reads, and the gated epilogue writes its outputs as the next
//    product's tiles. (Gathering here was measured: TMA gather4 of 128-byte rows takes 64 cycles a row quadruple, and
//    16-byte asynchronous copies occupied four warps and the load pipe; a prefill took 1407 and 527 us.) The k order
//    within 8 follows the code expansion (k, k + 4 adjacent);
//  * warp 1 issues 8 MMAs of K = 16 a stage into one of two 128-column accumulators;
//  * warp 11 looks a tile up ahead of the others: its item, its weight rows' factors, its columns' factors and output
//    rows, into a ring of 3 in shared memory (looked up by every warp for itself, two dependent trips to L2 stood at
//    the head of every tile: 132 us against 120 for a prefill's second product);
//  * warps 2-9, two sets of 4 for alternate 32 columns, read a finished accumulator (lane = output), scale it, apply
//    the gate, and store.
// Every column (row of x) is its own sum in K order, so a row's bits do not depend on the other rows.
//
// Measured, 128 experts of 2048 x 768, 8 a row: 4096 rows, 165 us for gate and up (1.25 PFLOP/s, tensor pipe 72% active,
// the clock at 1.54 GHz under the power limit) and 120 us for down (0.86); 160 rows, 54 and 37 us (4.1 and 3.1 TB/s of
// weights). No one role bounds it: without the expansion's arithmetic, three in four MMAs or the epilogue, 160 rows took
// 7, 4 and 4% less. What small tiles wait for is the round trip through the barriers (150 to 200 cycles a hop, three
// hops a stage). Tried and left out, no faster: stages of four groups; an item's rows resident for the whole tile;
// separate barriers for a stage's halves; five B stages against a weight ring of four.
//
// Every mbarrier wait is bounded (1 s, or im_set_wait_limit): one that runs out sets the plan's error word (and the
// caller's) and the CTA's abort flag, which every later wait that is not over at once honours. A role that gives up leaves its loop without
// touching tensor memory again; copies and MMAs in flight are drained before tensor memory is freed.
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"
#include "moe.cuh"
#include "tc.cuh"
#include "../../include/imspec.h"

namespace im {

constexpr int MT_N = MOE_ITEM_ROWS;     // rows of an item at most (MMA N)
constexpr int MT_S = 4;                 // A and B stages of two groups (128 of K)
constexpr int MT_W = 8;                 // weight ring, two groups each
constexpr int MT_I = 3;                 // tiles looked up ahead
constexpr int MT_B = 2 * MT_N * 128;    // bytes of a B stage
constexpr int MT_EPI = 8;               // epilogue warps
constexpr int MT_SETS = 4;              // expansion sets of four warps
constexpr int MT_W_EPI = 2, MT_W_LOAD = MT_W_EPI + MT_EPI, MT_W_TRANS = MT_W_LOAD + 2;  // first warps of the roles
constexpr int MT_THREADS = (MT_W_TRANS + 4 * MT_SETS) * 32;
// A set has its own A stage and its own slots of the weight ring: a slot that two sets take in turn would let one of
// them take the completion of its last use for that of the next (a wait knows only a phase's parity).
static_assert(MT_S == MT_SETS && MT_W % MT_SETS == 0, "ring lengths");
constexpr int MT_WBITS = -6;            // a weight row's largest lands in [2^-7, 2^-6)
constexpr uint32_t MT_TMEM = 512;       // 2 accumulators of 128 columns, 4 A stages of 64
constexpr int MT_A0 = 256;
constexpr size_t MT_OFF_W = (size_t)MT_S * MT_B;
constexpr size_t MT_OFF_BAR = MT_OFF_W + (size_t)MT_W * 2 * MOE_BLOCK_BYTES;
// barriers: a stage's MMAs completed; a stage's A and B in place; weight ring; accumulators
constexpr int MT_DONE = 0, MT_FULL = MT_DONE + MT_S, MT_W_FULL = MT_FULL + MT_S, MT_W_EMPTY = MT_W_FULL + MT_W,
              MT_D_FULL = MT_W_EMPTY + MT_W, MT_D_EMPTY = MT_D_FULL + 2, MT_I_FULL = MT_D_EMPTY + 2,
              MT_C_FULL = MT_I_FULL + MT_I, MT_I_EMPTY = MT_C_FULL + MT_I, MT_BARS = MT_I_EMPTY + MT_I;
// What the roles need to know of a tile.
struct MtTile {
  int4 item;
  float inv[128], wscale[128];  // the weight rows' factors: to the operands' range, and back
  float2 col[128];              // the columns' factors: of the gate and of the up input; or the factor and the output row
};
constexpr size_t MT_OFF_TILE = (MT_OFF_BAR + MT_BARS * 8 + 16 + 15) / 16 * 16;
constexpr size_t MT_SMEM = 1024 + MT_OFF_TILE + MT_I * sizeof(MtTile);
constexpr int MT_READERS = 3 + MT_EPI + 4 * MT_SETS;  // warps that read a tile's entry

struct TcArgs {
  MoeProduct p;
  const int4* items;
  unsigned* error;
  const unsigned char* tiles;  // the items' rows as tiles
  const float* scale;    // per padded row: the factor it was divided by
  const float* xlog;     // per padded row: log2 |x|_2 (first product of a gated MLP)
  unsigned char* next;   // the next product's tiles, and its rows' factors (written by the first product)
  float* hscale;
  const float* row_max;  // [E][128 cols]: a weight row's largest |w|
  const float* norm_max; // [E][2]: the largest 2-norm of an expert's gate rows (r & 16 == 0) and of its up rows
  size_t expert_bytes;
  int cols;              // 128-output blocks
  unsigned long long wait_ns;
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

// The exponent that gated activations are divided by, from the logarithms of the bounds on |g| and |u| and the row's own
// factor: their product lands below 2^15, and neither u nor the factor that u takes on overflows on the way (g may be
// tiny where u is large). 0 where g or u is zero throughout.
__device__ __forceinline__ int mt_hidden_exp(float g, float u, float factor) {
  if (!(g > -INFINITY) || !(u > -INFINITY)) return 0;
  const int least = max(max((int)ceilf(u), ilogbf(factor)) - 120, -110);
  return min(max((int)ceilf(g + u) - 15, least), 120);
}

// Position of element k (0..7) of 8 in the operands' order.
__device__ __forceinline__ int mt_perm(int k) { return k < 4 ? 2 * k : 2 * (k - 4) + 1; }

// An item's rows as tiles: per 64-wide group, its rows (rounded up to 16) of 128 bytes; 16-byte chunk c of row r at
// c ^ r % 8. Items lie one after another from their padded first row on.
__device__ __forceinline__ size_t mt_tile(int padded, int n16, int K, int group) {
  return (size_t)padded * K * 2 + (size_t)group * n16 * 128;
}
__device__ __forceinline__ uint32_t mt_chunk(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }

// ---- rows of x -> scaled fp16 tiles: a CTA per row, which it reads once and writes to the tiles of every expert that
// its token chose (per_row = top_k; 1 when x has a row per pair) ------------------------------------------------------
constexpr int MP_THREADS = 128;
__global__ void __launch_bounds__(MP_THREADS)
moe_prep_kernel(const uint16_t* __restrict__ x, const int2* __restrict__ where, int per_row, int K,
                unsigned char* __restrict__ tiles, float* __restrict__ scale, float* __restrict__ xlog) {
  __shared__ float sh[2][MP_THREADS / 32];
  __shared__ int2 to[MOE_MAX_TOP_K];
  pdl_wait();
  pdl_trigger();
  const size_t row = blockIdx.x;
  if ((int)threadIdx.x < per_row) to[threadIdx.x] = where[row * per_row + threadIdx.x];
  const uint4* src = reinterpret_cast<const uint4*>(x + row * K);
  const int n = K / 8;
  float top = 0.f;
#pragma unroll 2
  for (int i = threadIdx.x; i < n; i += MP_THREADS) {
    const uint4 u = __ldg(src + i);
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
  for (int w = 0; w < MP_THREADS / 32; w++) top = fmaxf(top, sh[0][w]);
  const int e = mt_exp(top, 10);
  const float inv = mt_pow2(-e);
  float ss = 0.f;
#pragma unroll 2
  for (int i = threadIdx.x; i < n; i += MP_THREADS) {
    const uint4 u = __ldg(src + i);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    float f[8];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      f[2 * j] = bf_lo(w[j]) * inv;
      f[2 * j + 1] = bf_hi(w[j]) * inv;
    }
    uint32_t h[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if (fabsf(f[j]) < INFINITY) ss = fmaf(f[j], f[j], ss);
      if (fabsf(f[j + 4]) < INFINITY) ss = fmaf(f[j + 4], f[j + 4], ss);
      const __half2 v = __floats2half2_rn(f[j], f[j + 4]);
      h[j] = *reinterpret_cast<const uint32_t*>(&v);
    }
    for (int j = 0; j < per_row; j++) {
      const int2 t = to[j];
      if (t.x >= 0)
        *reinterpret_cast<uint4*>(tiles + mt_tile(t.x, t.y >> 16, K, i >> 3) + mt_chunk(t.y & 0xffff, i & 7)) =
            make_uint4(h[0], h[1], h[2], h[3]);
    }
  }
  ss = warp_sum(ss);
  if ((threadIdx.x & 31) == 0) sh[1][threadIdx.x >> 5] = ss;
  __syncthreads();
  if ((int)threadIdx.x < per_row && to[threadIdx.x].x >= 0) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < MP_THREADS / 32; w++) t += sh[1][w];
    const int at = to[threadIdx.x].x + (to[threadIdx.x].y & 0xffff);
    scale[at] = mt_pow2(e);
    xlog[at] = 0.5f * log2f(t) + (float)e;  // -inf for a zero row
  }
}

// ---- the products ----------------------------------------------------------------------------------------------
// fp16 pairs (k, k + 4) of a word's eight codes: the code as a subnormal, times scale * 2^24 (low nibble of a byte) or
// scale * 2^20 (high nibble), plus the bias, one rounding.
__device__ __forceinline__ void mt_expand(uint32_t u, __half2 s24, __half2 s20, __half2 b, uint32_t* out) {
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const uint32_t v = u >> (8 * i);
    const uint32_t lo = v & 0x000F000Fu, hi = v & 0x00F000F0u;
    const __half2 wl = __hfma2(*reinterpret_cast<const __half2*>(&lo), s24, b);
    const __half2 wh = __hfma2(*reinterpret_cast<const __half2*>(&hi), s20, b);
    out[2 * i] = *reinterpret_cast<const uint32_t*>(&wl);
    out[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&wh);
  }
}

// act(g) * u. Both gates are g times a sigmoid: of g, or (gelu by tanh: 0.5 (1 + tanh t) = sigmoid(2 t)) of 2 t.
template <int EPI>
__device__ __forceinline__ float mt_gated(float g, float u) {
  const float t = EPI == IM_EPI_GEGLU ? 1.5957691216057308f * (g + 0.044715f * g * g * g) : g;
  return __fdividef(g, 1.0f + __expf(-t)) * u;
}

__device__ __forceinline__ void mt_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// `bytes` from src into shared memory, counted on (and arriving once at) the barrier.
__device__ __forceinline__ void mt_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

__device__ __forceinline__ void mt_mma(uint32_t d, uint32_t ta, uint64_t bd, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(ta), "l"(bd), "r"(idesc), "r"((uint32_t)add));
}

__device__ __forceinline__ void mt_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// One row's 64 codes of a group -> 32 fp16 pairs -> columns [col, + 32) of tensor memory, once ready() says so (the
// whole warp's answer, which is passed on).
template <typename F>
__device__ __forceinline__ bool mt_group(const unsigned char* codes, const unsigned char* affine, float inv, int q,
                                         uint32_t col, F ready) {
  const uint4 c0 = *reinterpret_cast<const uint4*>(codes), c1 = *reinterpret_cast<const uint4*>(codes + 512);
  const float sf = bf(*reinterpret_cast<const uint16_t*>(affine)) * inv;
  const __half2 s24 = __float2half2_rn(sf * 16777216.f), s20 = __float2half2_rn(sf * 1048576.f);
  const __half2 b2 = __float2half2_rn(bf(*reinterpret_cast<const uint16_t*>(affine + 8)) * inv);
  uint32_t p[32];
  const uint32_t words[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
#pragma unroll
  for (int i = 0; i < 8; i++) mt_expand(words[i], s24, s20, b2, p + 4 * i);
  if (!ready()) return false;
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
      "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(((uint32_t)(32 * q) << 16) + col),
      "r"(p[0]), "r"(p[1]), "r"(p[2]), "r"(p[3]), "r"(p[4]), "r"(p[5]), "r"(p[6]), "r"(p[7]), "r"(p[8]), "r"(p[9]),
      "r"(p[10]), "r"(p[11]), "r"(p[12]), "r"(p[13]), "r"(p[14]), "r"(p[15]), "r"(p[16]), "r"(p[17]), "r"(p[18]),
      "r"(p[19]), "r"(p[20]), "r"(p[21]), "r"(p[22]), "r"(p[23]), "r"(p[24]), "r"(p[25]), "r"(p[26]), "r"(p[27]),
      "r"(p[28]), "r"(p[29]), "r"(p[30]), "r"(p[31])
      : "memory");
  return true;
}

template <int EPI>
__global__ void __launch_bounds__(MT_THREADS, 1) moe_tc_kernel(TcArgs a) {
  constexpr bool GLU = EPI != IM_EPI_STORE;
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
      qt_init(&b[MT_FULL + s], 4u + 1u);  // four expansion warps, the rows' bytes
    }
    for (int s = 0; s < MT_W; s++) {
      qt_init(&b[MT_W_FULL + s], 1u);
      qt_init(&b[MT_W_EMPTY + s], 4u);
    }
    for (int s = 0; s < 2; s++) {
      qt_init(&b[MT_D_FULL + s], 1u);
      qt_init(&b[MT_D_EMPTY + s], MT_EPI);
    }
    for (int s = 0; s < MT_I; s++) {
      qt_init(&b[MT_I_FULL + s], 1u);
      qt_init(&b[MT_C_FULL + s], 1u);
      qt_init(&b[MT_I_EMPTY + s], MT_READERS);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  constexpr uint32_t tmem = 0;  // the whole tensor memory: its allocation can only start at column 0
  // The routing's plan was finished before the launch that precedes this one (the prep kernel, or the first product)
  // let this one begin: the plan and the weights are read without waiting (from L2, whatever an SM's L1 may hold of
  // them), rows and outputs only after pdl_wait().
  const int ntiles = __ldcg(a.p.plan) * a.cols;
  MtTile* const info = reinterpret_cast<MtTile*>(sbase + MT_OFF_TILE);
  uint32_t islot = 0, iphase = 0;  // this warp's place in the ring of tiles
  auto tile_wait = [&] { return qt_wait_short(bars + 8 * (MT_I_FULL + islot), iphase, abort_flag, a.error, a.wait_ns); };
  auto tile_free = [&] {  // this warp has read what it needs
    __syncwarp();
    if (lane == 0) mt_arrive(bars + 8 * (MT_I_EMPTY + islot));
    if (++islot == MT_I) islot = 0, iphase ^= 1u;
  };

  if (warp == 0) {
    // ---- weights -------------------------------------------------------------------------------------------
    // (as for the MMAs, the whole warp walks the loop and one lane issues)
    const bool leader = qt_elect();
    uint32_t s = 0, phase = 1;
    int k = 0;
    for (int tile = blockIdx.x; tile < ntiles; tile += gridDim.x) {
      if (!tile_wait()) goto weights_done;
      const int expert = info[islot].item.x;
      tile_free();
      if (expert == a.p.E) continue;
      const unsigned char* src =
          a.p.wp + (size_t)expert * a.expert_bytes + (size_t)(tile % a.cols) * G * MOE_BLOCK_BYTES;
      for (int g = 0; g < G; g += 2, k++) {
        if (!qt_wait_short(bars + 8 * (MT_W_EMPTY + s), phase, abort_flag, a.error, a.wait_ns)) goto weights_done;
        if (leader)
          mt_copy(base + (uint32_t)MT_OFF_W + s * 2 * MOE_BLOCK_BYTES, src, g + 1 < G ? 2 * MOE_BLOCK_BYTES : MOE_BLOCK_BYTES,
                  bars + 8 * (MT_W_FULL + s));
        __syncwarp();
        src += 2 * MOE_BLOCK_BYTES;
        if (++s == MT_W) s = 0, phase ^= 1u;
      }
    }
  weights_done:
    // copies still landing in this CTA's shared memory finish before it exits (in every case: another role may give up
    // after this one has issued its last)
    for (int j = k > MT_W ? k - MT_W : 0; j < k; j++)
      qt_drain(reinterpret_cast<unsigned long long*>(sbase + MT_OFF_BAR) + MT_W_FULL + j % MT_W,
               (uint32_t)((j / MT_W) & 1));
  } else if (warp == 1) {
    // ---- MMA issue -----------------------------------------------------------------------------------------
    // (the whole warp walks the loop, so that its addresses stay in uniform registers; one lane issues)
    const bool leader = qt_elect();
    uint32_t s = 0, phase = 0;
    int k = 0, t = 0;
    for (int tile = blockIdx.x; tile < ntiles; tile += gridDim.x) {
      if (!tile_wait()) break;
      const int4 item = info[islot].item;
      tile_free();
      if (item.x == a.p.E) continue;
      // f32 accumulate, f16 A and B, K-major, N = the item's rows in sixteens, M = 128
      const uint32_t idesc = (1u << 4) | ((uint32_t)((item.z + 15) / 16 * 2) << 17) | ((128u >> 4) << 24);
      const uint32_t tile_step = (uint32_t)((item.z + 15) / 16 * 128);  // (16 bytes units) to the second group's rows
      const int buf = t & 1;
      if (!qt_wait_short(bars + 8 * (MT_D_EMPTY + buf), (uint32_t)((t / 2 + 1) & 1), abort_flag, a.error, a.wait_ns)) break;
      const uint32_t d = tmem + (uint32_t)(buf * MT_N);
      int g = 0;
      for (; g < G; g += 2, k++) {
        if (!qt_wait_short(bars + 8 * (MT_FULL + s), phase, abort_flag, a.error, a.wait_ns)) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (leader) {
          const uint64_t bd = qt_desc(base + s * MT_B), bd1 = bd + tile_step;
          const uint32_t ta = tmem + MT_A0 + 64 * s;
#pragma unroll
          for (int q = 0; q < 4; q++) mt_mma(d, ta + 8 * q, bd + 2 * q, idesc, g + q > 0);
          if (g + 1 < G) {
#pragma unroll
            for (int q = 0; q < 4; q++) mt_mma(d, ta + 32 + 8 * q, bd1 + 2 * q, idesc, true);
          }
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
    // so do the MMAs, before tensor memory is freed, and the arrivals that follow them
    unsigned long long* const b = reinterpret_cast<unsigned long long*>(sbase + MT_OFF_BAR);
    for (int j = k > MT_S ? k - MT_S : 0; j < k; j++) qt_drain(b + MT_DONE + j % MT_S, (uint32_t)((j / MT_S) & 1));
    for (int j = t > 2 ? t - 2 : 0; j < t; j++) qt_drain(b + MT_D_FULL + (j & 1), (uint32_t)((j / 2) & 1));
  } else if (warp < MT_W_LOAD) {
    // ---- epilogue: lane = output of the block, columns = the item's rows ---------------------------------------
    const int q = warp & 3, set = (warp - MT_W_EPI) >> 2;
    const bool paired = (nout & 1) == 0 && (reinterpret_cast<uintptr_t>(a.p.y) & 3) == 0;
    pdl_wait();
    pdl_trigger();
    int t = 0;
    for (int tile = blockIdx.x; tile < ntiles; tile += gridDim.x) {
      if (!tile_wait() || !qt_wait_short(bars + 8 * (MT_C_FULL + islot), iphase, abort_flag, a.error, a.wait_ns)) break;
      const int4 item = info[islot].item;
      const float wscale = info[islot].wscale[q * 32 + lane];
      const float2* meta = info[islot].col;
      const int col = tile % a.cols, rows = item.z;
      if (item.x == a.p.E) {  // places without an expert: zeros
        if (!GLU) {
          const int f = col * 128 + q * 32 + lane;
          for (int j = set; j < rows; j += 2)
            if (f < nout) a.p.y[(size_t)a.p.pairs[item.y + j] * nout + f] = 0;
        }
        tile_free();
        continue;
      }
      const int buf = t & 1;
      if (!qt_wait_short(bars + 8 * (MT_D_FULL + buf), (uint32_t)((t / 2) & 1), abort_flag, a.error, a.wait_ns)) break;
      t++;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
      for (int i = 0; 64 * i + 32 * set < rows; i++) {
        const int c0 = 64 * i + 32 * set, n = min(32, rows - c0);
        uint32_t v[32];
        const uint32_t ta = ((uint32_t)(32 * q) << 16) + (uint32_t)(buf * MT_N + c0);
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
            "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
            : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
              "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
              "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
              "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
            : "r"(ta));
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        // Of two columns j, j + 1 each lane finishes one, with its partner lane's value of it (the partner: the other
        // half of a gated output, or the neighbouring output, so that two outputs leave in one store).
        const int other = GLU ? 16 : 1, second = (lane & other) != 0;
        const float2* m = meta + c0 + second;
        if constexpr (GLU) {
          // The next product's tiles: group f / 64, chunk f % 64 / 8, the element's place in the operand order; rows up
          // to the next sixteen exist there and are written too. Row c0 + j + second swizzles with (j + second) % 8,
          // so four pointers serve every j.
          const int f = (col * 4 + q) * 16 + (lane & 15), n16 = (rows + 15) & ~15, chunk = (f & 63) >> 3;
          unsigned char* h = a.next + mt_tile(item.w, n16, nout, f >> 6) + 2 * mt_perm(f & 7) + (c0 + second) * 128;
          unsigned char* at[4];
#pragma unroll
          for (int w = 0; w < 4; w++) at[w] = h + ((chunk ^ (2 * w + second)) << 4);
#pragma unroll
          for (int half = 0; half < 2; half++) {
            if (c0 + 16 * half >= n16) break;
#pragma unroll
            for (int j = 16 * half; j < 16 * half + 16; j += 2) {
              const float give = __uint_as_float(second ? v[j] : v[j + 1]) * wscale;
              const float keep = __uint_as_float(second ? v[j + 1] : v[j]) * wscale;
              const float got = __shfl_xor_sync(0xffffffffu, give, 16);
              const float2 mj = m[j];
              // lanes 0-15 hold gate features, 16-31 the matching up features
              const float g = (second ? got : keep) * mj.x, u = (second ? keep : got) * mj.y;
              *reinterpret_cast<__half*>(at[j / 2 % 4] + j * 128) = __float2half_rn(mt_gated<EPI>(g, u));
            }
          }
        } else {
          const int f = col * 128 + q * 32 + lane;
          uint16_t* y = a.p.y + (f & ~1);
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float give = __uint_as_float(second ? v[j] : v[j + 1]) * wscale;
            const float keep = __uint_as_float(second ? v[j + 1] : v[j]) * wscale;
            const float got = __shfl_xor_sync(0xffffffffu, give, 1);
            const float2 mj = m[j];
            const float k1 = keep * mj.x, g1 = got * mj.x;
            uint32_t o;
            asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(o) : "f"(second ? k1 : g1), "f"(second ? g1 : k1));
            if (j + second < n && (f & ~1) < nout) {
              uint16_t* to = y + (size_t)__float_as_int(mj.y) * nout;
              if (paired) {
                *reinterpret_cast<uint32_t*>(to) = o;
              } else {
                to[0] = (uint16_t)o;
                if ((f | 1) < nout) to[1] = (uint16_t)(o >> 16);
              }
            }
          }
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mt_arrive(bars + 8 * (MT_D_EMPTY + buf));
      tile_free();
    }
  } else if (warp < MT_W_TRANS) {
    if (warp == MT_W_LOAD + 1) {
      // ---- the tiles, ahead of the other warps -----------------------------------------------------------------------
      const int step = gridDim.x;
      int4 item = (int)blockIdx.x < ntiles ? __ldcg(a.items + blockIdx.x / a.cols) : make_int4(0, 0, 0, 0);
      bool waited = false;
      for (int tile = blockIdx.x; tile < ntiles; tile += step) {
        const int4 next = tile + step < ntiles ? __ldcg(a.items + (tile + step) / a.cols) : item;
        const bool closed = item.x == a.p.E;
        float top[4] = {};
        if (!closed) {
          const float* rm = a.row_max + ((size_t)item.x * a.cols + tile % a.cols) * 128 + lane;
#pragma unroll
          for (int i = 0; i < 4; i++) top[i] = __ldcg(rm + 32 * i);
        }
        if (!qt_wait_short(bars + 8 * (MT_I_EMPTY + islot), iphase ^ 1u, abort_flag, a.error, a.wait_ns)) break;
        MtTile& out = info[islot];
        if (lane == 0) out.item = item;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int e = mt_exp(top[i], MT_WBITS);
          out.inv[32 * i + lane] = mt_pow2(-e);
          out.wscale[32 * i + lane] = mt_pow2(e);
        }
        __syncwarp();
        if (lane == 0) mt_arrive(bars + 8 * (MT_I_FULL + islot));
        if (!waited) {
          pdl_wait();
          waited = true;
        }
        if (!closed) {
          float lg = 0.f, lu = 0.f;  // what bounds g and u of a row of |x|_2 = 1
          if constexpr (GLU) {
            lg = log2f(a.norm_max[2 * item.x]);
            lu = log2f(a.norm_max[2 * item.x + 1]);
          }
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int c = 32 * i + lane, row = item.w + c;
            if (c < item.z) {
              float2 m = make_float2(a.scale[row], 0.f);
              if constexpr (GLU) {
                const int e = mt_hidden_exp(a.xlog[row] + lg, a.xlog[row] + lu, m.x);
                m.y = m.x * mt_pow2(-e);
                if (tile % a.cols == 0) a.hscale[row] = mt_pow2(e);
              } else {
                m.y = __int_as_float(a.p.pairs[item.y + c]);
              }
              out.col[c] = m;
            }
          }
        }
        __syncwarp();
        if (lane == 0) mt_arrive(bars + 8 * (MT_C_FULL + islot));
        if (++islot == MT_I) islot = 0, iphase ^= 1u;
        item = next;
      }
    }
    // ---- rows ----------------------------------------------------------------------------------------------------
    if (warp == MT_W_LOAD) {
      const bool leader = qt_elect();
      pdl_wait();
      uint32_t s = 0, phase = 1;
      int k = 0;
      for (int tile = blockIdx.x; tile < ntiles; tile += gridDim.x) {
        if (!tile_wait()) goto rows_done;
        const int4 item = info[islot].item;
        tile_free();
        if (item.x == a.p.E) continue;
        const uint32_t bytes = (uint32_t)((item.z + 15) & ~15) * 128u;
        const unsigned char* src = a.tiles + (size_t)item.w * a.p.K * 2;
        for (int g = 0; g < G; g += 2, k++) {
          if (!qt_wait_short(bars + 8 * (MT_DONE + s), phase, abort_flag, a.error, a.wait_ns)) goto rows_done;
          if (leader) mt_copy(base + s * MT_B, src, g + 1 < G ? 2 * bytes : bytes, bars + 8 * (MT_FULL + s));
          __syncwarp();
          src += 2 * bytes;
          if (++s == MT_S) s = 0, phase ^= 1u;
        }
      }
    rows_done:
      // as for the weights (a second a stage is ample, and the limit where the expansion's arrivals never come)
      for (int j = k > MT_S ? k - MT_S : 0; j < k; j++)
        qt_drain(reinterpret_cast<unsigned long long*>(sbase + MT_OFF_BAR) + MT_FULL + j % MT_S,
                 (uint32_t)((j / MT_S) & 1));
    }
  } else {
    // ---- code expansion: set i takes every fourth stage of the CTA's sequence, from stage i on -----------------------
    const int set = (warp - MT_W_TRANS) >> 2, q = warp & 3;
    const unsigned char* codes = sbase + MT_OFF_W + q * 1024 + lane * 16;
    const unsigned char* affine = sbase + MT_OFF_W + 4096 + q * 128 + (lane & 7) * 16 + (lane >> 3) * 2;
    uint32_t phase = 1, sw = set, wphase = 0;
    int skip = 2 * set;  // groups of the next tile that lie before this set's next stage
    const int even = G + (G & 1);
    for (int tile = blockIdx.x; tile < ntiles; tile += gridDim.x) {
      if (!tile_wait()) goto expand_done;
      const int expert = info[islot].item.x;
      const float inv = info[islot].inv[q * 32 + lane];
      tile_free();
      if (expert == a.p.E) continue;
      int g = skip;
      for (; g < G; g += 2 * MT_SETS) {
        if (!qt_wait_short(bars + 8 * (MT_W_FULL + sw), wphase, abort_flag, a.error, a.wait_ns)) goto expand_done;
        const uint32_t at = sw * 2 * MOE_BLOCK_BYTES;
        if (!mt_group(codes + at, affine + at, inv, q, MT_A0 + 64 * set, [&] {
              return qt_wait_short(bars + 8 * (MT_DONE + set), phase, abort_flag, a.error, a.wait_ns);
            }))
          goto expand_done;
        if (g + 1 < G)
          mt_group(codes + at + MOE_BLOCK_BYTES, affine + at + MOE_BLOCK_BYTES, inv, q, MT_A0 + 64 * set + 32,
                   [] { return true; });
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          mt_arrive(bars + 8 * (MT_W_EMPTY + sw));
          mt_arrive(bars + 8 * (MT_FULL + set));
        }
        if ((sw += MT_SETS) >= MT_W) sw -= MT_W, wphase ^= 1u;
        phase ^= 1u;
      }
      skip = g - even;
    }
  expand_done:;
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();  // every MMA of this CTA has completed (or been drained)
  if (threadIdx.x == 0 && *abort_flag) {
    int* const word = *reinterpret_cast<int* const*>(a.p.plan + 2);
    if (word) atomicExch(word, 1);
  }
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(MT_TMEM));
  }
}

// The products' workspace: the items' rows as tiles (each item rounded up to 16 rows), their factors, the
// same of the gated activations (I > 0).
MoeSpace moe_space(const MoePlan& p, int64_t pairs, int64_t K, int64_t I) {
  MoeSpace s;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t r = at;
    at += (bytes + 1023) / 1024 * 1024;
    return r;
  };
  const size_t padded = (size_t)(pairs + 15 * p.max_items);
  s.tiles = take(padded * K * 2);
  s.scale = take(padded * 4);
  s.xlog = take(padded * 4);
  s.next = take(padded * I * 2);
  s.hscale = take(I ? padded * 4 : 0);
  s.total = at;
  return s;
}

int moe_prep_launch(const MoePlan& p, const MoeProduct& a, const uint16_t* x, int by_pair, const MoeSpace& s,
                    void* workspace, cudaStream_t st) {
  char* ws = reinterpret_cast<char*>(workspace);
  const int64_t rows = by_pair ? (int64_t)a.M * a.top_k : a.M;
  return launch("moe_prep_kernel", moe_prep_kernel, dim3((unsigned)rows), dim3(MP_THREADS), 0, st, x,
                reinterpret_cast<const int2*>(a.plan + p.where), by_pair ? 1 : a.top_k, a.K,
                reinterpret_cast<unsigned char*>(ws + s.tiles), reinterpret_cast<float*>(ws + s.scale),
                reinterpret_cast<float*>(ws + s.xlog));
}

template <int EPI>
static int mt_launch(const TcArgs& a, int64_t tiles, cudaStream_t st) {
  static int per_device[64];  // SMs, once the kernel is configured there
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev < 0 || dev >= 64)) e = cudaErrorInvalidDevice;
  int sms = e == cudaSuccess ? per_device[dev] : 0;
  if (e == cudaSuccess && !sms) {
    e = cudaFuncSetAttribute(moe_tc_kernel<EPI>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)MT_SMEM);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess) per_device[dev] = sms;
  }
  if (e != cudaSuccess) {
    set_error("moe_tc_kernel: %s", cudaGetErrorString(e));
    return IM_CUDA_ERROR;
  }
  return launch("moe_tc_kernel", moe_tc_kernel<EPI>, dim3((unsigned)(tiles < sms ? tiles : sms)), dim3(MT_THREADS),
                MT_SMEM, st, a);
}

int moe_product_launch(const MoePlan& p, const MoeProduct& prod, const MoeSpace& s, void* workspace, cudaStream_t st) {
  char* ws = reinterpret_cast<char*>(workspace);
  TcArgs a = {};
  a.p = prod;
  a.items = reinterpret_cast<const int4*>(prod.plan + MOE_PLAN_HEADER);
  a.error = reinterpret_cast<unsigned*>(const_cast<int*>(prod.plan)) + 1;
  a.tiles = reinterpret_cast<const unsigned char*>(ws + (prod.second ? s.next : s.tiles));
  a.scale = reinterpret_cast<const float*>(ws + (prod.second ? s.hscale : s.scale));
  a.xlog = reinterpret_cast<const float*>(ws + s.xlog);
  a.next = reinterpret_cast<unsigned char*>(ws + s.next);
  a.hscale = reinterpret_cast<float*>(ws + s.hscale);
  const int G = prod.K / 64;
  a.cols = (prod.N + 127) / 128;
  a.expert_bytes = (size_t)a.cols * G * MOE_BLOCK_BYTES;
  a.row_max = reinterpret_cast<const float*>(prod.wp + (size_t)prod.E * a.expert_bytes);
  a.norm_max = a.row_max + (size_t)prod.E * a.cols * 128;
  a.wait_ns = wait_limit();
  const int64_t tiles = p.max_items * a.cols;
  IM_REQUIRE(tiles < (1ll << 31), IM_UNSUPPORTED, "grouped product: too many tiles");
  switch (prod.epilogue) {
    case IM_EPI_STORE: return mt_launch<IM_EPI_STORE>(a, tiles, st);
    case IM_EPI_SWIGLU: return mt_launch<IM_EPI_SWIGLU>(a, tiles, st);
    default: return mt_launch<IM_EPI_GEGLU>(a, tiles, st);
  }
}

}  // namespace im
