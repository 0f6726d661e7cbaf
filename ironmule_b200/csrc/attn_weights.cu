// Attention of a few new rows a sequence over the paged cache, which also adds up every slot's attention weight.
//
//   s[r, g, j] = scale q[r, g] . k[j] for the slots j that row r sees, p = softmax over j, out = sum_j p v[j]
//   weights'[h, j] = (j before the sequence's first new slot ? weights[h, j] : 0) + sum over rows r and the query heads
//   g of kv head h of p[r, g, j]
//
// Bound: HBM, K and V of every visible slot read once (2 * 2 D bytes a slot and kv head). One row of 32/8 heads of 128 over
// 131071 slots takes 99 us, 32 rows over 4096 to 8192 slots 150 us (the first kernel at 5.6 and 6.0 TB/s).
//
// First kernel (aw_split_kernel): a block takes one split of a (sequence, kv head) and a tile of its (row, query head)
// vectors. Its four warps (two, or two pairs, of wide heads) take the split's pages in turn, each with a ring of pages of its own in
// shared memory (asynchronous copies, no barrier between warps), a running maximum and sum and a D x vectors accumulator in
// registers; they are joined once at the split's end. The products are transposed, so that the few vectors are the warp MMA's n = 8
// (one or two of them) and slots and head values its m = 16: S^T = K Q^T, out^T = V^T P^T. With Q as the m = 16 rows, half
// and more of the products would be of rows that are not there, and at 16 cycles each they would take half of a
// page's time; tcgen05's tiles of 64 rows and more would add more of that. Scores go to the workspace in float32 (4 bytes
// a vector and slot beside 4 D of K and V): the weights need the final maximum and sum.
// Second kernel (aw_finish_kernel): joins the splits, and adds up exp2(s - max) / sum slot by slot.
// Calls of few and short splits are one kernel's (aw_split_kernel with ONE): the splits of a (sequence, kv head) are a
// cluster, scores stay in shared memory, and the blocks tell each other their maxima, sums and accumulators through
// distributed shared memory. One token over 2048 slots takes one launch and no workspace then.
//
// Weights that meet v are two numbers of the cache's type, high part and rest (16 bits and more of each weight are kept);
// in float16 they are scaled by 2^6 to 2^14 first, so that weights down to 2^-20 of the largest are not subnormal. Masked
// slots never reach a row: behind the last visible slot v is zeroed on its way in; between rows of one call a page is
// checked for values that are not finite, and if it has any its products are done one by one.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace im {

namespace cg = cooperative_groups;

constexpr int AW_FIN_THREADS = 256;
constexpr float AW_LOG2E = 1.4426950408889634f;
constexpr float AW_SLACK = 8.f;
constexpr int AW_CLUSTER = 16;             // splits of a call that one kernel does
constexpr int AW_HELD = 24 * 1024;         // and bytes of scores that its blocks hold

struct AwArgs {
  const char* q;
  const char* k;
  const char* v;
  const int* page_table;
  long long seqs, max_pages, pages;
  const int* seq_rows;
  const int* seq_slot;
  const int* row_slot;
  const float* weights;
  float* weights_out;
  long long cap;
  int M, max_rows, hq, hkv, d;
  int max_kv, kv_pad;
  int window;
  float scale;
  char* out;
  int kps, splits, tile, tiles;  // keys a split, splits of max_kv, vectors a tile, tiles
  int vecs;                // max_rows * Hq / Hkv
  float* scores;           // [B][Hkv][vecs][kv_pad], in log2 units
  float2* stats;           // [B][Hkv][splits][vecs]: maximum and sum
  float* parts;            // [B][Hkv][splits][vecs][d]
  int seen;                // splits that a sequence's rows see, if they follow one another: the first kernel's blocks
  int groups;              // threads of the second kernel that share four slots
  int joins, join_warps;   // blocks of the second kernel that join outputs, warps a job of theirs
  int wide_weights;        // weights and weights_out start on 16 bytes
};

// What a block knows of its sequence: first its rows and table row, then, from the rows' slots, what they see.
struct AwSeq {
  int row0, rows;       // its rows that the call computes
  long long slot;       // its page-table row (-1: none)
  int n, lo;            // visible slots lie in [lo, n)
};

__device__ __forceinline__ AwSeq aw_seq(const AwArgs& a, int b) {
  AwSeq s;
  s.row0 = min(max(a.seq_rows[b], 0), a.M);
  s.rows = max(0, min(min(a.seq_rows[b + 1], a.M) - s.row0, a.max_rows));
  s.slot = a.seq_slot ? a.seq_slot[b] : b;
  if (s.slot < 0 || s.slot >= a.seqs) s.slot = -1;
  return s;
}

// By a whole warp.
__device__ __forceinline__ void aw_span(const AwArgs& a, AwSeq& s) {
  int top = -1, low = 0x7fffffff;
  for (int r = threadIdx.x & 31; r < s.rows; r += 32) {
    const int at = a.row_slot[s.row0 + r];
    top = max(top, at);
    if (at >= 0) low = min(low, at);
  }
  top = __reduce_max_sync(0xffffffffu, top), low = __reduce_min_sync(0xffffffffu, low);
  const long long most = min((long long)a.max_kv, a.max_pages * 16);
  s.n = s.slot < 0 ? 0 : (int)min((long long)top + 1, most);
  s.lo = a.window > 0 && low != 0x7fffffff ? max(0, low - a.window + 1) : 0;
}

// The slot of the first row that has one: weights from it on start from zero.
__device__ __forceinline__ int aw_first(const AwArgs& a, const AwSeq& s) {
  int first = a.row_slot[s.row0];
  for (int r = 1; first < 0 && r < s.rows; r++) first = a.row_slot[s.row0 + r];  // padding before a sequence's rows
  return first;
}

// 2^x to two ulps; what would be subnormal is 0.
__device__ __forceinline__ float aw_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// L2 policy of K and V: read once where one block reads them (they leave room for the scores, which the second kernel
// reads back), kept where several tiles do.
__device__ __forceinline__ uint64_t aw_policy(bool once) {
  uint64_t p;
  if (once) asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  else asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ void aw_copy16(uint32_t dst, const char* src, bool in, uint64_t policy) {
  const int n = in ? 16 : 0;  // 0: zeros, nothing is read
  asm volatile("cp.async.cg.shared.global.L2::cache_hint.L2::128B [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(n),
               "l"(policy)
               : "memory");
}
__device__ __forceinline__ void aw_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void aw_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void aw_ldsm(uint32_t* r, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at));
}
// An 8 x 8 matrix of 16-bit values, two a lane, transposed.
__device__ __forceinline__ uint32_t aw_turn(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void aw_ldsm_t(uint32_t* r, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at));
}

template <typename T>
struct AwType;
template <>
struct AwType<__nv_bfloat16> {
  static constexpr float SHIFT = 0.f;
  static __device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  // two weights as (high parts, rests)
  static __device__ __forceinline__ uint2 parts(float x, float y) {
    const __nv_bfloat162 hi = __floats2bfloat162_rn(x, y);
    const __nv_bfloat162 lo = __floats2bfloat162_rn(x - __low2float(hi), y - __high2float(hi));
    return make_uint2(*(const uint32_t*)&hi, *(const uint32_t*)&lo);
  }
  static __device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ bool finite(uint32_t u) {
    return (u & 0x7f80u) != 0x7f80u && (u & 0x7f800000u) != 0x7f800000u;
  }
  static __device__ __forceinline__ __nv_bfloat16 down(float f) { return __float2bfloat16_rn(f); }
};
template <>
struct AwType<__half> {
  static constexpr float SHIFT = 6.f;  // with AW_SLACK, weights stay below 2^14
  static __device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint2 parts(float x, float y) {
    const __half2 hi = __floats2half2_rn(x, y);
    const __half2 lo = __floats2half2_rn(x - __low2float(hi), y - __high2float(hi));
    return make_uint2(*(const uint32_t*)&hi, *(const uint32_t*)&lo);
  }
  static __device__ __forceinline__ float up(__half v) { return __half2float(v); }
  static __device__ __forceinline__ bool finite(uint32_t u) {
    return (u & 0x7c00u) != 0x7c00u && (u & 0x7c000000u) != 0x7c000000u;
  }
  static __device__ __forceinline__ __half down(float f) { return __float2half_rn(f); }
};

// Adds a split's maximum and sum to (m, l). -inf and 0 are those of no visible slot; a sum of NaN (scores of NaN have no
// maximum: it may be -inf) stays one.
__device__ __forceinline__ void aw_add(float& m, float& l, float m2, float l2) {
  const float top = fmaxf(m, m2);
  l = top != -INFINITY ? l * aw_exp2(m - top) + l2 * aw_exp2(m2 - top) : l + l2;
  m = top;
}

// The total of a vector whose splits' maxima and sums lie in a warp's lanes (-inf and 0 where there is none): maximum and
// 1 / sum, in every lane.
__device__ __forceinline__ float2 aw_join(float m, float l) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), l2 = __shfl_xor_sync(0xffffffffu, l, o);
    aw_add(m, l, m2, l2);
  }
  return make_float2(m == -INFINITY ? 0.f : m, l == 0.f ? 0.f : 1.f / l);
}

// Four values of vector v's output.
template <typename T>
__device__ __forceinline__ void aw_store(const AwArgs& a, const AwSeq& q, int h, int group, int v, int c, const float4& o,
                                         float inv) {
  const long long row = q.row0 + v / group;
  alignas(8) T r[4] = {AwType<T>::down(o.x * inv), AwType<T>::down(o.y * inv), AwType<T>::down(o.z * inv),
                       AwType<T>::down(o.w * inv)};
  *(uint2*)((T*)a.out + (row * a.hq + h * group + v % group) * a.d + c) = *(const uint2*)r;
}

// DP: head_dim rounded up to what is built; columns from d on are zeros in shared memory. NT: tiles of 8 vectors a warp.
// WPP: warps that work on a page, each with its own vectors.
template <int DP, int NT, int WPP>
struct AwShape {
  static constexpr int TILE = NT * WPP * 8;   // vectors of a block
  static constexpr int RINGS = DP > 128 ? 2 : 4;
  static constexpr int WARPS = RINGS * WPP;
  static constexpr int PITCH = DP * 2 + 16;   // an odd number of 16-byte steps: ldmatrix without bank conflicts
  static constexpr int PAGE = 16 * PITCH;     // one page's K or V
  static constexpr int STAGES = DP > 64 ? 2 : 3;
  static constexpr int RING = STAGES * 2 * PAGE;
  static constexpr int JOIN = DP + 4;         // floats of a vector where the warps' accumulators are joined
  static_assert(NT * DP <= 384, "Q stays in registers");
  static constexpr int SMEM = RINGS * RING;
  static constexpr int SMEM_ONE = SMEM + TILE * JOIN * 4 + AW_HELD + TILE * 16;  // with accumulators and scores, padded
  static_assert(TILE * JOIN * 4 <= RING, "a ring takes its accumulator at the end");
  static constexpr int BLOCKS = WPP > 1 ? (DP > 128 ? 3 : 2) : NT > 2 ? 2 : DP > 64 ? 3 : 4;  // on an SM
};

template <typename T, int DP, int NT, int WPP, bool ONE>
__global__ void __launch_bounds__(AwShape<DP, NT, WPP>::WARPS * 32, AwShape<DP, NT, WPP>::BLOCKS)
    aw_split_kernel(AwArgs a) {
  using S = AwShape<DP, NT, WPP>;
  using Ty = AwType<T>;
  constexpr int TILE = S::TILE, WARPS = S::WARPS, RINGS = S::RINGS;
  extern __shared__ __align__(128) char smem[];
  __shared__ float s_m[RINGS][TILE], s_l[RINGS][TILE];
  // ONE: this block's maxima and sums, the whole cluster's, the final ones
  __shared__ float2 s_stat[ONE ? TILE : 1], s_all[ONE ? AW_CLUSTER : 1][ONE ? TILE : 1], s_total[ONE ? TILE : 1];
  __shared__ int2 s_sees[ONE ? TILE : 1];  // ONE: the slots that a vector sees, [x, y]
  float* s_out = (float*)(smem + S::SMEM);  // ONE: [TILE][JOIN]
  float* s_scores = s_out + TILE * S::JOIN;  // ONE: [TILE][kps + 4]
  const int held = a.kps + 4;
  pdl_wait();
  pdl_trigger();
  int split = blockIdx.x;  // of two kernels' with a window: counted from the first that a row sees
  const int h = blockIdx.y / a.tiles, tile = blockIdx.y % a.tiles, b = blockIdx.z;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int worker = warp / WPP, part = warp % WPP;  // which pages, which vectors
  constexpr int STEPS = DP / 16, CP = DP / 8;
  AwSeq q = aw_seq(a, b);
  const int group = a.hq / a.hkv;
  const int vecs = q.rows * group;  // live ones
  if (tile * TILE >= vecs || (!ONE && q.slot < 0)) return;  // the whole cluster
  const int* table = a.page_table + max(q.slot, 0ll) * a.max_pages;
  // pages of this warp: those whose number is its worker's mod RINGS, so that a slot's place does not depend on the call. The page
  // numbers are fetched a round ahead of the copies that need them, the first before it is known how many there are
  int next = split * a.kps / 16;
  next += (worker - next) & (RINGS - 1);
  int entry = a.window == 0 && q.slot >= 0 && next < a.max_pages ? table[next] : 0;
  // this lane's vectors of each tile of 8: 2 (lane mod 4) and the next (accumulators), lane / 4 (Q as an operand)
  int last[NT][2], from[NT][2];
  bool live[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; nt++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int vec = tile * TILE + (part * NT + nt) * 8 + lane % 4 * 2 + e;
      live[nt][e] = vec < vecs;
      last[nt][e] = live[nt][e] ? a.row_slot[q.row0 + vec / group] : -1;
    }
  uint32_t qf[STEPS][NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    const int vec = tile * TILE + (part * NT + nt) * 8 + lane / 4;
    const char* p = a.q + (((long long)q.row0 + vec / group) * a.hq + h * group + vec % group) * a.d * 2;
#pragma unroll
    for (int st = 0; st < STEPS; st++)
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const int c = st * 16 + i * 8 + lane % 4 * 2;
        qf[st][nt][i] = vec < vecs && c < a.d ? *(const uint32_t*)(p + c * 2) : 0u;
      }
  }
  aw_span(a, q);
  if (!ONE && a.window > 0) split += q.lo / 16 * 16 / a.kps;
  char* ring = smem + worker * S::RING;
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  auto clear = [&]() {  // columns behind the head: zeros; the accumulators of a split lie over them at its end
    for (int c = lane + 32 * part; c < S::STAGES * 2 * 16 * CP; c += 32 * WPP)
      if (c % CP * 8 >= a.d) *(uint4*)(ring + c / CP * S::PITCH + c % CP * 16) = make_uint4(0, 0, 0, 0);
  };
  if (a.d < DP) clear();
  const uint64_t policy = aw_policy(a.tiles == 1);
  int all_last = 0x7fffffff, all_from = 0;  // slots that every row of the tile sees: pages inside need no mask
#pragma unroll
  for (int nt = 0; nt < NT; nt++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
      from[nt][e] = a.window > 0 ? last[nt][e] - a.window + 1 : 0;
      if (live[nt][e]) all_last = min(all_last, last[nt][e]), all_from = max(all_from, from[nt][e]);
    }
  all_last = __reduce_min_sync(0xffffffffu, all_last), all_from = __reduce_max_sync(0xffffffffu, all_from);
  const float scale2 = a.scale * AW_LOG2E;
  float* scores = a.scores + (((long long)b * a.hkv + h) * a.vecs + tile * TILE + part * NT * 8 + lane % 4 * 2) * a.kv_pad + lane / 4;
  // ldmatrix: lane i gives row i % 8 of matrix i / 8
  const int lr = lane & 7, lm = lane >> 3;
  const uint32_t k_off = (lr + (lm & 1) * 8) * S::PITCH + (lm >> 1) * 16;  // slots 0-7, 8-15, then the next 8 values
  const uint32_t v_off = (lr + (lm >> 1) * 8) * S::PITCH + (lm & 1) * 16;  // turned: values 0-7, 8-15, then slots 8-15

  // the warps of a page: what they copied is there for all, and what they read may be overwritten
  auto meet = [&]() {
    if (WPP == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(worker + 1), "n"(WPP * 32) : "memory");
  };

  // one split, unless rows with a window lie so far apart that there are more than blocks
  bool redo = false;  // the same split once more
  for (;; split += redo ? 0 : (int)gridDim.x) {
    const int k0 = max(split * a.kps, q.lo / 16 * 16), k1 = min(split * a.kps + a.kps, q.n);
    if (!ONE && k0 >= k1) return;  // the whole block
    const int p0 = k0 / 16, p1 = k0 < k1 ? (k1 + 15) / 16 : p0;
    const int count = min(TILE, vecs - tile * TILE);
    // A weight's high part and rest times an infinite value are not its product (the rest may be 0 or negative): where an
    // output comes out NaN and its sum of weights did not, the split is done again, with every page looked through
    auto run = [&](auto again) __attribute__((always_inline)) -> bool {
      if (a.window > 0 || split != (int)blockIdx.x || again) {
        next = p0 + ((worker - p0) & (RINGS - 1));
        entry = next < p1 ? table[next] : 0;
      }
      int page = next;
      uint32_t pages_ok = 0;  // of the pages in flight, the newest in bit 0: the table names one of the cache
      auto fetch = [&](int stage) {
        const bool ok = entry >= 0 && entry < a.pages;
        pages_ok = pages_ok << 1 | (ok ? 1u : 0u);
        if (next < p1) {
          const long long at = ok ? ((long long)entry * a.hkv + h) * 16 * a.d * 2 : 0;
          const int rows = ok ? min(16, q.n - next * 16) : 0;
          const uint32_t dst = ring_at + stage * 2 * S::PAGE;
          if (rows == 16 && a.d == DP) {  // a page lies in one piece
            const char* k = a.k + at + lane * 16;
            const char* v = a.v + at + lane * 16;
#pragma unroll
            for (int i = part; i < 16 * CP / 32; i += WPP) {
              const int c = lane + 32 * i;
              aw_copy16(dst + c / CP * S::PITCH + c % CP * 16, k + i * 512, true, policy);
              aw_copy16(dst + S::PAGE + c / CP * S::PITCH + c % CP * 16, v + i * 512, true, policy);
            }
          } else {
#pragma unroll
            for (int i = part; i < 16 * CP / 32; i += WPP) {
              const int c = lane + 32 * i, row = c / CP, col = c % CP;
              if (col * 8 < a.d) {
                const bool in = row < rows;
                const long long off = at + (in ? (row * a.d + col * 8) * 2 : 0);
                aw_copy16(dst + row * S::PITCH + col * 16, a.k + off, in, policy);
                aw_copy16(dst + S::PAGE + row * S::PITCH + col * 16, a.v + off, in, policy);
              }
            }
          }
        }
        aw_commit();
        next += RINGS;
        entry = next < p1 ? table[next] : 0;
      };
      meet();
#pragma unroll
      for (int i = 0; i < S::STAGES - 1; i++) fetch(i);

      float o[STEPS][NT][4];  // head values 16 i + lane / 4 (+ 8) of vectors 2 (lane mod 4) (+ 1)
#pragma unroll
      for (int i = 0; i < STEPS; i++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.f;
      float m[NT][2], l[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; nt++) m[nt][0] = m[nt][1] = -INFINITY, l[nt][0] = l[nt][1] = 0.f;
      for (int stage = 0; page < p1; page += RINGS) {
        aw_wait<S::STAGES - 2>();
        meet();
        const bool ok = pages_ok >> (S::STAGES - 2) & 1;
        const int ahead = stage + S::STAGES - 1;
        fetch(ahead >= S::STAGES ? ahead - S::STAGES : ahead);
        const uint32_t kp = ring_at + stage * 2 * S::PAGE, vp = kp + S::PAGE;
        const char* v_page = ring + stage * 2 * S::PAGE + S::PAGE;
        // slots lane / 4 (c0, c1) and + 8 (c2, c3) of vectors 2 (lane mod 4) and the next; even and odd steps apart, two
        // shorter chains of products
        float s[NT][4], s_odd[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 4; e++) s[nt][e] = s_odd[nt][e] = 0.f;
#pragma unroll
        for (int st = 0; st < STEPS; st++) {
          uint32_t ka[4];
          aw_ldsm(ka, kp + k_off + st * 32);
#pragma unroll
          for (int nt = 0; nt < NT; nt++) {
            Ty::mma(st & 1 ? s_odd[nt] : s[nt], ka, qf[st][nt][0], qf[st][nt][1]);
          }
        }
        const int j0 = page * 16 + lane / 4;  // this lane's slots: j0, j0 + 8
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 4; e++) s[nt][e] = (s[nt][e] + s_odd[nt][e]) * scale2;
        const bool whole = page * 16 + 15 <= all_last && page * 16 >= all_from && page * 16 + 16 <= q.n && ok;
        if (!whole) {
#pragma unroll
          for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const int j = j0 + (e >> 1) * 8;
              if (!ok || j > last[nt][e & 1] || j < from[nt][e & 1] || j >= q.n) s[nt][e] = -INFINITY;
            }
        }
        // the largest of each vector's scores: every step for all vectors, so that their shuffles overlap
        float top[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 2; e++) top[nt][e] = fmaxf(s[nt][e], s[nt][e + 2]);
#pragma unroll
        for (int x = 4; x < 32; x <<= 1)
#pragma unroll
          for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 2; e++)
              top[nt][e] = fmaxf(top[nt][e], __shfl_xor_sync(0xffffffffu, top[nt][e], x));
        // a vector's base follows its maximum when that is AW_SLACK and more above it: weights of up to 2^AW_SLACK lose
        // nothing, and most pages leave the accumulators alone. Each vector decides for itself, whatever its neighbours
        bool more = false;
        float f[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const float base = top[nt][e] - Ty::SHIFT;
            f[nt][e] = 1.f;
            if (base > m[nt][e] + AW_SLACK) {
              f[nt][e] = aw_exp2(m[nt][e] - base);
              m[nt][e] = base;
              more = true;
            }
          }
        if (__any_sync(0xffffffffu, more)) {
#pragma unroll
          for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              l[nt][e] *= f[nt][e];
#pragma unroll
              for (int i = 0; i < STEPS; i++) o[i][nt][e] *= f[nt][e], o[i][nt][e + 2] *= f[nt][e];
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 2; e++)
            if (live[nt][e]) {
              float* to = ONE ? s_scores + ((part * NT + nt) * 8 + lane % 4 * 2 + e) * held + page * 16 - split * a.kps + lane / 4
                              : scores + (long long)(nt * 8 + e) * a.kv_pad + page * 16;
              to[0] = s[nt][e];
              to[8] = s[nt][e + 2];
            }
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float base = m[nt][e & 1] == -INFINITY ? 0.f : m[nt][e & 1];
            s[nt][e] = aw_exp2(s[nt][e] - base);
            l[nt][e & 1] += s[nt][e];
          }
        bool by_mma = true;
        if (again || (!whole && (a.max_rows > 1 || a.window > 0))) {  // a row may be blind to a slot that holds anything
          bool fine = true;
#pragma unroll 4
          for (int c = lane; c < 16 * CP; c += 32) {
            const uint4 x = *(const uint4*)(v_page + c / CP * S::PITCH + c % CP * 16);
            fine = fine && Ty::finite(x.x) && Ty::finite(x.y) && Ty::finite(x.z) && Ty::finite(x.w);
          }
          by_mma = __all_sync(0xffffffffu, fine);
        }
        if (by_mma) {
          uint32_t hi[NT][2], rest[NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
              const uint2 x = Ty::parts(s[nt][2 * i], s[nt][2 * i + 1]);
              hi[nt][i] = aw_turn(x.x), rest[nt][i] = aw_turn(x.y);
            }
#pragma unroll
          for (int st = 0; st < STEPS; st++) {
            uint32_t va[4];
            aw_ldsm_t(va, vp + v_off + st * 32);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) Ty::mma(o[st][nt], va, hi[nt][0], hi[nt][1]);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) Ty::mma(o[st][nt], va, rest[nt][0], rest[nt][1]);
          }
        } else {
#pragma unroll 1
          for (int kk = 0; kk < 16; kk++) {
            const int src = (kk & 7) * 4 + lane % 4, j = page * 16 + kk;
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
              for (int e = 0; e < 2; e++) {
                const float p = __shfl_sync(0xffffffffu, kk < 8 ? s[nt][e] : s[nt][e + 2], src);
                if (j > last[nt][e] || j < from[nt][e] || j >= q.n) continue;
#pragma unroll
                for (int i = 0; i < STEPS; i++) {
                  const T* v = (const T*)(v_page + kk * S::PITCH) + i * 16 + lane / 4;
                  o[i][nt][e] = fmaf(p, Ty::up(v[0]), o[i][nt][e]);
                  o[i][nt][e + 2] = fmaf(p, Ty::up(v[8]), o[i][nt][e + 2]);
                }
              }
          }
        }
        __syncwarp();
        stage = stage + 1 == S::STAGES ? 0 : stage + 1;
      }
      aw_wait<0>();
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], x);
          const int row = (part * NT + nt) * 8 + lane * 2 + e;
          if (lane < 4) s_m[worker][row] = m[nt][e], s_l[worker][row] = l[nt][e];
          if (ONE && worker == 0 && lane < 4) s_sees[row] = make_int2(from[nt][e], last[nt][e]);
        }
      __syncthreads();  // every warp is done with its ring, which now takes its accumulator
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int row = (part * NT + nt) * 8 + lane % 4 * 2 + e;
          float top = s_m[0][row];
#pragma unroll
          for (int w = 1; w < RINGS; w++) top = fmaxf(top, s_m[w][row]);
          const float f = m[nt][e] == -INFINITY ? 0.f : aw_exp2(m[nt][e] - top);
          float* to = (float*)ring + row * S::JOIN + lane / 4;
          if (live[nt][e]) {
#pragma unroll
            for (int i = 0; i < STEPS; i++) to[i * 16] = o[i][nt][e] * f, to[i * 16 + 8] = o[i][nt][e + 2] * f;
          }
        }
      __syncthreads();
      const long long at = (((long long)b * a.hkv + h) * a.splits + split) * a.vecs + tile * TILE;
      bool odd = false;
      for (int row = warp; row < count; row += WARPS)
        for (int c = lane * 4; c < a.d; c += 128) {
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < RINGS; w++) {
            const float4 y = *(const float4*)(smem + w * S::RING + (row * S::JOIN + c) * 4);
            x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
          }
          if (x.x != x.x || x.y != x.y || x.z != x.z || x.w != x.w) {
            float sums = 0.f;
#pragma unroll
            for (int w = 0; w < RINGS; w++) sums += s_l[w][row];
            odd = odd || sums == sums;
          }
          if (ONE) *(float4*)(s_out + row * S::JOIN + c) = x;
          else *(float4*)(a.parts + (at + row) * a.d + c) = x;
        }
      if (t < count) {
        float mm = s_m[0][t];
#pragma unroll
        for (int w = 1; w < RINGS; w++) mm = fmaxf(mm, s_m[w][t]);
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < RINGS; w++) sum += s_l[w][t] == 0.f ? 0.f : aw_exp2(s_m[w][t] - mm) * s_l[w][t];  // 0: no slot
        if (ONE) s_stat[t] = make_float2(mm, sum);
        else a.stats[at + t] = make_float2(mm, sum);
      }
      return __syncthreads_or(odd);  // the ring is the copies' again
    };
    if constexpr (ONE) {  // two copies: with a loop the only split's pages take 0.7 us longer (3500 slots and more)
      if (run(std::false_type())) {
        if (a.d < DP) clear();
        run(std::true_type());
      }
      cg::cluster_group cluster = cg::this_cluster();
      const int ranks = gridDim.x;
      // this block's slots and their weights so far, on their way while the blocks meet
      const int n = (int)min((long long)min(split * a.kps + a.kps, q.n), a.cap), first = aw_first(a, q);
      const long long base = (q.slot * a.hkv + h) * a.cap;
      constexpr int MOST = 768 / (WARPS * 32);  // slots of a thread: AW_HELD / 4 / 8 of a block
      float old[MOST];
#pragma unroll
      for (int i = 0; i < MOST; i++) {
        const int j = split * a.kps + t + i * WARPS * 32;
        old[i] = j < n && j < first ? a.weights[base + j] : 0.f;
      }
      cluster.sync();
      for (int i = t; i < ranks * count; i += WARPS * 32) {
        const int r = i / count, v = i - r * count;
        s_all[r][v] = *cluster.map_shared_rank(&s_stat[v], r);
      }
      __syncthreads();
      for (int v = warp; v < count; v += WARPS) {  // as aw_total does
        float mm = lane < ranks ? s_all[lane % AW_CLUSTER][v].x : -INFINITY;
        float ll = lane < ranks ? s_all[lane % AW_CLUSTER][v].y : 0.f;
        const float2 st = aw_join(mm, ll);
        if (lane == 0) s_total[v] = st;
      }
      __syncthreads();
      // the output: splits in eight runs, as aw_finish_kernel joins them; four values a thread, dealt to the blocks
      for (int u = split + ranks * t; u < count * (a.d / 4); u += ranks * WARPS * 32) {
        const int v = u / (a.d / 4), c = (u - v * (a.d / 4)) * 4;
        const float2 st = s_total[v];
        float4 x[AW_CLUSTER];
#pragma unroll
        for (int r = 0; r < AW_CLUSTER; r++)
          if (r < ranks) x[r] = *(const float4*)cluster.map_shared_rank(s_out + v * S::JOIN + c, r);
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int run = 0; run < 8; run++) {
          float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int r = run; r < AW_CLUSTER; r += 8) {
            const float at_r = r < ranks ? s_all[r][v].x : -INFINITY;
            if (at_r != -INFINITY) {
              const float f = aw_exp2(at_r - st.x);
              y.x = fmaf(f, x[r].x, y.x), y.y = fmaf(f, x[r].y, y.y);
              y.z = fmaf(f, x[r].z, y.z), y.w = fmaf(f, x[r].w, y.w);
            }
          }
          sum.x += y.x, sum.y += y.y, sum.z += y.z, sum.w += y.w;
        }
        aw_store<T>(a, q, h, group, v, c, sum, st.y);
      }
      // the weights of this block's slots
#pragma unroll
      for (int i = 0; i < MOST; i++) {
        const int j = split * a.kps + t + i * WARPS * 32;
        if (j >= n) continue;
        float sum = 0.f;
        for (int v = 0; v < count && j >= k0; v++) {  // no row sees the slots before
          const float2 st = s_total[v];
          const int2 sees = s_sees[v];
          if (j >= sees.x && j <= sees.y) sum = fmaf(aw_exp2(s_scores[v * held + j - split * a.kps] - st.x), st.y, sum);
        }
        a.weights_out[base + j] = old[i] + sum;
      }
      cluster.sync();  // nobody leaves while its accumulators are read
      return;
    }
    redo = run(redo) && !redo;
    if (a.d < DP) clear();
  }
}

// The final maximum and 1 / sum of one vector over its splits [s0, s1), by a warp; every lane gets them. Split s is lane
// s mod 32's, whatever s0 and s1 are: splits that a row does not see change no bit of its sum.
__device__ __forceinline__ float2 aw_total(const AwArgs& a, long long head, int v, int s0, int s1) {
  const int lane = threadIdx.x & 31;
  float m = -INFINITY, l = 0.f;
  for (int s = s0 + ((lane - s0) & 31); s < s1; s += 32) {
    const float2 x = a.stats[(head * a.splits + s) * a.vecs + v];
    aw_add(m, l, x.x, x.y);
  }
  return aw_join(m, l);
}

// Joins the splits of a (sequence, kv head): the first a.joins blocks of x the output, 128 values of one vector a job of
// a.join_warps warps, which share its splits; the others add up the slots' weights, four a thread or a few threads.
template <typename T>
__global__ void __launch_bounds__(AW_FIN_THREADS, 4) aw_finish_kernel(AwArgs a) {
  extern __shared__ __align__(16) char fin[];
  // Before the wait only what the first kernel does not write: its blocks let this one start after their own wait, so
  // everything before the first kernel is done. weights_out is written behind the wait (weights may be it).
  const int b = blockIdx.z, h = blockIdx.y, t = threadIdx.x, lane = t & 31, warp = t >> 5;
  constexpr int WARPS = AW_FIN_THREADS / 32;
  AwSeq q = aw_seq(a, b);
  aw_span(a, q);
  const int group = a.hq / a.hkv, vecs = q.rows * group;
  const long long head = (long long)b * a.hkv + h;
  const int lo = q.lo / 16 * 16;  // splits [s0, s1) hold a visible slot
  const int s0 = lo / a.kps, s1 = lo < q.n ? (q.n + a.kps - 1) / a.kps : s0;
  if ((int)blockIdx.x < a.joins) {
    pdl_wait();
    pdl_trigger();
    const int segments = (a.d + 127) / 128;  // of 128 values
    const int job = blockIdx.x * (WARPS / a.join_warps) + warp / a.join_warps;
    const int v = job / segments, c = job % segments * 128 + lane * 4;
    // the splits are added in eight runs, split s to run s mod 8, and the runs in their order, however many warps do it
    constexpr int RUNS = AW_FIN_THREADS / 32;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float2 st = make_float2(0.f, 0.f);
    auto add = [&](int run) {
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int s = s0 + ((run - s0) & (RUNS - 1)); s < s1; s += RUNS) {
        const long long at = (head * a.splits + s) * a.vecs + v;
        const float m = a.stats[at].x;
        const float4 x = *(const float4*)(a.parts + at * a.d + c);
        if (m != -INFINITY) {
          const float f = aw_exp2(m - st.x);
          y.x = fmaf(f, x.x, y.x), y.y = fmaf(f, x.y, y.y), y.z = fmaf(f, x.z, y.z), y.w = fmaf(f, x.w, y.w);
        }
      }
      return y;
    };
    if (v < vecs) st = aw_total(a, head, v, s0, s1);
    if (a.join_warps > 1) {
      float4* sums = (float4*)fin;
      if (v < vecs && c < a.d) o = add(warp);
      sums[t] = o;
      __syncthreads();
      if (warp) return;
      for (int w = 1; w < RUNS; w++) {
        const float4 x = sums[t + w * 32];
        o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
      }
    } else if (v < vecs && c < a.d && s1 - s0 <= RUNS) {  // a split a run at most: all loads on their way at once
      float4 x[RUNS];
      float m[RUNS];
#pragma unroll
      for (int run = 0; run < RUNS; run++) {
        const int s = s0 + ((run - s0) & (RUNS - 1));
        const long long at = (head * a.splits + s) * a.vecs + v;
        m[run] = s < s1 ? a.stats[at].x : -INFINITY;
        if (s < s1) x[run] = *(const float4*)(a.parts + at * a.d + c);
      }
#pragma unroll
      for (int run = 0; run < RUNS; run++)
        if (m[run] != -INFINITY) {
          const float f = aw_exp2(m[run] - st.x);
          // not contracted: a run's sum is rounded before it joins
          o.x = __fadd_rn(o.x, __fmul_rn(f, x[run].x)), o.y = __fadd_rn(o.y, __fmul_rn(f, x[run].y));
          o.z = __fadd_rn(o.z, __fmul_rn(f, x[run].z)), o.w = __fadd_rn(o.w, __fmul_rn(f, x[run].w));
        }
    } else if (v < vecs && c < a.d) {
      o = add(0);
#pragma unroll
      for (int run = 1; run < RUNS; run++) {
        const float4 x = add(run);
        o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
      }
    }
    if (v < vecs && c < a.d) aw_store<T>(a, q, h, group, v, c, o, st.y);
    return;
  }
  // a.groups threads share four slots, each with its part of the vectors
  const int n = (int)min((long long)q.n, a.cap);
  const int quads = AW_FIN_THREADS / a.groups, part = t / quads;
  int j0 = (blockIdx.x - a.joins) * quads * 4;
  if (j0 >= n) return;  // no wait: nothing is read or written
  const int step = (gridDim.x - a.joins) * quads * 4;
  const int first = aw_first(a, q);
  const bool aligned4 = a.cap % 4 == 0 && a.wide_weights;
  const float* scores = a.scores + head * a.vecs * a.kv_pad;
  const long long base = (q.slot * a.hkv + h) * a.cap;
  constexpr int AHEAD = 4;  // vectors whose scores are on their way at a time, the first while the sums are found
  float4 ahead[AHEAD];
  float old[4];
  int j = j0 + t % quads * 4;
  auto load_old = [&]() {
#pragma unroll
    for (int i = 0; i < 4; i++) old[i] = 0.f;
    if (part) return;
    if (aligned4 && j + 3 < n && j + 3 < first) {
      const float4 x = *(const float4*)(a.weights + base + j);
      old[0] = x.x, old[1] = x.y, old[2] = x.z, old[3] = x.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (j + i < n && j + i < first) old[i] = a.weights[base + j + i];
    }
  };
  auto load_scores = [&](int v0) {
#pragma unroll
    for (int i = 0; i < AHEAD; i++) {  // what lies behind n was never written, and is not used
      const int v = v0 + i * a.groups;
      if (v < vecs && j < n && j + 3 >= q.lo) ahead[i] = *(const float4*)(scores + (long long)v * a.kv_pad + j);
    }
  };
  load_old();
  pdl_wait();
  pdl_trigger();
  load_scores(part);
  // of each vector: maximum, 1 / sum, and the slots that it sees, [from, last]
  float4* s_vec = (float4*)fin;
  float4* s_sum = s_vec + a.vecs;  // [AW_FIN_THREADS]
  auto keep = [&](int v, float2 st) {
    const int slot = a.row_slot[q.row0 + v / group];
    s_vec[v] = make_float4(st.x, st.y, __int_as_float(a.window > 0 ? slot - a.window + 1 : 0), __int_as_float(slot));
  };
  if (vecs > 2 * WARPS && s1 - s0 <= 16) {  // many vectors of few splits: a thread each
    for (int v = t; v < vecs; v += AW_FIN_THREADS) {
      float m = -INFINITY, l = 0.f;
#pragma unroll 4
      for (int s = s0; s < s1; s++) {
        const float2 x = a.stats[(head * a.splits + s) * a.vecs + v];
        aw_add(m, l, x.x, x.y);
      }
      keep(v, make_float2(m == -INFINITY ? 0.f : m, l == 0.f ? 0.f : 1.f / l));
    }
  } else {
    for (int v = warp; v < vecs; v += WARPS) {
      const float2 st = aw_total(a, head, v, s0, s1);
      if (lane == 0) keep(v, st);
    }
  }
  __syncthreads();
  for (; j0 < n; j0 += step) {
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    if (j < n && j + 3 >= q.lo) {  // else no row sees them
      for (int v0 = part; v0 < vecs; v0 += AHEAD * a.groups) {
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
          const int v = v0 + i * a.groups;
          if (v >= vecs) continue;
          const float4 vec = s_vec[v];
          const float y[4] = {ahead[i].x, ahead[i].y, ahead[i].z, ahead[i].w};
          const int from = __float_as_int(vec.z), to = __float_as_int(vec.w);
#pragma unroll
          for (int e = 0; e < 4; e++)
            if (j + e >= from && j + e <= to) sum[e] = fmaf(aw_exp2(y[e] - vec.x), vec.y, sum[e]);
        }
        load_scores(v0 + AHEAD * a.groups);
      }
    }
    if (a.groups > 1) {  // the parts, in their order
      s_sum[t] = make_float4(sum[0], sum[1], sum[2], sum[3]);
      __syncthreads();
      if (part == 0)
        for (int g = 1; g < a.groups; g++) {
          const float4 x = s_sum[t + g * quads];
          sum[0] += x.x, sum[1] += x.y, sum[2] += x.z, sum[3] += x.w;
        }
      __syncthreads();
    }
    if (part == 0 && j < n) {
      float* to = a.weights_out + base + j;
      if (aligned4 && j + 3 < n) {
        *(float4*)to = make_float4(old[0] + sum[0], old[1] + sum[1], old[2] + sum[2], old[3] + sum[3]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (j + i < n) to[i] = old[i] + sum[i];
      }
    }
    j += step;
    load_old();
    load_scores(part);
  }
}

struct AwPlan {
  int kps, splits, tile, tiles, seen;
  long long vecs, kv_pad;
  bool one;                     // one kernel does it
  size_t scores, stats, parts;  // bytes
};

static size_t aw_round(size_t n) { return (n + 255) / 256 * 256; }

// Blocks of the first kernel on an SM, by their shared memory (tiles of 24: registers). For head_dim 128 three with rings of two pages read 5.7 TB/s
// where two with rings of three read 5.5 (131071 slots 99.9 against 102.7 us, 32 sequences 156.8 against 162.1 us).
static int aw_resident(int64_t D, int tile) { return tile == 24 ? 2 : D > 64 ? 3 : 4; }

// How a call is cut: keys_per_split as given, or such that the groups (sequence, kv head, tile) fill the device's resident
// blocks once; where there are groups enough for that, splits of up to 768 keys, since the groups' lengths differ (shorter
// ones cost more in the blocks' starts than they even out: 12 sequences of 9 rows over a window of 512 took 56 us with 64
// keys a split).
static AwPlan aw_plan(int64_t B, int64_t rows, int64_t Hq, int64_t Hkv, int64_t D, int64_t kv, int64_t window,
                      int64_t kps) {
  AwPlan p;
  p.vecs = rows * (Hq / Hkv);
  // of 8, 16 or (heads up to 128) 24 vectors; a page costs about 10, 16 and 23
  p.tile = p.vecs <= 8 ? 8 : 16;
  if (D <= 128 && p.vecs > 16 && (p.vecs + 23) / 24 * 23 < (p.vecs + 15) / 16 * 16) p.tile = 24;
  p.tiles = (int)((p.vecs + p.tile - 1) / p.tile);
  p.kv_pad = (kv + 63) / 64 * 64;
  // one kernel: no window, or one of half the slots and more (the blocks are those of all slots), one tile, blocks that are
  // on the device at once. One row with a window of 512 over 1000 slots 10.9 us a call, with two kernels 14.7 (as a graph 9.4 and
  // 11.0); of 1024 over 2048 11.0 and 14.8 (10.2 and 8.2)
  const int64_t groups = B * Hkv * p.tiles;
  auto one = [&](int64_t k) {
    const int64_t n = (kv + k - 1) / k;
    return (window == 0 || 2 * (window + rows) >= kv) && p.tiles == 1 && n <= AW_CLUSTER && groups * n <= 296 && p.tile * k * 4 <= AW_HELD;
  };
  if (kps == 0) {
    const int64_t resident = 148 * aw_resident(D, p.tile);
    const int64_t seen = window > 0 && window + rows < kv ? window + rows : kv;  // slots a sequence's rows can see
    const int64_t most = groups <= 296 ? 296 / groups : 1, few = most < AW_CLUSTER ? most : AW_CLUSTER;
    kps = ((kv + few - 1) / few + 63) / 64 * 64;
    // up to 320 keys a block (128 for wide heads or 16 vectors, 64 for 24): one row over 5000 slots takes 13.9 us a call with
    // one kernel and 14.7 with two (as a graph 13.7 and 11.6), over 6144 slots 14.8 and 15.0 (14.6 and 12.5); 5 rows of 32/8
    // heads over 2048 slots 18.2 with blocks of 128 keys and 16.8 with two kernels
    if (!one(kps) || kps > (p.tile == 24 ? 64 : D <= 128 && p.tile == 8 ? 320 : 128)) {
      const int64_t want = groups * 2 >= resident ? (seen + 767) / 768 : resident / groups;
      kps = ((seen + want - 1) / want + 63) / 64 * 64;
    }
  }
  if (kps > p.kv_pad) kps = p.kv_pad;
  p.kps = (int)kps;
  p.splits = (int)((kv + kps - 1) / kps);
  p.one = one(kps);
  p.seen = !p.one && window > 0 && (window + rows) / kps + 2 < p.splits ? (int)((window + rows) / kps + 2) : p.splits;
  const size_t heads = p.one ? 0 : (size_t)B * Hkv;
  p.scores = aw_round(heads * p.vecs * p.kv_pad * 4);
  p.stats = aw_round(heads * p.splits * p.vecs * 8);
  p.parts = aw_round(heads * p.splits * p.vecs * D * 4);
  return p;
}

template <typename T, int DP, int NT, int WPP>
int launch_split(const AwArgs& a, bool one, dim3 grid, cudaStream_t st) {
  constexpr int threads = AwShape<DP, NT, WPP>::WARPS * 32;
  if (one) {
    const int rc = configure<aw_split_kernel<T, DP, NT, WPP, true>>("aw_split_kernel", AwShape<DP, NT, WPP>::SMEM_ONE, true);
    if (rc != IM_OK) return rc;
    return launch_cluster("aw_split_kernel", aw_split_kernel<T, DP, NT, WPP, true>, grid, dim3(threads), (int)grid.x,
                          AwShape<DP, NT, WPP>::SMEM + AwShape<DP, NT, WPP>::TILE * (AwShape<DP, NT, WPP>::JOIN + a.kps + 4) * 4, st, a);
  }
  constexpr int smem = AwShape<DP, NT, WPP>::SMEM;
  const int rc = configure<aw_split_kernel<T, DP, NT, WPP, false>>("aw_split_kernel", smem, false);
  if (rc != IM_OK) return rc;
  return launch("aw_split_kernel", aw_split_kernel<T, DP, NT, WPP, false>, grid, dim3(threads), smem, st, a);
}

// Wide heads leave an SM room for six rings; a warp a tile of 8 vectors there: 9 rows of 32/8 heads of 256 over 6762 slots
// take 44.5 us, with one warp for both tiles 48.6; 2 rows of 16/2 over 3000 slots 14.4 and 17.1. Up to 128 the products bound it
// with either, and a second warp that reads the same page costs more than it hides: 8 x 5 rows of 32/8 heads of 128 over
// 8192 slots 77 us with one, 89 with three.
template <typename T, int NT>
int launch_split_d(const AwArgs& a, bool one, dim3 grid, cudaStream_t st) {
  return a.d <= 64    ? launch_split<T, 64, NT, 1>(a, one, grid, st)
         : a.d <= 96  ? launch_split<T, 96, NT, 1>(a, one, grid, st)
         : a.d <= 128 ? launch_split<T, 128, NT, 1>(a, one, grid, st)
                      : launch_split<T, 256, 1, NT < 3 ? NT : 2>(a, one, grid, st);  // NT 3 is not chosen for them
}

template <typename T>
int launch_attention_weights(AwArgs& a, bool one, int64_t B, cudaStream_t st) {
  const dim3 grid((unsigned)a.seen, (unsigned)(a.hkv * a.tiles), (unsigned)B);
  const int rc = a.tile == 8    ? launch_split_d<T, 1>(a, one, grid, st)
                 : a.tile == 16 ? launch_split_d<T, 2>(a, one, grid, st)
                                : launch_split_d<T, 3>(a, one, grid, st);
  if (rc != IM_OK || one) return rc;
  // many splits that a row can see: a block's eight warps share a job's, else each has a job
  a.join_warps = a.seen >= 16 ? AW_FIN_THREADS / 32 : 1;
  a.joins = (int)(((int64_t)a.vecs * ((a.d + 127) / 128) * a.join_warps * 32 + AW_FIN_THREADS - 1) / AW_FIN_THREADS);
  // blocks of slots a (sequence, kv head): the device's worth in all, so that a block's sums serve many slots; where the
  // slots are too few for them, threads share slots by vectors
  const int64_t share = (369 + B * a.hkv) / (B * a.hkv);
  auto blocks = [&](int groups) { return ((int64_t)a.max_kv * groups + AW_FIN_THREADS * 4 - 1) / (AW_FIN_THREADS * 4); };
  a.groups = 1;
  while (a.groups < 8 && a.vecs >= a.groups * 16 && blocks(a.groups * 2) <= (share > 2 ? share : 2)) a.groups *= 2;
  const int chunks = (int)(blocks(a.groups) < share ? blocks(a.groups) : share);
  const size_t join = sizeof(float4) * AW_FIN_THREADS, sums = sizeof(float4) * (a.vecs + AW_FIN_THREADS);
  return launch("aw_finish_kernel", aw_finish_kernel<T>, dim3((unsigned)(a.joins + chunks), (unsigned)a.hkv, (unsigned)B),
                dim3(AW_FIN_THREADS), join > sums ? join : sums, st, a);
}

}  // namespace im

using namespace im;

extern "C" size_t im_attention_weights_workspace_bytes(int64_t B, int64_t max_rows_per_seq, int64_t Hq, int64_t Hkv,
                                                       int64_t D, int64_t max_kv_len, int64_t keys_per_split,
                                                       int64_t window) {
  if (B < 1 || max_rows_per_seq < 1 || Hkv < 1 || Hq < 1 || Hq % Hkv || D < 16 || max_kv_len < 1 || keys_per_split < 0 || window < 0)
    return 0;
  const AwPlan p = aw_plan(B, max_rows_per_seq, Hq, Hkv, D, max_kv_len, window, keys_per_split);
  return p.scores + p.stats + p.parts;
}

extern "C" int im_attention_weights(const void* q, const void* k_cache, const void* v_cache, int dtype,
                                    const int32_t* page_table, int64_t seqs, int64_t max_pages, int64_t pages,
                                    const int32_t* seq_rows, const int32_t* seq_slot, const int32_t* row_slot, int64_t M,
                                    int64_t B, int64_t max_rows_per_seq, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_kv_len,
                                    int64_t keys_per_split, int64_t window, float scale, const float* weights,
                                    float* weights_out, int64_t cap, void* out, void* workspace, size_t workspace_bytes,
                                    void* stream) {
  clear_error();
  IM_REQUIRE(M >= 0 && B >= 0 && max_rows_per_seq >= 0 && Hkv >= 1 && Hq >= 1 && Hq % Hkv == 0 && max_kv_len >= 0 && window >= 0 &&
                 cap >= 0 && seqs >= 0 && pages >= 0 && max_pages >= 0,
             IM_INVALID, "im_attention_weights: bad sizes");
  IM_REQUIRE(keys_per_split >= 0 && keys_per_split % 64 == 0, IM_INVALID,
             "im_attention_weights: keys_per_split %lld (a multiple of 64, or 0)", (long long)keys_per_split);
  IM_REQUIRE(dtype == IM_BF16 || dtype == IM_F16, IM_UNSUPPORTED, "im_attention_weights: type %d (bf16 or fp16)", dtype);
  IM_REQUIRE(D >= 16 && D <= 256 && D % 16 == 0, IM_UNSUPPORTED,
             "im_attention_weights: head_dim %lld (multiples of 16 up to 256)", (long long)D);
  if (M == 0 || B == 0 || max_rows_per_seq == 0) return IM_OK;
  IM_REQUIRE(q && k_cache && v_cache && page_table && seq_rows && row_slot && out && ((weights && weights_out) || cap == 0),
             IM_INVALID,
             "im_attention_weights: null pointer");
  IM_REQUIRE(aligned(q, 16) && aligned(k_cache, 16) && aligned(v_cache, 16) && aligned(out, 16), IM_INVALID,
             "im_attention_weights: q, the caches and out must be 16-byte aligned");
  IM_REQUIRE(aligned(weights, 4) && aligned(weights_out, 4) && aligned(page_table, 4) && aligned(seq_rows, 4) &&
                 aligned(seq_slot, 4) && aligned(row_slot, 4),
             IM_INVALID, "im_attention_weights: misaligned pointer");
  IM_REQUIRE(M < (1ll << 31) && B < 65536 && Hkv <= 4096 && max_rows_per_seq <= 4096 && Hq / Hkv <= 256 &&
                 max_rows_per_seq * (Hq / Hkv) <= 2048 && max_kv_len < (1ll << 30) && window < (1ll << 30),
             IM_UNSUPPORTED, "im_attention_weights: too large");
  const int64_t kv = max_kv_len > 0 ? max_kv_len : 1;
  const size_t need = im_attention_weights_workspace_bytes(B, max_rows_per_seq, Hq, Hkv, D, kv, keys_per_split, window);
  IM_REQUIRE(need == 0 || (workspace && aligned(workspace, 256) && workspace_bytes >= need), IM_INVALID,
             "im_attention_weights: a workspace of %zu bytes needed, %zu given", need, workspace_bytes);
  AwArgs a = {};
  const AwPlan p = aw_plan(B, max_rows_per_seq, Hq, Hkv, D, kv, window, keys_per_split);
  IM_REQUIRE(Hkv * p.tiles < 65536, IM_UNSUPPORTED, "im_attention_weights: too large");
  a.q = (const char*)q, a.k = (const char*)k_cache, a.v = (const char*)v_cache;
  a.page_table = page_table, a.seqs = seqs, a.max_pages = max_pages, a.pages = pages;
  a.seq_rows = seq_rows, a.seq_slot = seq_slot, a.row_slot = row_slot;
  a.weights = weights, a.weights_out = weights_out, a.cap = cap;
  a.M = (int)M, a.max_rows = (int)max_rows_per_seq, a.hq = (int)Hq, a.hkv = (int)Hkv, a.d = (int)D;
  a.max_kv = (int)max_kv_len, a.kv_pad = (int)p.kv_pad, a.window = (int)window, a.scale = scale, a.out = (char*)out;
  a.kps = p.kps, a.splits = p.splits, a.tile = p.tile, a.tiles = p.tiles, a.seen = p.seen, a.vecs = (int)p.vecs;
  a.wide_weights = aligned(weights, 16) && aligned(weights_out, 16);
  a.scores = (float*)workspace;
  a.stats = (float2*)((char*)workspace + p.scores);
  a.parts = (float*)((char*)workspace + p.scores + p.stats);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return dtype == IM_BF16 ? launch_attention_weights<__nv_bfloat16>(a, p.one, B, st)
                          : launch_attention_weights<__half>(a, p.one, B, st);
}
