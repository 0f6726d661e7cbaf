// Attention of a few new rows a sequence over the paged cache, which also adds up every slot's attention weight.
//
//   s[r, g, j] = scale q[r, g] . k[j] for the slots j that row r sees, p = softmax over j, out = sum_j p v[j]
//   weights'[h, j] = (j before the sequence's first new slot ? weights[h, j] : 0) + sum over rows r and the query heads
//   g of kv head h of p[r, g, j]
//
// Bound: HBM, K and V of every visible slot read once (2 * 2 D bytes a slot and kv head).
//
// First kernel (aw_split_kernel): a block takes one split of a (sequence, kv head) and up to 16 of its (row, query head)
// vectors, one row each of the warp MMA's m16. Its four warps take the split's pages in turn, each with a ring of pages of
// its own in shared memory (asynchronous copies, no barrier between warps), a running maximum and sum and a 16 x D
// accumulator in registers; they are joined once at the split's end. With one query group of 4 to 16 vectors the products
// are under a tenth of what mma.sync gives, so tcgen05's tiles of 64 rows and more would only add work. Scores go to
// the workspace in float32 (4 bytes a vector and slot beside 4 D of K and V): the weights need the final maximum and sum.
// Second kernel (aw_finish_kernel): joins the splits, and adds up exp2(s - max) / sum slot by slot.
//
// Weights that meet v are two numbers of the cache's type, high part and rest (16 bits and more of each weight are kept);
// in float16 they are scaled by 2^14 first, so that weights down to 2^-28 of the largest are whole numbers' worth. Masked
// slots never reach a row: behind the last visible slot v is zeroed on its way in; between rows of one call a page is
// checked for values that are not finite, and if it has any its products are done one by one.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace im {

constexpr int AW_WARPS = 4;
constexpr int AW_THREADS = AW_WARPS * 32;
constexpr int AW_FIN_THREADS = 256;
constexpr int AW_FIN_SLOTS = AW_FIN_THREADS * 4;
constexpr float AW_LOG2E = 1.4426950408889634f;

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
  int kps, splits, tiles;  // keys a split, splits of max_kv, tiles of 16 vectors
  int vecs;                // max_rows * Hq / Hkv
  float* scores;           // [B][Hkv][vecs][kv_pad], in log2 units
  float2* stats;           // [B][Hkv][splits][vecs]: maximum and sum
  float* parts;            // [B][Hkv][splits][vecs][d]
  int wide_weights;        // weights and weights_out start on 16 bytes
};

// What a block knows of its sequence.
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
  int top = -1, low = 0x7fffffff;
  for (int r = 0; r < s.rows; r++) {
    const int at = a.row_slot[s.row0 + r];
    top = max(top, at);
    if (at >= 0) low = min(low, at);
  }
  const long long most = min((long long)a.max_kv, a.max_pages * 16);
  s.n = s.slot < 0 ? 0 : (int)min((long long)top + 1, most);
  s.lo = a.window > 0 && low != 0x7fffffff ? max(0, low - a.window + 1) : 0;
  return s;
}

__device__ __forceinline__ void aw_copy16(uint32_t dst, const char* src, bool in) {
  const int n = in ? 16 : 0;  // 0: zeros, nothing is read
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
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
  static __device__ __forceinline__ float2 up(uint32_t u) { return make_float2(bf_lo(u), bf_hi(u)); }
  static __device__ __forceinline__ bool finite(uint32_t u) {
    return (u & 0x7f80u) != 0x7f80u && (u & 0x7f800000u) != 0x7f800000u;
  }
  static __device__ __forceinline__ __nv_bfloat16 down(float f) { return __float2bfloat16_rn(f); }
};
template <>
struct AwType<__half> {
  static constexpr float SHIFT = 14.f;
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
  static __device__ __forceinline__ float2 up(uint32_t u) { return __half22float2(*(const __half2*)&u); }
  static __device__ __forceinline__ bool finite(uint32_t u) {
    return (u & 0x7c00u) != 0x7c00u && (u & 0x7c000000u) != 0x7c000000u;
  }
  static __device__ __forceinline__ __half down(float f) { return __float2half_rn(f); }
};

// DP: head_dim rounded up to what is built; columns from d on are zeros in shared memory.
template <int DP>
struct AwShape {
  static constexpr int PITCH = DP * 2 + 16;   // an odd number of 16-byte steps: ldmatrix without bank conflicts
  static constexpr int PAGE = 16 * PITCH;     // one page's K or V
  static constexpr int STAGES = 3;
  static constexpr int RING = STAGES * 2 * PAGE;
  static constexpr int JOIN = 16 * DP * 4;    // a warp's accumulator
  static constexpr bool Q_REGS = DP <= 128;
  static constexpr int Q_BYTES = Q_REGS ? 0 : PAGE;
  static constexpr int SMEM = AW_WARPS * (RING > JOIN ? RING : JOIN) + Q_BYTES;
};

template <typename T, int DP>
__global__ void __launch_bounds__(AW_THREADS) aw_split_kernel(AwArgs a) {
  using S = AwShape<DP>;
  using Ty = AwType<T>;
  extern __shared__ __align__(128) char smem[];
  __shared__ float s_m[AW_WARPS][16], s_l[AW_WARPS][16];
  pdl_wait();
  pdl_trigger();
  const int split = blockIdx.x, h = blockIdx.y / a.tiles, tile = blockIdx.y % a.tiles, b = blockIdx.z;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const AwSeq q = aw_seq(a, b);
  const int k0 = max(split * a.kps, q.lo / 16 * 16), k1 = min(split * a.kps + a.kps, q.n);
  const int group = a.hq / a.hkv;
  const int vecs = q.rows * group;  // live ones
  if (tile * 16 >= vecs || k0 >= k1) return;

  // this lane's two rows of the tile: vectors tile * 16 + lane / 4 (+ 8)
  int last[2], from[2];
  const char* qp[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int vec = tile * 16 + lane / 4 + 8 * i;
    last[i] = -1, from[i] = 0, qp[i] = nullptr;
    if (vec < vecs) {
      const int r = q.row0 + vec / group;
      last[i] = a.row_slot[r];
      from[i] = a.window > 0 ? last[i] - a.window + 1 : 0;
      qp[i] = a.q + ((long long)r * a.hq + h * group + vec % group) * a.d * 2;
    }
  }
  // slots that every row of the tile sees: pages inside need no mask
  int all_last = vecs > tile * 16 ? 0x7fffffff : -1, all_from = 0;
#pragma unroll
  for (int i = 0; i < 2; i++)
    if (qp[i]) all_last = min(all_last, last[i]), all_from = max(all_from, from[i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    all_last = min(all_last, __shfl_xor_sync(0xffffffffu, all_last, o));
    all_from = max(all_from, __shfl_xor_sync(0xffffffffu, all_from, o));
  }

  char* ring = smem + warp * (S::SMEM - S::Q_BYTES) / AW_WARPS;
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  constexpr int STEPS = DP / 16, CP = DP / 8;
  if (a.d < DP) {  // columns behind the head: zeros, once
    for (int c = lane; c < S::STAGES * 2 * 16 * CP; c += 32)
      if (c % CP * 8 >= a.d) *(uint4*)(ring + c / CP * S::PITCH + c % CP * 16) = make_uint4(0, 0, 0, 0);
  }
  uint32_t qf[S::Q_REGS ? STEPS : 1][4];
  const char* q_smem = smem + S::SMEM - S::Q_BYTES;
  if (S::Q_REGS) {
#pragma unroll
    for (int st = 0; st < STEPS; st++) {
      const int col = st * 16 + lane % 4 * 2;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int c = col + (i & 2) * 4;
        const char* p = qp[i & 1];
        qf[S::Q_REGS ? st : 0][i] = p && c < a.d ? *(const uint32_t*)(p + c * 2) : 0u;
      }
    }
  } else {
    for (int c = t; c < 16 * CP; c += AW_THREADS) {
      const int vec = tile * 16 + c / CP, col = c % CP * 8;
      uint4 x = make_uint4(0, 0, 0, 0);
      if (vec < vecs && col < a.d)
        x = *(const uint4*)(a.q + (((long long)(q.row0 + vec / group) * a.hq + h * group + vec % group) * a.d + col) * 2);
      *(uint4*)(smem + S::SMEM - S::Q_BYTES + c / CP * S::PITCH + col * 2) = x;
    }
    __syncthreads();
  }

  const int* table = a.page_table + q.slot * a.max_pages;
  const int p0 = k0 / 16, p1 = (k1 + 15) / 16;
  // pages of this warp: those whose number is warp mod 4, so that a slot's place does not depend on the call
  int next = p0 + ((warp - p0) & (AW_WARPS - 1));
  int page = next;
  // the page numbers are fetched a round ahead of the copies that need them
  int entry = next < p1 ? table[next] : 0;
  uint32_t pages_ok = 0;  // of the pages in flight, the newest in bit 0: the table names one of the cache
  auto fetch = [&](int stage) {
    const bool ok = entry >= 0 && entry < a.pages;
    pages_ok = pages_ok << 1 | (ok ? 1u : 0u);
    if (next < p1) {
      const long long at = ok ? ((long long)entry * a.hkv + h) * 16 * a.d * 2 : 0;
      const int rows = ok ? min(16, q.n - next * 16) : 0;
      const uint32_t dst = ring_at + stage * 2 * S::PAGE;
#pragma unroll
      for (int i = 0; i < 16 * CP / 32; i++) {
        const int c = lane + 32 * i, row = c / CP, col = c % CP;
        if (col * 8 < a.d) {
          const bool in = row < rows;
          const long long off = at + (in ? (row * a.d + col * 8) * 2 : 0);
          aw_copy16(dst + row * S::PITCH + col * 16, a.k + off, in);
          aw_copy16(dst + S::PAGE + row * S::PITCH + col * 16, a.v + off, in);
        }
      }
    }
    aw_commit();
    next += AW_WARPS;
    entry = next < p1 ? table[next] : 0;
  };
  __syncwarp();
#pragma unroll
  for (int i = 0; i < S::STAGES - 1; i++) fetch(i);

  float o[DP / 8][4];
#pragma unroll
  for (int i = 0; i < DP / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  const float scale2 = a.scale * AW_LOG2E;
  float* scores = a.scores + (((long long)b * a.hkv + h) * a.vecs + tile * 16 + lane / 4) * a.kv_pad;
  // ldmatrix: lane i gives row i % 8 of matrix i / 8
  const int lr = lane & 7, lm = lane >> 3;
  const uint32_t k_off = (lr + (lm >> 1) * 8) * S::PITCH + (lm & 1) * 16;
  const uint32_t v_off = (lr + (lm & 1) * 8) * S::PITCH + (lm >> 1) * 16;
  const uint32_t q_off = (uint32_t)__cvta_generic_to_shared(q_smem) + (lr + (lm & 1) * 8) * S::PITCH + (lm >> 1) * 16;

  for (int stage = 0; page < p1; page += AW_WARPS) {
    aw_wait<S::STAGES - 2>();
    __syncwarp();
    const bool ok = pages_ok >> (S::STAGES - 2) & 1;
    const int ahead = stage + S::STAGES - 1;
    fetch(ahead >= S::STAGES ? ahead - S::STAGES : ahead);
    const uint32_t kp = ring_at + stage * 2 * S::PAGE, vp = kp + S::PAGE;
    float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int st = 0; st < STEPS; st++) {
      uint32_t kb[4];
      aw_ldsm(kb, kp + k_off + st * 32);
      if (S::Q_REGS) {
        Ty::mma(s[0], qf[S::Q_REGS ? st : 0], kb[0], kb[1]);
        Ty::mma(s[1], qf[S::Q_REGS ? st : 0], kb[2], kb[3]);
      } else {
        uint32_t qa[4];
        aw_ldsm(qa, q_off + st * 32);
        Ty::mma(s[0], qa, kb[0], kb[1]);
        Ty::mma(s[1], qa, kb[2], kb[3]);
      }
    }
    const int j0 = page * 16 + lane % 4 * 2;  // this lane's slots: j0, j0 + 1, j0 + 8, j0 + 9
#pragma unroll
    for (int nt = 0; nt < 2; nt++)
#pragma unroll
      for (int e = 0; e < 4; e++) s[nt][e] *= scale2;
    const bool whole = page * 16 + 15 <= all_last && page * 16 >= all_from && page * 16 + 16 <= q.n && ok;
    if (!whole) {
#pragma unroll
      for (int nt = 0; nt < 2; nt++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int j = j0 + nt * 8 + (e & 1);
          if (!ok || j > last[e >> 1] || j < from[e >> 1] || j >= q.n) s[nt][e] = -INFINITY;
        }
    }
#pragma unroll
    for (int i = 0; i < 2; i++)
      if (qp[i]) {
        float* to = scores + (long long)i * 8 * a.kv_pad + j0;
        *(float2*)to = make_float2(s[0][2 * i], s[0][2 * i + 1]);
        *(float2*)(to + 8) = make_float2(s[1][2 * i], s[1][2 * i + 1]);
      }
    float top[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      float x = fmaxf(fmaxf(s[0][2 * i], s[0][2 * i + 1]), fmaxf(s[1][2 * i], s[1][2 * i + 1]));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
      top[i] = fmaxf(m[i], x - Ty::SHIFT);
    }
    if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const float f = top[i] > m[i] ? exp2f(m[i] - top[i]) : 1.f;
        m[i] = top[i];
        l[i] *= f;
#pragma unroll
        for (int c = 0; c < DP / 8; c++) o[c][2 * i] *= f, o[c][2 * i + 1] *= f;
      }
    }
    const float base[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll
    for (int nt = 0; nt < 2; nt++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        s[nt][e] = exp2f(s[nt][e] - base[e >> 1]);
        l[e >> 1] += s[nt][e];
      }
    bool by_mma = true;
    if (!whole && (a.max_rows > 1 || a.window > 0)) {  // a row may be blind to a slot of this page that holds anything
      bool fine = true;
      for (int c = lane; c < 16 * (a.d / 2); c += 32)
        fine = fine && Ty::finite(*(const uint32_t*)(ring + stage * 2 * S::PAGE + S::PAGE + c / (a.d / 2) * S::PITCH +
                                                     c % (a.d / 2) * 4));
      by_mma = __all_sync(0xffffffffu, fine);
    }
    if (by_mma) {
      uint32_t hi[4], rest[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint2 x = Ty::parts(s[i >> 1][(i & 1) * 2], s[i >> 1][(i & 1) * 2 + 1]);
        hi[i] = x.x, rest[i] = x.y;
      }
#pragma unroll
      for (int st = 0; st < STEPS; st++) {
        uint32_t vb[4];
        aw_ldsm_t(vb, vp + v_off + st * 32);
        Ty::mma(o[2 * st], hi, vb[0], vb[1]);
        Ty::mma(o[2 * st + 1], hi, vb[2], vb[3]);
        Ty::mma(o[2 * st], rest, vb[0], vb[1]);
        Ty::mma(o[2 * st + 1], rest, vb[2], vb[3]);
      }
    } else {
#pragma unroll 1
      for (int kk = 0; kk < 16; kk++) {
        const int src = (lane & ~3) | ((kk & 7) >> 1);
        float p[2];
        bool see[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const float x = kk < 8 ? (kk & 1 ? s[0][2 * i + 1] : s[0][2 * i]) : (kk & 1 ? s[1][2 * i + 1] : s[1][2 * i]);
          p[i] = __shfl_sync(0xffffffffu, x, src);
          const int j = page * 16 + kk;
          see[i] = j <= last[i] && j >= from[i] && j < q.n;
        }
#pragma unroll
        for (int c = 0; c < DP / 8; c++) {
          const float2 x = Ty::up(*(const uint32_t*)(ring + stage * 2 * S::PAGE + S::PAGE + kk * S::PITCH + c * 16 +
                                                     lane % 4 * 4));
          if (see[0]) o[c][0] = fmaf(p[0], x.x, o[c][0]), o[c][1] = fmaf(p[0], x.y, o[c][1]);
          if (see[1]) o[c][2] = fmaf(p[1], x.x, o[c][2]), o[c][3] = fmaf(p[1], x.y, o[c][3]);
        }
      }
    }
    __syncwarp();
    stage = stage + 1 == S::STAGES ? 0 : stage + 1;
  }
  aw_wait<0>();
#pragma unroll
  for (int i = 0; i < 2; i++) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    if (lane % 4 == 0) s_m[warp][lane / 4 + 8 * i] = m[i], s_l[warp][lane / 4 + 8 * i] = l[i];
  }
  __syncthreads();  // every warp is done with its ring, which now takes its accumulator
  float top[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int row = lane / 4 + 8 * i;
    top[i] = fmaxf(fmaxf(s_m[0][row], s_m[1][row]), fmaxf(s_m[2][row], s_m[3][row]));
    const float f = m[i] == -INFINITY ? 0.f : exp2f(m[i] - top[i]);
    float* to = (float*)ring + row * DP + lane % 4 * 2;
#pragma unroll
    for (int c = 0; c < DP / 8; c++) *(float2*)(to + c * 8) = make_float2(o[c][2 * i] * f, o[c][2 * i + 1] * f);
  }
  __syncthreads();
  const long long at = (((long long)b * a.hkv + h) * a.splits + split) * a.vecs + tile * 16;
  const int live = min(16, vecs - tile * 16);
  constexpr int WARP_BYTES = (S::SMEM - S::Q_BYTES) / AW_WARPS;
  for (int c = t; c < live * (a.d / 4); c += AW_THREADS) {
    const int row = c / (a.d / 4), col = c % (a.d / 4) * 4;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < AW_WARPS; w++) {
      const float4 y = *(const float4*)(smem + w * WARP_BYTES + (row * DP + col) * 4);
      x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
    }
    *(float4*)(a.parts + (at + row) * a.d + col) = x;
  }
  if (t < live) {
    const float mm = fmaxf(fmaxf(s_m[0][t], s_m[1][t]), fmaxf(s_m[2][t], s_m[3][t]));
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < AW_WARPS; w++) sum += s_m[w][t] == -INFINITY ? 0.f : exp2f(s_m[w][t] - mm) * s_l[w][t];
    a.stats[at + t] = make_float2(mm, sum);
  }
}

// The final maximum and 1 / sum of one vector over its splits [s0, s1), by a warp; every lane gets them.
__device__ __forceinline__ float2 aw_total(const AwArgs& a, long long head, int v, int s0, int s1) {
  const int lane = threadIdx.x & 31;
  float m = -INFINITY, l = 0.f;
  for (int s = s0 + lane; s < s1; s += 32) {
    const float2 x = a.stats[(head * a.splits + s) * a.vecs + v];
    const float top = fmaxf(m, x.x);
    if (top != -INFINITY) l = l * exp2f(m - top) + x.y * exp2f(x.x - top);
    m = top;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), l2 = __shfl_xor_sync(0xffffffffu, l, o);
    const float top = fmaxf(m, m2);
    if (top != -INFINITY) l = l * exp2f(m - top) + l2 * exp2f(m2 - top);
    m = top;
  }
  return make_float2(m == -INFINITY ? 0.f : m, l == 0.f ? 0.f : 1.f / l);
}

// Joins the splits of a (sequence, kv head): the first a.vecs blocks of x one vector's output each, its splits dealt to the
// warps; the others add up the weights of AW_FIN_SLOTS slots each, four a thread.
template <typename T>
__global__ void __launch_bounds__(AW_FIN_THREADS) aw_finish_kernel(AwArgs a) {
  extern __shared__ __align__(16) char fin[];
  pdl_wait();
  pdl_trigger();
  const int b = blockIdx.z, h = blockIdx.y, t = threadIdx.x, lane = t & 31, warp = t >> 5;
  constexpr int WARPS = AW_FIN_THREADS / 32;
  const AwSeq q = aw_seq(a, b);
  const int group = a.hq / a.hkv, vecs = q.rows * group;
  const long long head = (long long)b * a.hkv + h;
  const int lo = q.lo / 16 * 16;  // splits [s0, s1) hold a visible slot
  const int s0 = lo / a.kps, s1 = lo < q.n ? (q.n + a.kps - 1) / a.kps : s0;
  if ((int)blockIdx.x < a.vecs) {
    const int v = blockIdx.x;
    if (v >= vecs) return;
    const float2 st = aw_total(a, head, v, s0, s1);
    float* part = (float*)fin;  // [WARPS][d]
    for (int c = lane * 4; c < a.d; c += 128) {
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int s = s0 + warp; s < s1; s += WARPS) {
        const long long at = (head * a.splits + s) * a.vecs + v;
        const float m = a.stats[at].x;
        const float4 x = *(const float4*)(a.parts + at * a.d + c);
        if (m != -INFINITY) {
          const float f = exp2f(m - st.x);
          o.x = fmaf(f, x.x, o.x), o.y = fmaf(f, x.y, o.y), o.z = fmaf(f, x.z, o.z), o.w = fmaf(f, x.w, o.w);
        }
      }
      *(float4*)(part + warp * a.d + c) = o;
    }
    __syncthreads();
    const long long row = q.row0 + v / group;
    for (int c = t; c < a.d; c += AW_FIN_THREADS) {
      float o = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; w++) o += part[w * a.d + c];
      ((T*)a.out)[(row * a.hq + h * group + v % group) * a.d + c] = AwType<T>::down(o * st.y);
    }
    return;
  }
  const int n = (int)min((long long)q.n, a.cap);
  const int j_first = (blockIdx.x - a.vecs) * AW_FIN_SLOTS;
  if (j_first >= n) return;
  float2* s_stat = (float2*)fin;  // [vecs]
  for (int v = warp; v < vecs; v += WARPS) {
    const float2 st = aw_total(a, head, v, s0, s1);
    if (lane == 0) s_stat[v] = st;
  }
  __syncthreads();
  const int j = j_first + t * 4;
  if (j >= n) return;
  const int first = a.row_slot[q.row0];
  const long long at = (q.slot * a.hkv + h) * a.cap + j;
  const float* scores = a.scores + head * a.vecs * a.kv_pad + j;
  const bool wide = j + 3 < n && a.cap % 4 == 0 && a.wide_weights;
  float old[4] = {0.f, 0.f, 0.f, 0.f}, sum[4] = {0.f, 0.f, 0.f, 0.f};
  if (wide && j + 3 < first) {
    const float4 x = *(const float4*)(a.weights + at);
    old[0] = x.x, old[1] = x.y, old[2] = x.z, old[3] = x.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (j + i < n && j + i < first) old[i] = a.weights[at + i];
  }
  for (int r = 0; r < q.rows; r++) {
    const int slot = a.row_slot[q.row0 + r], from = a.window > 0 ? slot - a.window + 1 : 0;
    if (j > slot || j + 3 < from) continue;
#pragma unroll 4
    for (int g = 0; g < group; g++) {
      const float2 st = s_stat[r * group + g];
      const float4 x = *(const float4*)(scores + (long long)(r * group + g) * a.kv_pad);
      const float y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (j + i <= slot && j + i >= from) sum[i] += exp2f(y[i] - st.x) * st.y;
    }
  }
  if (wide) {
    *(float4*)(a.weights_out + at) = make_float4(old[0] + sum[0], old[1] + sum[1], old[2] + sum[2], old[3] + sum[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (j + i < n) a.weights_out[at + i] = old[i] + sum[i];
  }
}

struct AwPlan {
  int kps, splits, tiles;
  long long vecs, kv_pad;
  size_t scores, stats, parts;  // bytes
};

static size_t aw_round(size_t n) { return (n + 255) / 256 * 256; }

// How a call is cut: keys_per_split as given, or such that the groups (sequence, kv head, tile) fill the device's resident
// blocks about once, or several times where there are many groups, since their lengths differ.
static AwPlan aw_plan(int64_t B, int64_t rows, int64_t Hq, int64_t Hkv, int64_t D, int64_t kv, int64_t window,
                      int64_t kps) {
  AwPlan p;
  p.vecs = rows * (Hq / Hkv);
  p.tiles = (int)((p.vecs + 15) / 16);
  p.kv_pad = (kv + 63) / 64 * 64;
  if (kps == 0) {
    const int64_t groups = B * Hkv * p.tiles, resident = D > 128 ? 148 : 296;
    const int64_t seen = window > 0 && window + rows < kv ? window + rows : kv;  // slots a sequence's rows can see
    int64_t want = groups * 2 >= resident ? (resident * 6 + groups - 1) / groups : resident / groups;
    if (want < 1) want = 1;
    kps = ((seen + want - 1) / want + 63) / 64 * 64;
  }
  if (kps > p.kv_pad) kps = p.kv_pad;
  p.kps = (int)kps;
  p.splits = (int)((kv + kps - 1) / kps);
  const size_t heads = (size_t)B * Hkv;
  p.scores = aw_round(heads * p.vecs * p.kv_pad * 4);
  p.stats = aw_round(heads * p.splits * p.vecs * 8);
  p.parts = aw_round(heads * p.splits * p.vecs * D * 4);
  return p;
}

template <typename T, int DP>
int launch_split(const AwArgs& a, dim3 grid, cudaStream_t st) {
  const cudaError_t e = cudaFuncSetAttribute(aw_split_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             AwShape<DP>::SMEM);
  if (e != cudaSuccess) {
    set_error("aw_split_kernel: %s", cudaGetErrorString(e));
    return IM_CUDA_ERROR;
  }
  return launch("aw_split_kernel", aw_split_kernel<T, DP>, grid, dim3(AW_THREADS), AwShape<DP>::SMEM, st, a);
}

template <typename T>
int launch_attention_weights(const AwArgs& a, int64_t B, cudaStream_t st) {
  const dim3 grid((unsigned)a.splits, (unsigned)(a.hkv * a.tiles), (unsigned)B);
  const int rc = a.d <= 64    ? launch_split<T, 64>(a, grid, st)
                 : a.d <= 96  ? launch_split<T, 96>(a, grid, st)
                 : a.d <= 128 ? launch_split<T, 128>(a, grid, st)
                              : launch_split<T, 256>(a, grid, st);
  if (rc != IM_OK) return rc;
  const int chunks = (a.max_kv + AW_FIN_SLOTS - 1) / AW_FIN_SLOTS;
  const size_t join = (size_t)AW_FIN_THREADS / 32 * a.d * 4, sums = sizeof(float2) * a.vecs;
  return launch("aw_finish_kernel", aw_finish_kernel<T>, dim3((unsigned)(a.vecs + chunks), (unsigned)a.hkv, (unsigned)B),
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
  IM_REQUIRE(q && k_cache && v_cache && page_table && seq_rows && row_slot && weights && weights_out && out, IM_INVALID,
             "im_attention_weights: null pointer");
  IM_REQUIRE(aligned(q, 16) && aligned(k_cache, 16) && aligned(v_cache, 16) && aligned(out, 16), IM_INVALID,
             "im_attention_weights: q, the caches and out must be 16-byte aligned");
  IM_REQUIRE(M < (1ll << 31) && B < 65536 && Hkv <= 4096 && max_rows_per_seq <= 4096 && Hq / Hkv <= 256 &&
                 max_rows_per_seq * (Hq / Hkv) <= 4096 && max_kv_len < (1ll << 30) && window < (1ll << 30),
             IM_UNSUPPORTED, "im_attention_weights: too large");
  const int64_t kv = max_kv_len > 0 ? max_kv_len : 1;
  const size_t need = im_attention_weights_workspace_bytes(B, max_rows_per_seq, Hq, Hkv, D, kv, keys_per_split, window);
  IM_REQUIRE(workspace && aligned(workspace, 256) && workspace_bytes >= need, IM_INVALID,
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
  a.kps = p.kps, a.splits = p.splits, a.tiles = p.tiles, a.vecs = (int)p.vecs;
  a.wide_weights = aligned(weights, 16) && aligned(weights_out, 16);
  a.scores = (float*)workspace;
  a.stats = (float2*)((char*)workspace + p.scores);
  a.parts = (float*)((char*)workspace + p.scores + p.stats);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return dtype == IM_BF16 ? launch_attention_weights<__nv_bfloat16>(a, B, st) : launch_attention_weights<__half>(a, B, st);
}
