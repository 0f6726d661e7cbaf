// Rotary positions: rows turned to their positions (or back), and the serving form that also writes the paged cache.
//
// A pair (a, b) of frequency f at position p turns by t = p f: a' = c a - s b, b' = s a + c b with c = factor cos t,
// s = factor sin t. Pairs are (i, i + R/2) (half) or (2i, 2i + 1) (interleaved) of a head's first R values; the rest is
// copied. The angle is a float64 product reduced to a quarter turn before it is rounded to float32: at position 10^6 a
// float32 product would be off by 0.06 rad. What is left of it is within 2^-26 quarter turns, so c and s are float32
// exact to an ulp or two wherever the position is. Rotations are float32, rounded once to the rows' type.
//
// Bound: HBM, every value read and written once. A block takes a row (a part of one where rows are few, several where they
// are short), works c and s out once (R/2 of them a row) and uses them for every head from shared memory; the first values
// are on their way meanwhile. Values move 16 bytes a thread.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace im {

constexpr int RP_THREADS = 256;
constexpr int RP_ROWS = 16;   // rows a block at most
constexpr int RP_BATCH = 2;   // units a thread has on their way

struct RopeArgs {
  const char* x;            // rows
  long long x_row, x_head;  // strides in values
  const void* pos;
  const void* freq;
  int pos64, freq64;
  double factor;
  int inverse, interleaved;
  int rotary, d;
  int heads;           // heads of a row that the launch walks (rope_kv: q, k and v heads)
  int heads_per_block;
  int rows_per_block;
  long long rows;
  char* out;
  long long o_row, o_head;
  // the serving form
  int hq, hkv;
  const int* row_slot;
  const int* row_seq;
  const int* page_table;
  long long seqs, max_pages, pages;
  char* k_cache;
  char* v_cache;
  int* slot_pos;
  long long cap;
};

template <typename T>
struct RopeType;
template <>
struct RopeType<__nv_bfloat16> {
  static __device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 down(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct RopeType<__half> {
  static __device__ __forceinline__ float up(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half down(float v) { return __float2half_rn(v); }
};
template <>
struct RopeType<float> {
  static __device__ __forceinline__ float up(float v) { return v; }
  static __device__ __forceinline__ float down(float v) { return v; }
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) RopeVec {
  T v[VEC];
};

// c and s of pair i at position p.
__device__ __forceinline__ float2 rope_turn(double p, double f, float factor, bool inverse) {
  const double quarters = p * f * 0.63661977236758134308;  // 2 / pi
  const double whole = rint(quarters);
  const float rest = (float)(quarters - whole);  // within half a quarter turn
  float s, c;
  sincospif(0.5f * rest, &s, &c);
  const int q = (int)((long long)whole & 3);
  if (q & 1) {
    const float t = c;
    c = -s;
    s = t;
  }
  if (q & 2) {
    c = -c;
    s = -s;
  }
  if (inverse) s = -s;
  return make_float2(factor * c, factor * s);
}

// One block: `heads_per_block` heads of `rows_per_block` rows. VEC values a load; a unit is two loads of a half-layout pair
// of runs, or one load of neighbouring pairs, or one load of the part that is copied (VEC 1: one pair, or one value).
template <typename T, int VEC, bool KV>
__global__ void __launch_bounds__(RP_THREADS) rope_kernel(RopeArgs a) {
  typedef RopeVec<T, VEC> V;
  extern __shared__ float2 turn[];       // [rows][R / 2]
  __shared__ long long s_cache[RP_ROWS];  // where a row's keys and values go: head 0's, in values; -1: nowhere
  pdl_wait();
  pdl_trigger();
  const int t = threadIdx.x;
  const long long m0 = (long long)blockIdx.x * a.rows_per_block;
  const int rows = (int)min((long long)a.rows_per_block, a.rows - m0);
  const int h0 = blockIdx.y * a.heads_per_block, heads = min(a.heads, h0 + a.heads_per_block) - h0;
  const int pairs = a.rotary / 2;
  const int turned = a.interleaved && VEC > 1 ? a.rotary / VEC : pairs / VEC;
  const int units = turned + (a.d - a.rotary) / VEC, row_units = heads * units;
  const int total = rows * row_units;
  // exact for numbers under 2^22
  const float per_row = 1.f / row_units, per_head = 1.f / units;
  auto place = [&](int idx, int& r, int& h, int& u) {
    r = (int)((idx + 0.5f) * per_row);
    const int rest = idx - r * row_units;
    h = (int)((rest + 0.5f) * per_head);
    u = rest - h * units;
    h += h0;
  };
  V v[RP_BATCH], w[RP_BATCH];
  auto load = [&](int idx0) {
    if constexpr (VEC > 1) {  // single values are read where they are turned
#pragma unroll
      for (int i = 0; i < RP_BATCH; i++) {
        const int idx = idx0 + i * RP_THREADS;
        if (idx < total) {
          int r, h, u;
          place(idx, r, h, u);
          const T* src = (const T*)a.x + (m0 + r) * a.x_row + h * a.x_head;
          if (u >= turned) {
            v[i] = *(const V*)(src + a.rotary + (u - turned) * VEC);
          } else {
            v[i] = *(const V*)(src + u * VEC);
            if (!a.interleaved) w[i] = *(const V*)(src + u * VEC + pairs);
          }
        }
      }
    }
  };
  load(t);
  for (int i = t; i < rows * pairs; i += RP_THREADS) {
    const int r = i / pairs, pair = i - r * pairs;
    const double p = a.pos64 ? (double)((const long long*)a.pos)[m0 + r] : (double)((const int*)a.pos)[m0 + r];
    const double f = a.freq64 ? ((const double*)a.freq)[pair] : (double)((const float*)a.freq)[pair];
    turn[i] = rope_turn(p, f, (float)a.factor, a.inverse != 0);
  }
  if (KV && t < rows) {  // rows without a slot of the cache are turned, and written nowhere
    const long long slot = a.row_slot[m0 + t], seq = a.row_seq[m0 + t];
    long long at = -1;
    if (slot >= 0 && slot < a.max_pages * 16 && seq >= 0 && seq < a.seqs) {
      const long long page = a.page_table[seq * a.max_pages + slot / 16];
      if (page >= 0 && page < a.pages) at = (page * a.hkv * 16 + slot % 16) * a.d;
    }
    s_cache[t] = at;
    if (a.slot_pos && at >= 0 && slot < a.cap && blockIdx.y == 0) {
      const int pos = ((const int*)a.pos)[m0 + t];
      for (int h = 0; h < a.hkv; h++) a.slot_pos[(seq * a.hkv + h) * a.cap + slot] = pos;
    }
  }
  __syncthreads();
  for (int idx0 = t; idx0 < total; idx0 += RP_BATCH * RP_THREADS) {
    if (idx0 != t) load(idx0);
#pragma unroll
    for (int i = 0; i < RP_BATCH; i++) {
      const int idx = idx0 + i * RP_THREADS;
      if (idx >= total) continue;
      int r, h, u;
      place(idx, r, h, u);
      T* dst;
      bool turns = true;
      if (!KV || h < a.hq) {
        dst = (T*)a.out + (m0 + r) * a.o_row + h * a.o_head;
      } else {
        turns = h < a.hq + a.hkv;
        if (s_cache[r] < 0) continue;
        dst = (T*)(turns ? a.k_cache : a.v_cache) + s_cache[r] + (long long)(turns ? h - a.hq : h - a.hq - a.hkv) * 16 * a.d;
      }
      const float2* c = turn + r * pairs;
      if (VEC == 1) {
        const T* src = (const T*)a.x + (m0 + r) * a.x_row + h * a.x_head;
        if (u >= turned) {
          dst[a.rotary + u - turned] = src[a.rotary + u - turned];
          continue;
        }
        const int at = a.interleaved ? 2 * u : u, to = a.interleaved ? at + 1 : at + pairs;
        const T x = src[at], y = src[to];
        if (turns) {
          const float fx = RopeType<T>::up(x), fy = RopeType<T>::up(y);
          dst[at] = RopeType<T>::down(fmaf(fx, c[u].x, -(fy * c[u].y)));
          dst[to] = RopeType<T>::down(fmaf(fx, c[u].y, fy * c[u].x));
        } else {
          dst[at] = x;
          dst[to] = y;
        }
      } else if (u >= turned) {
        *(V*)(dst + a.rotary + (u - turned) * VEC) = v[i];
      } else if (a.interleaved) {
        if (turns) {
#pragma unroll
          for (int e = 0; e + 1 < VEC; e += 2) {
            const float2 k = c[(u * VEC + e) / 2];
            const float x = RopeType<T>::up(v[i].v[e]), y = RopeType<T>::up(v[i].v[e + 1]);
            v[i].v[e] = RopeType<T>::down(fmaf(x, k.x, -(y * k.y)));
            v[i].v[e + 1] = RopeType<T>::down(fmaf(x, k.y, y * k.x));
          }
        }
        *(V*)(dst + u * VEC) = v[i];
      } else {
        if (turns) {
#pragma unroll
          for (int e = 0; e < VEC; e++) {
            const float2 k = c[u * VEC + e];
            const float x = RopeType<T>::up(v[i].v[e]), y = RopeType<T>::up(w[i].v[e]);
            v[i].v[e] = RopeType<T>::down(fmaf(x, k.x, -(y * k.y)));
            w[i].v[e] = RopeType<T>::down(fmaf(x, k.y, y * k.x));
          }
        }
        *(V*)(dst + u * VEC) = v[i];
        *(V*)(dst + u * VEC + pairs) = w[i];
      }
    }
  }
}

template <typename T, bool KV>
int launch_rope(RopeArgs& a, long long M, bool vec, cudaStream_t st) {
  constexpr int WIDE = 16 / sizeof(T);
  const int n = vec ? WIDE : 1;
  const int units = (a.interleaved && vec ? a.rotary / n : a.rotary / 2 / n) + (a.d - a.rotary) / n;
  // few rows: their heads are spread over several blocks, so that one row's are not one block's latency; many:
  // several a block, so that every thread works out a pair's c and s
  int blocks_y = 1, rows = 1;
  while (M * blocks_y < 148 && blocks_y * 4 < a.heads) blocks_y *= 2;
  while (rows < RP_ROWS && rows * 2 * (a.rotary / 2) <= RP_THREADS && M >= rows * 2 * 592) rows *= 2;
  a.rows = M, a.rows_per_block = rows;
  a.heads_per_block = (a.heads + blocks_y - 1) / blocks_y;
  blocks_y = (a.heads + a.heads_per_block - 1) / a.heads_per_block;
  const dim3 grid((unsigned)((M + rows - 1) / rows), (unsigned)blocks_y);
  const size_t smem = sizeof(float2) * rows * (a.rotary / 2);
  if (vec) return launch("rope_kernel", rope_kernel<T, WIDE, KV>, grid, dim3(RP_THREADS), smem, st, a);
  return launch("rope_kernel", rope_kernel<T, 1, KV>, grid, dim3(RP_THREADS), smem, st, a);
}

template <bool KV>
int launch_rope_type(RopeArgs& a, int dtype, long long M, bool vec, cudaStream_t st) {
  if (dtype == IM_BF16) return launch_rope<__nv_bfloat16, KV>(a, M, vec, st);
  if (dtype == IM_F16) return launch_rope<__half, KV>(a, M, vec, st);
  return launch_rope<float, KV>(a, M, vec, st);
}

// Whether 16-byte accesses fit: each base 16-byte aligned, strides, head and the turned part whole vectors.
static bool rope_wide(const RopeArgs& a, int size) {
  const int n = 16 / size;
  const int run = a.interleaved ? a.rotary : a.rotary / 2;
  return aligned(a.x, 16) && aligned(a.out, 16) && a.x_row % n == 0 && a.x_head % n == 0 && a.o_row % n == 0 &&
         a.o_head % n == 0 && a.d % n == 0 && run % n == 0;
}

}  // namespace im

using namespace im;

extern "C" int im_rope(const void* x, int64_t row_stride, int64_t head_stride, const void* pos, int pos_64,
                       const void* inv_freq, int freq_f64, int64_t rotary, double factor, int layout, int inverse,
                       int64_t M, int64_t H, int64_t D, int dtype, void* out, int64_t out_row_stride,
                       int64_t out_head_stride, void* stream) {
  clear_error();
  IM_REQUIRE(M >= 0 && H >= 0 && D >= 1 && rotary >= 0, IM_INVALID, "im_rope: bad sizes");
  IM_REQUIRE(layout == IM_ROPE_HALF || layout == IM_ROPE_INTERLEAVED, IM_INVALID, "im_rope: layout %d", layout);
  IM_REQUIRE(dtype >= IM_BF16 && dtype <= IM_F32, IM_INVALID, "im_rope: type %d", dtype);
  IM_REQUIRE(rotary % 2 == 0 && rotary <= D, IM_INVALID, "im_rope: %lld of %lld values turn", (long long)rotary,
             (long long)D);
  if (M == 0 || H == 0) return IM_OK;
  IM_REQUIRE(x && pos && out && (inv_freq || rotary == 0), IM_INVALID, "im_rope: null pointer");
  IM_REQUIRE(M < (1ll << 31) && D <= 4096 && H * D < (1 << 20), IM_UNSUPPORTED,
             "im_rope: rows of %lld heads of %lld (under 2^20 values, heads up to 4096)", (long long)H, (long long)D);
  const int size = dtype == IM_F32 ? 4 : 2;
  IM_REQUIRE(aligned(x, size) && aligned(out, size) && aligned(pos, pos_64 ? 8 : 4) && aligned(inv_freq, freq_f64 ? 8 : 4),
             IM_INVALID, "im_rope: misaligned pointer");
  RopeArgs a = {};
  a.x = (const char*)x, a.x_row = row_stride, a.x_head = head_stride;
  a.pos = pos, a.pos64 = pos_64, a.freq = inv_freq, a.freq64 = freq_f64, a.factor = factor;
  a.inverse = inverse, a.interleaved = layout == IM_ROPE_INTERLEAVED, a.rotary = (int)rotary, a.d = (int)D;
  a.heads = (int)H;
  a.out = (char*)out, a.o_row = out_row_stride, a.o_head = out_head_stride;
  return launch_rope_type<false>(a, dtype, M, rope_wide(a, size), reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int im_rope_kv(const void* qkv, const void* inv_freq, int freq_f64, int64_t rotary, double factor, int layout,
                          const int32_t* row_pos, const int32_t* row_slot, const int32_t* row_seq,
                          const int32_t* page_table, int64_t seqs, int64_t max_pages, int64_t pages, int64_t M,
                          int64_t Hq, int64_t Hkv, int64_t D, int dtype, void* q_out, void* k_cache, void* v_cache,
                          int32_t* slot_pos, int64_t cap, void* stream) {
  clear_error();
  IM_REQUIRE(M >= 0 && Hq >= 1 && Hkv >= 1 && Hq % Hkv == 0 && D >= 1 && rotary >= 0 && seqs >= 0 && max_pages >= 0 &&
                 pages >= 0 && cap >= 0,
             IM_INVALID, "im_rope_kv: bad sizes");
  IM_REQUIRE(layout == IM_ROPE_HALF || layout == IM_ROPE_INTERLEAVED, IM_INVALID, "im_rope_kv: layout %d", layout);
  IM_REQUIRE(dtype >= IM_BF16 && dtype <= IM_F32, IM_INVALID, "im_rope_kv: type %d", dtype);
  IM_REQUIRE(rotary % 2 == 0 && rotary <= D, IM_INVALID, "im_rope_kv: %lld of %lld values turn", (long long)rotary,
             (long long)D);
  if (M == 0) return IM_OK;
  IM_REQUIRE(qkv && row_pos && row_slot && row_seq && page_table && q_out && k_cache && v_cache &&
                 (inv_freq || rotary == 0),
             IM_INVALID, "im_rope_kv: null pointer");
  IM_REQUIRE(M < (1ll << 31) && D <= 4096 && (Hq + 2 * Hkv) * D < (1 << 20), IM_UNSUPPORTED,
             "im_rope_kv: rows of %lld values (under 2^20, heads up to 4096)", (long long)((Hq + 2 * Hkv) * D));
  const int size = dtype == IM_F32 ? 4 : 2;
  IM_REQUIRE(aligned(qkv, size) && aligned(q_out, size) && aligned(k_cache, size) && aligned(v_cache, size) &&
                 aligned(inv_freq, freq_f64 ? 8 : 4) && aligned(row_pos, 4) && aligned(row_slot, 4) &&
                 aligned(row_seq, 4) && aligned(page_table, 4) && aligned(slot_pos, 4),
             IM_INVALID, "im_rope_kv: misaligned pointer");
  RopeArgs a = {};
  a.x = (const char*)qkv, a.x_row = (Hq + 2 * Hkv) * D, a.x_head = D;
  a.pos = row_pos, a.freq = inv_freq, a.freq64 = freq_f64, a.factor = factor;
  a.interleaved = layout == IM_ROPE_INTERLEAVED, a.rotary = (int)rotary, a.d = (int)D;
  a.heads = (int)(Hq + 2 * Hkv);
  a.out = (char*)q_out, a.o_row = Hq * D, a.o_head = D;
  a.hq = (int)Hq, a.hkv = (int)Hkv, a.row_slot = row_slot, a.row_seq = row_seq, a.page_table = page_table;
  a.seqs = seqs, a.max_pages = max_pages, a.pages = pages;
  a.k_cache = (char*)k_cache, a.v_cache = (char*)v_cache, a.slot_pos = slot_pos, a.cap = cap;
  const bool vec = rope_wide(a, size) && aligned(k_cache, 16) && aligned(v_cache, 16);
  return launch_rope_type<true>(a, dtype, M, vec, reinterpret_cast<cudaStream_t>(stream));
}
