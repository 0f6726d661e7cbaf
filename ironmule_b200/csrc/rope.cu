// Rotary positions: rows turned to their positions (or back), and the serving form that also writes the paged cache.
//
// A pair (a, b) of frequency f at position p turns by t = p f: a' = c a - s b, b' = s a + c b with c = factor cos t,
// s = factor sin t. Pairs are (i, i + R/2) (half) or (2i, 2i + 1) (interleaved) of a head's first R values; the rest is
// copied. The angle is a float64 product reduced to a quarter turn before it is rounded to float32: at position 10^6 a
// float32 product would be off by 0.06 rad. The product and 2 / pi are rounded, within 2^-51 of the angle together, and what is
// left of a turn within 2^-26 quarter turns: up to angles of 2^25 rad c and s are float32 exact to an ulp or two, beyond
// that they lose what the float64 angle has lost (2^-11 rad at 2^40). Rotations are float32, rounded once to the rows' type.
//
// Bound: HBM, every value read and written once. A warp takes a part of a row's heads, for itself: it works the row's c and
// s out (R/2 of them, two or so a lane), hands them over in shared memory of its own, and walks the heads; a lane keeps to
// one run of pairs, whose c and s it holds in registers. Nothing waits for another warp, so some load while others work:
// 8192 rows of 48 heads of 128 take 35 us (0.88 of the copy rate), with a block a row and a barrier behind c and s 50.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace im {

constexpr int RP_WARPS = 8;  // of a block, where their c and s fit 48 KB
constexpr int RP_HEADS = 3;  // heads that a lane has on their way

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
  int parts, heads_per_part;  // of a row's heads, a warp each
  int lanes;                  // units of a row that lie side by side in a warp
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

// Values as float32 and back, singly and two at a time (one conversion instruction for two 16-bit values).
template <typename T>
struct RopeType;
template <>
struct RopeType<__nv_bfloat16> {
  static __device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 down(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ float2 up2(const __nv_bfloat16* v) {
    return __bfloat1622float2(*(const __nv_bfloat162*)v);
  }
  static __device__ __forceinline__ void down2(__nv_bfloat16* v, float x, float y) {
    *(__nv_bfloat162*)v = __floats2bfloat162_rn(x, y);
  }
};
template <>
struct RopeType<__half> {
  static __device__ __forceinline__ float up(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half down(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ float2 up2(const __half* v) { return __half22float2(*(const __half2*)v); }
  static __device__ __forceinline__ void down2(__half* v, float x, float y) { *(__half2*)v = __floats2half2_rn(x, y); }
};
template <>
struct RopeType<float> {
  static __device__ __forceinline__ float up(float v) { return v; }
  static __device__ __forceinline__ float down(float v) { return v; }
  static __device__ __forceinline__ float2 up2(const float* v) { return make_float2(v[0], v[1]); }
  static __device__ __forceinline__ void down2(float* v, float x, float y) { v[0] = x, v[1] = y; }
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

// A unit is VEC values: neighbouring pairs (interleaved), or the first halves of VEC pairs with the second halves `pairs`
// further on; VEC 1 is one pair, wherever its values lie.
template <typename T, int VEC, bool KV>
__global__ void __launch_bounds__(RP_WARPS * 32) rope_kernel(RopeArgs a) {
  typedef RopeVec<T, VEC> V;
  extern __shared__ float2 turns_of[];  // [warps][R / 2]
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long id = (long long)blockIdx.x * (blockDim.x / 32) + warp, m = id / a.parts;
  if (m >= a.rows) return;
  const int h0 = (int)(id - m * a.parts) * a.heads_per_part, h1 = min(a.heads, h0 + a.heads_per_part);
  const int pairs = a.rotary / 2;
  float2* turn = turns_of + warp * pairs;
  const bool near = a.interleaved;
  const int units = near && VEC > 1 ? a.rotary / VEC : pairs / VEC;
  // this lane's first unit and head: a.lanes units side by side, as many heads as fit
  const int groups = 32 / a.lanes, g = lane / a.lanes;
  int u = lane - g * a.lanes;
  const int h_first = h0 + g;
  const bool works = g < groups && units > 0;
  const T* src = (const T*)a.x + m * a.x_row;
  V v[RP_HEADS], w[RP_HEADS];
  auto load = [&](int h) {
#pragma unroll
    for (int i = 0; i < RP_HEADS; i++) {
      if (h + i * groups < h1) {
        const T* p = src + (h + i * groups) * a.x_head;
        if constexpr (VEC > 1) {
          v[i] = *(const V*)(p + u * VEC);
          if (!near) w[i] = *(const V*)(p + u * VEC + pairs);
        } else {
          v[i].v[0] = p[near ? 2 * u : u];
          w[i].v[0] = p[near ? 2 * u + 1 : u + pairs];
        }
      }
    }
  };
  if (works) load(h_first);
  const double p = a.pos64 ? (double)((const long long*)a.pos)[m] : (double)((const int*)a.pos)[m];
  // where the row's key and value of head 0 go; a row without a slot of the cache is turned, and written nowhere
  long long cache = -1;
  if (KV) {
    const long long slot = a.row_slot[m], seq = a.row_seq[m];
    if (slot >= 0 && slot < a.max_pages * 16 && seq >= 0 && seq < a.seqs) {
      const long long page = a.page_table[seq * a.max_pages + slot / 16];
      if (page >= 0 && page < a.pages) cache = (page * a.hkv * 16 + slot % 16) * a.d;
    }
    if (a.slot_pos && cache >= 0 && slot < a.cap && h0 == 0)
      for (int h = lane; h < a.hkv; h += 32) a.slot_pos[(seq * a.hkv + h) * a.cap + slot] = ((const int*)a.pos)[m];
  }
  // where head h goes (nullptr: nowhere), and whether it is turned
  auto place = [&](int h, bool& turns) -> T* {
    turns = true;
    if (!KV || h < a.hq) return (T*)a.out + m * a.o_row + h * a.o_head;
    turns = h < a.hq + a.hkv;
    if (cache < 0) return nullptr;
    return (T*)(turns ? a.k_cache : a.v_cache) + cache + (long long)(h - a.hq - (turns ? 0 : a.hkv)) * 16 * a.d;
  };
  // what is copied as it is, while the first heads are on their way
  const int rest = (a.d - a.rotary) / VEC;
#pragma unroll 4
  for (int idx = lane; idx < (h1 - h0) * rest; idx += 32) {
    const int head = idx / rest, at = a.rotary + (idx - head * rest) * VEC;
    bool turns;
    T* dst = place(h0 + head, turns);
    if (dst) *(V*)(dst + at) = *(const V*)(src + (h0 + head) * a.x_head + at);
  }
  for (int i = lane; i < pairs; i += 32) {
    const double f = a.freq64 ? ((const double*)a.freq)[i] : (double)((const float*)a.freq)[i];
    turn[i] = rope_turn(p, f, (float)a.factor, a.inverse != 0);
  }
  __syncwarp();
  if (works) {
    for (bool loaded = true; u < units; u += a.lanes) {
      float c[VEC], s[VEC];  // of VEC pairs; of half as many where they lie side by side
      const float2* from = turn + (near && VEC > 1 ? u * VEC / 2 : u * VEC);
#pragma unroll
      for (int e = 0; e < VEC; e++) {
        if (e < (VEC + 1) / 2 || !near) {
          const float2 x = from[e];
          c[e] = x.x, s[e] = x.y;
        }
      }
      for (int h = h_first; h < h1; h += RP_HEADS * groups, loaded = false) {
        if (!loaded) load(h);
#pragma unroll
        for (int i = 0; i < RP_HEADS; i++) {
          if (h + i * groups >= h1) continue;
          bool turns;
          T* dst = place(h + i * groups, turns);
          if (!dst) continue;
          if constexpr (VEC > 1) {
            if (near) {
              if (turns) {
#pragma unroll
                for (int e = 0; e < VEC; e += 2) {
                  const float2 x = RopeType<T>::up2(v[i].v + e);
                  RopeType<T>::down2(v[i].v + e, fmaf(x.x, c[e / 2], -(x.y * s[e / 2])),
                                     fmaf(x.x, s[e / 2], x.y * c[e / 2]));
                }
              }
              *(V*)(dst + u * VEC) = v[i];
              continue;
            }
            if (turns) {
#pragma unroll
              for (int e = 0; e < VEC; e += 2) {
                const float2 x = RopeType<T>::up2(v[i].v + e), y = RopeType<T>::up2(w[i].v + e);
                RopeType<T>::down2(v[i].v + e, fmaf(x.x, c[e], -(y.x * s[e])), fmaf(x.y, c[e + 1], -(y.y * s[e + 1])));
                RopeType<T>::down2(w[i].v + e, fmaf(x.x, s[e], y.x * c[e]), fmaf(x.y, s[e + 1], y.y * c[e + 1]));
              }
            }
          } else if (turns) {
            const float x = RopeType<T>::up(v[i].v[0]), y = RopeType<T>::up(w[i].v[0]);
            v[i].v[0] = RopeType<T>::down(fmaf(x, c[0], -(y * s[0])));
            w[i].v[0] = RopeType<T>::down(fmaf(x, s[0], y * c[0]));
          }
          if constexpr (VEC > 1) {
            *(V*)(dst + u * VEC) = v[i];
            *(V*)(dst + u * VEC + pairs) = w[i];
          } else {
            dst[near ? 2 * u : u] = v[i].v[0];
            dst[near ? 2 * u + 1 : u + pairs] = w[i].v[0];
          }
        }
      }
      loaded = false;
    }
  }
}

template <typename T, bool KV>
int launch_rope(RopeArgs& a, long long M, int n, cudaStream_t st) {
  constexpr int WIDE = 16 / sizeof(T);
  const int pairs = a.rotary / 2;
  const int units = n > 1 && a.interleaved ? a.rotary / n : pairs / n;
  a.lanes = units < 1 ? 1 : units < 32 ? units : 32;
  // parts of a row: so many that the device has three rounds of warps, as long as a part is a load of every lane
  const int least = RP_HEADS * (32 / a.lanes);
  int parts = 1;
  while (M * parts < 148 * 32 * 3 && a.heads >= parts * 2 * least) parts *= 2;
  a.rows = M, a.heads_per_part = (a.heads + parts - 1) / parts;
  a.parts = (a.heads + a.heads_per_part - 1) / a.heads_per_part;
  int warps = RP_WARPS;
  while (warps * pairs * sizeof(float2) > 48 * 1024) warps /= 2;
  const long long blocks = (M * a.parts + warps - 1) / warps;
  IM_REQUIRE(blocks < (1ll << 31), IM_UNSUPPORTED, "rope_kernel: too many rows");
  const size_t smem = warps * pairs * sizeof(float2);
  const dim3 grid((unsigned)blocks), block(warps * 32);
  if (n == WIDE) return launch("rope_kernel", rope_kernel<T, WIDE, KV>, grid, block, smem, st, a);
  if (n == 4) return launch("rope_kernel", rope_kernel<T, 4, KV>, grid, block, smem, st, a);
  return launch("rope_kernel", rope_kernel<T, 1, KV>, grid, block, smem, st, a);
}

template <bool KV>
int launch_rope_type(RopeArgs& a, int dtype, long long M, int n, cudaStream_t st) {
  if (dtype == IM_BF16) return launch_rope<__nv_bfloat16, KV>(a, M, n, st);
  if (dtype == IM_F16) return launch_rope<__half, KV>(a, M, n, st);
  return launch_rope<float, KV>(a, M, n, st);
}

// The widest access that fits, in values: 16 bytes, 8 (16-bit types whose turned part is an odd number of them), or one value.
// Bases (k and v: the caches', or NULL) and strides, head and turned part have to be whole. 4096 rows of 32 heads of 144
// bf16 values, 72 turned in halves: 23.8 us with 8 bytes, 50.0 with one value.
static int rope_wide(const RopeArgs& a, int size, const void* k, const void* v) {
  const int run = a.interleaved ? a.rotary : a.rotary / 2;
  for (int bytes = 16; bytes >= 8; bytes /= 2) {
    const int n = bytes / size;
    if (n >= 4 && aligned(a.x, bytes) && aligned(a.out, bytes) && aligned(k, bytes) && aligned(v, bytes) && a.x_row % n == 0 &&
        a.x_head % n == 0 && a.o_row % n == 0 && a.o_head % n == 0 && a.d % n == 0 && run % n == 0)
      return n;
  }
  return 1;
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
  return launch_rope_type<false>(a, dtype, M, rope_wide(a, size, nullptr, nullptr), reinterpret_cast<cudaStream_t>(stream));
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
  return launch_rope_type<true>(a, dtype, M, rope_wide(a, size, k_cache, v_cache), reinterpret_cast<cudaStream_t>(stream));
}
