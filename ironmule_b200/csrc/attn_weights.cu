// Attention of a few new rows a sequence over the paged cache, which also adds up every slot's attention weight.
//
//   s[r, g, j] = scale q[r, g] . k[j] for the slots j that row r sees, p = softmax over j, out = sum_j p v[j]
//   weights'[h, j] = (j before the sequence's first new slot ? weights[h, j] : 0) + sum over rows r and the query heads
//   g of kv head h of p[r, g, j]
//
// First kernel: one block a (row, query head); scores to the workspace, their maximum and sum, the output. Second kernel:
// a thread a slot, which adds up exp(s - max) / sum over the rows and heads.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace im {

constexpr int AW_THREADS = 256;

struct AwArgs {
  const void* q;
  const void* k;
  const void* v;
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
  void* out;
  float* scores;  // [B][Hkv][max_rows * G][kv_pad], in log2 units
  float2* stats;  // [B][Hkv][max_rows * G]: maximum and 1 / sum
};

__device__ __forceinline__ float aw_value(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float aw_value(__half v) { return __half2float(v); }

// The rows of sequence b: first row, and how many of them the call computes.
__device__ __forceinline__ int2 aw_rows(const AwArgs& a, int b) {
  const int r0 = min(max(a.seq_rows[b], 0), a.M), r1 = min(a.seq_rows[b + 1], a.M);
  return make_int2(r0, max(0, min(r1 - r0, a.max_rows)));
}

// The page-table row of sequence b (-1: none).
__device__ __forceinline__ long long aw_slot(const AwArgs& a, int b) {
  const long long s = a.seq_slot ? a.seq_slot[b] : b;
  return s >= 0 && s < a.seqs ? s : -1;
}

template <typename T>
__global__ void __launch_bounds__(AW_THREADS) aw_plain_kernel(AwArgs a) {
  __shared__ float red[AW_THREADS];
  extern __shared__ float acc[];
  pdl_wait();
  pdl_trigger();
  const int b = blockIdx.z, r = blockIdx.y, hq = blockIdx.x, t = threadIdx.x;
  const int group = a.hq / a.hkv, h = hq / group, vec = r * group + hq % group;
  const int2 rows = aw_rows(a, b);
  if (r >= rows.y) return;
  const long long row = rows.x + r, slot_row = aw_slot(a, b);
  const int last = slot_row < 0 ? -1 : (int)min((long long)a.row_slot[row], min((long long)a.max_kv, a.max_pages * 16) - 1);
  const int from = a.window > 0 ? max(0, a.row_slot[row] - a.window + 1) : 0;
  const long long at = ((long long)b * a.hkv + h) * a.max_rows * group + vec;
  float* s_out = a.scores + at * a.kv_pad;
  const T* q = (const T*)a.q + (row * a.hq + hq) * a.d;
  float top = -INFINITY;
  for (int j = from + t; j <= last; j += AW_THREADS) {
    const long long page = a.page_table[slot_row * a.max_pages + j / 16];
    float s = -INFINITY;
    if (page >= 0 && page < a.pages) {
      const T* k = (const T*)a.k + ((page * a.hkv + h) * 16 + j % 16) * a.d;
      s = 0.f;
      for (int i = 0; i < a.d; i++) s = fmaf(aw_value(q[i]), aw_value(k[i]), s);
      s *= a.scale;
    }
    s_out[j] = s;
    top = fmaxf(top, s);
  }
  red[t] = top;
  __syncthreads();
  for (int o = AW_THREADS / 2; o > 0; o >>= 1) {
    if (t < o) red[t] = fmaxf(red[t], red[t + o]);
    __syncthreads();
  }
  top = red[0] > -INFINITY ? red[0] : 0.f;
  __syncthreads();
  float sum = 0.f;
  for (int j = from + t; j <= last; j += AW_THREADS) sum += expf(s_out[j] - top);
  red[t] = sum;
  __syncthreads();
  for (int o = AW_THREADS / 2; o > 0; o >>= 1) {
    if (t < o) red[t] += red[t + o];
    __syncthreads();
  }
  sum = red[0];
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (t == 0) a.stats[at] = make_float2(top, inv);
  for (int i = t; i < a.d; i += AW_THREADS) {
    float o = 0.f;
    for (int j = from; j <= last; j++) {
      const long long page = a.page_table[slot_row * a.max_pages + j / 16];
      if (page < 0 || page >= a.pages) continue;
      o = fmaf(expf(s_out[j] - top), aw_value(((const T*)a.v)[((page * a.hkv + h) * 16 + j % 16) * a.d + i]), o);
    }
    ((T*)a.out)[(row * a.hq + hq) * a.d + i] = (T)(o * inv);
  }
}

__global__ void __launch_bounds__(AW_THREADS) aw_finish_kernel(AwArgs a) {
  pdl_wait();
  pdl_trigger();
  const int b = blockIdx.z, h = blockIdx.y;
  const int2 rows = aw_rows(a, b);
  const long long slot_row = aw_slot(a, b);
  if (rows.y == 0 || slot_row < 0) return;
  int n = -1;
  for (int r = 0; r < rows.y; r++) n = max(n, a.row_slot[rows.x + r]);
  n = (int)min((long long)n + 1, min(min((long long)a.max_kv, a.max_pages * 16), a.cap));
  const int first = a.row_slot[rows.x], group = a.hq / a.hkv;
  const long long at = ((long long)b * a.hkv + h) * a.max_rows * group;
  const long long base = (slot_row * a.hkv + h) * a.cap;
  for (int j = blockIdx.x * AW_THREADS + threadIdx.x; j < n; j += gridDim.x * AW_THREADS) {
    float sum = 0.f;
    for (int r = 0; r < rows.y; r++) {
      const int slot = a.row_slot[rows.x + r];
      if (j > slot || (a.window > 0 && j <= slot - a.window)) continue;
      for (int g = 0; g < group; g++) {
        const long long vec = at + r * group + g;
        const float2 st = a.stats[vec];
        sum += expf(a.scores[vec * a.kv_pad + j] - st.x) * st.y;
      }
    }
    a.weights_out[base + j] = (j < first ? a.weights[base + j] : 0.f) + sum;
  }
}

static int aw_pad(int64_t max_kv_len) { return (int)((max_kv_len + 63) / 64 * 64); }

}  // namespace im

using namespace im;

extern "C" size_t im_attention_weights_workspace_bytes(int64_t B, int64_t max_rows_per_seq, int64_t Hq, int64_t Hkv,
                                                       int64_t D, int64_t max_kv_len, int64_t keys_per_split) {
  if (B < 1 || max_rows_per_seq < 1 || Hkv < 1 || Hq < 1 || Hq % Hkv || D < 16 || max_kv_len < 1 || keys_per_split < 0)
    return 0;
  const size_t vecs = (size_t)B * Hq * max_rows_per_seq;
  return vecs * aw_pad(max_kv_len) * 4 + vecs * 8;
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
  IM_REQUIRE(M < (1ll << 31) && B < 65536 && Hkv < 65536 && max_rows_per_seq * Hq < (1 << 20) && max_kv_len < (1ll << 30) &&
                 window < (1ll << 30),
             IM_UNSUPPORTED, "im_attention_weights: too large");
  const int64_t kv = max_kv_len > 0 ? max_kv_len : 1;
  const size_t need = im_attention_weights_workspace_bytes(B, max_rows_per_seq, Hq, Hkv, D, kv, keys_per_split);
  IM_REQUIRE(workspace && aligned(workspace, 256) && workspace_bytes >= need, IM_INVALID,
             "im_attention_weights: a workspace of %zu bytes needed, %zu given", need, workspace_bytes);
  AwArgs a = {};
  a.q = q, a.k = k_cache, a.v = v_cache, a.page_table = page_table, a.seqs = seqs, a.max_pages = max_pages;
  a.pages = pages, a.seq_rows = seq_rows, a.seq_slot = seq_slot, a.row_slot = row_slot;
  a.weights = weights, a.weights_out = weights_out, a.cap = cap;
  a.M = (int)M, a.max_rows = (int)max_rows_per_seq, a.hq = (int)Hq, a.hkv = (int)Hkv, a.d = (int)D;
  a.max_kv = (int)max_kv_len, a.kv_pad = aw_pad(kv), a.window = (int)window, a.scale = scale, a.out = out;
  a.scores = (float*)workspace;
  a.stats = (float2*)(a.scores + (size_t)B * Hq * max_rows_per_seq * a.kv_pad);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)Hq, (unsigned)max_rows_per_seq, (unsigned)B);
  int rc = dtype == IM_BF16
               ? launch("aw_plain_kernel", aw_plain_kernel<__nv_bfloat16>, grid, dim3(AW_THREADS), 0, st, a)
               : launch("aw_plain_kernel", aw_plain_kernel<__half>, grid, dim3(AW_THREADS), 0, st, a);
  if (rc != IM_OK) return rc;
  const int64_t chunks = (max_kv_len + AW_THREADS - 1) / AW_THREADS;
  return launch("aw_finish_kernel", aw_finish_kernel,
                dim3((unsigned)(chunks < 1 ? 1 : chunks > 4096 ? 4096 : chunks), (unsigned)Hkv, (unsigned)B),
                dim3(AW_THREADS), 0, st, a);
}
