// The router of a mixture-of-experts block: per row the k experts with the largest keys and their weights, then the
// (row, place) pairs sorted by expert and cut into the work items of the grouped products.
//
// Selection is exact: the key of expert e is float32(logit) + bias[e] (one rounding; -0 counts as +0), the k largest
// keys are taken in order, ties to the lower expert. A logit or bias of -inf or NaN closes the expert to the row; a row
// with fewer than k open experts has id -1 and weight 0 in its remaining places. With IM_MOE_BIAS_ON_SCORE the key is
// the expert's float32 score plus the bias (the correction of a load-balanced router is defined so): 1 / (1 + exp(-v)),
// or the softmax over the open experts. The two orders differ, as the scores are not linear in the logits.
//   softmax: p_e = exp(v_e - max v) / sum over the chosen (normalise) or over every open expert
//   sigmoid: p_e = 1 / (1 + exp(-v_e)), over the chosen's sum when normalised. There the sums run over
//            exp(ls - max ls), ls = log sigmoid(v), so that far-negative logits do not underflow to 0 / 0.
// Weights are float32 and unbiased by `bias`.
//
// One warp per row: lane l holds experts l, l + 32, ...; each of the k rounds takes the warp's largest 32-bit sortable
// key with one reduction and the lowest expert holding it with a second (bf16 logits without a bias: key and expert in
// one word, one reduction; 8192 rows of 128 experts 18.6 us against 20.6). Up to 64 rows one block does all of it in one
// launch. More rows are cut over up to 296 blocks: the first launch selects and counts, the second sums the blocks'
// counts (every block for itself), scans them and places its pairs. The order is stable: within an expert, pairs ascend.
// Bytes are few (a row's logits once, 12 bytes a place); what bounds it is launch and barrier latency.
#include <math.h>

#include "common.cuh"
#include "moe.cuh"
#include "../../include/imspec.h"

namespace im {

constexpr int MR_WARPS = 16;
constexpr int MR_THREADS = MR_WARPS * 32;

struct RouteArgs {
  const void* logits;
  const float* bias;
  int* ids;
  float* weights;
  int* offsets;
  int* pairs;
  int* plan;
  int2* where;
  int* counts;   // [E + 1][blocks]
  int* error;    // the caller's error word, or NULL
  int f32, scoring, on_score, normalise;
  float scale;
  int M, E, top_k, rows_per_block, blocks;
  long long ld;
};

MoePlan moe_plan(int64_t M, int64_t E, int64_t top_k) {
  MoePlan p;
  const int64_t pairs = M * top_k, buckets = pairs < E + 1 ? pairs : E + 1;
  p.max_items = buckets + pairs / MOE_ITEM_ROWS;
  const int64_t per = (M + MOE_ROUTE_BLOCKS - 1) / MOE_ROUTE_BLOCKS;
  p.rows_per_block = M <= MOE_ROUTE_ROWS ? MOE_ROUTE_ROWS : (per < 16 ? 16 : per);
  p.blocks = M <= MOE_ROUTE_ROWS ? 1 : (M + p.rows_per_block - 1) / p.rows_per_block;
  p.where = MOE_PLAN_HEADER + 4 * p.max_items;
  p.counts = p.where + 2 * pairs;
  p.bytes = (size_t)(p.counts + (p.blocks > 1 ? p.blocks * (E + 1) : 0)) * 4;
  return p;
}

__device__ __forceinline__ unsigned mr_key(float f) {
  const unsigned u = __float_as_uint(f + 0.f);  // -0 -> +0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float mr_warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// The chosen experts of one row: lane j < top_k returns place j's expert (-1: none) and writes its weight.
// PACK (bf16 logits without a bias): key and expert share one word, so that a round is one reduction.
template <int EL, bool PACK>
__device__ __forceinline__ int mr_row(const RouteArgs& a, int row, int lane) {
  float v[EL];
  unsigned key[EL];
  const float neg = -INFINITY;
#pragma unroll
  for (int i = 0; i < EL; i++) {
    const int e = i * 32 + lane;
    v[i] = neg;
    key[i] = 0u;
    if (e < a.E) {
      const size_t at = (size_t)row * a.ld + e;
      const float l = a.f32 ? reinterpret_cast<const float*>(a.logits)[at]
                            : bf(reinterpret_cast<const uint16_t*>(a.logits)[at]);
      const float k = PACK || !a.bias ? l : a.on_score ? a.bias[e] : l + a.bias[e];
      if (l > neg && k > neg) {  // false for NaN too
        v[i] = l;
        key[i] = PACK ? (mr_key(k) & 0xffff0000u) | (0xffffu - e) : mr_key(k);
      }
    }
  }
  if (!PACK && a.on_score) {  // keys from the scores (held in their place meanwhile)
    float top = neg, total = 0.f;
#pragma unroll
    for (int i = 0; i < EL; i++) top = fmaxf(top, v[i]);
    top = mr_warp_max(top);
#pragma unroll
    for (int i = 0; i < EL; i++) {
      float score = 0.f;
      if (v[i] > neg)
        score = a.scoring == IM_MOE_SIGMOID ? 1.f / (1.f + expf(-v[i])) : v[i] == top ? 1.f : expf(v[i] - top);
      total += score;
      key[i] = __float_as_uint(score);
    }
    total = a.scoring == IM_MOE_SIGMOID ? 1.f : warp_sum(total);
#pragma unroll
    for (int i = 0; i < EL; i++)
      key[i] = v[i] > neg ? mr_key(__uint_as_float(key[i]) / total + a.bias[i * 32 + lane]) : 0u;
  }
  int mine = -1;
  float value = neg;
  for (int j = 0; PACK && j < a.top_k; j++) {
    unsigned best = key[0];
#pragma unroll
    for (int i = 1; i < EL; i++) best = max(best, key[i]);
    const unsigned top = __reduce_max_sync(0xffffffffu, best);
    if (top == 0u) break;  // no open expert is left (the same in every lane)
#pragma unroll
    for (int i = 0; i < EL; i++)
      if (key[i] == top) key[i] = 0u;
    if (lane == j) {
      mine = (int)(0xffffu - (top & 0xffffu));
      const unsigned hi = top >> 16;
      value = bf((uint16_t)(hi & 0x8000u ? hi ^ 0x8000u : ~hi));
    }
  }
  for (int j = 0; !PACK && j < a.top_k; j++) {
    unsigned best = 0u;
    int at = 0;
    float bv = neg;
#pragma unroll
    for (int i = 0; i < EL; i++)
      if (key[i] > best) {
        best = key[i];
        at = i;
        bv = v[i];
      }
    const unsigned top = __reduce_max_sync(0xffffffffu, best);
    if (top == 0u) break;  // no open expert is left (the same in every lane)
    const unsigned cand = best == top ? (unsigned)(at * 32 + lane) : 0xffffffffu;
    const unsigned e = __reduce_min_sync(0xffffffffu, cand);
    const float ev = __shfl_sync(0xffffffffu, bv, (int)(e & 31u));
    if (cand == e) {
#pragma unroll
      for (int i = 0; i < EL; i++)
        if (i == at) key[i] = 0u;
    }
    if (lane == j) {
      mine = (int)e;
      value = ev;
    }
  }
  // the weights
  const bool live = mine >= 0;
  float w = 0.f;
  if (a.scoring == IM_MOE_SOFTMAX) {
    // relative to the largest of the terms that are summed: a bias can choose experts far below the row's largest
    float top = neg;
    if (a.normalise) {
      top = value;
    } else {
#pragma unroll
      for (int i = 0; i < EL; i++) top = fmaxf(top, v[i]);
    }
    top = mr_warp_max(top);
    const float p = live ? (value == top ? 1.f : expf(value - top)) : 0.f;  // (inf - inf counts as 0)
    float total = p;
    if (!a.normalise) {
      total = 0.f;
#pragma unroll
      for (int i = 0; i < EL; i++) total += v[i] > neg ? (v[i] == top ? 1.f : expf(v[i] - top)) : 0.f;
    }
    total = warp_sum(total);
    w = live ? p / total : 0.f;
  } else if (a.normalise) {
    const float ls = live ? fminf(value, 0.f) - log1pf(expf(-fabsf(value))) : neg;
    const float top = mr_warp_max(ls);
    const float p = live ? expf(ls - top) : 0.f;
    const float total = warp_sum(p);
    w = live ? p / total : 0.f;
  } else {
    w = live ? 1.f / (1.f + expf(-value)) : 0.f;
  }
  if (lane < a.top_k) {
    a.ids[(size_t)row * a.top_k + lane] = mine;
    a.weights[(size_t)row * a.top_k + lane] = w * a.scale;
  }
  return mine;
}

// Exclusive scan of v[0..n) in shared memory into out[0..n) (out may be v); returns the total. All threads call it.
__device__ __forceinline__ int mr_scan(const int* v, int* out, int n, int* sh) {
  const int per = (n + MR_THREADS - 1) / MR_THREADS, lo = threadIdx.x * per;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int sum = 0;
  for (int i = lo; i < min(lo + per, n); i++) sum += v[i];
  int incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += t;
  }
  if (lane == 31) sh[warp] = incl;
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < MR_WARPS; w++) {
    if (w < warp) before += sh[w];
    total += sh[w];
  }
  int run = before + incl - sum;
  for (int i = lo; i < min(lo + per, n); i++) {
    const int t = v[i];
    out[i] = run;
    run += t;
  }
  __syncthreads();
  return total;
}

struct RouteSmem {
  int total[MOE_MAX_EXPERTS + 1];   // pairs of each bucket over all blocks
  int base[MOE_MAX_EXPERTS + 1];    // pairs of each bucket in earlier blocks, then where the next one goes
  int first[MOE_MAX_EXPERTS + 1];   // where each bucket begins
  int scan[MOE_MAX_EXPERTS + 1];    // work items before each bucket's
  int pad[MOE_MAX_EXPERTS + 1];     // rows before each bucket's when every item is rounded up to 16
  int cnt[MR_WARPS][MOE_MAX_EXPERTS + 1];
  int sh[MR_WARPS];
};

// A bucket of c pairs is cut into as few items as it fits, evenly, in multiples of 8 rows.
__device__ __forceinline__ int mr_items(int c) { return (c + MOE_ITEM_ROWS - 1) / MOE_ITEM_ROWS; }
__device__ __forceinline__ int mr_item_rows(int c) {
  const int n = mr_items(c);
  return n ? ((c + n - 1) / n + 7) / 8 * 8 : 0;
}
__device__ __forceinline__ int mr_ceil16(int n) { return (n + 15) & ~15; }

__device__ __forceinline__ void mr_header(const RouteArgs& a, int items) {
  a.plan[0] = items;
  a.plan[1] = 0;
  *reinterpret_cast<int**>(a.plan + 2) = a.error;
}

// Offsets, work items (block 0) and this block's pairs, from s.total and s.base.
__device__ __forceinline__ void mr_place(const RouteArgs& a, RouteSmem& s) {
  const int nb = a.E + 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int e = threadIdx.x; e < nb; e += MR_THREADS) {
    const int c = s.total[e], each = mr_item_rows(c), n = mr_items(c);
    s.scan[e] = n;
    s.pad[e] = n ? (n - 1) * mr_ceil16(each) + mr_ceil16(c - (n - 1) * each) : 0;
  }
  __syncthreads();
  const int all = mr_scan(s.total, s.first, nb, s.sh);
  mr_scan(s.pad, s.pad, nb, s.sh);
  if (blockIdx.x == 0) {
    const int items_all = mr_scan(s.scan, s.scan, nb, s.sh);
    int4* items = reinterpret_cast<int4*>(a.plan + MOE_PLAN_HEADER);
    for (int e = threadIdx.x; e < nb; e += MR_THREADS) {
      const int c = s.total[e], first = s.first[e], n = mr_items(c), each = mr_item_rows(c);
      a.offsets[e] = first;
      for (int i = 0; i < n; i++)
        items[s.scan[e] + i] = make_int4(e, first + i * each, min(each, c - i * each), s.pad[e] + i * mr_ceil16(each));
    }
    if (threadIdx.x == 0) {
      a.offsets[nb] = all;
      mr_header(a, items_all);
    }
  }
  for (int e = threadIdx.x; e < nb; e += MR_THREADS) s.base[e] += s.first[e];
  const int row0 = blockIdx.x * a.rows_per_block;
  const int p0 = row0 * a.top_k, p1 = min(a.M, row0 + a.rows_per_block) * a.top_k;
  for (int c0 = p0; c0 < p1; c0 += MR_THREADS) {
    for (int e = lane; e < nb; e += 32) s.cnt[warp][e] = 0;
    __syncthreads();
    const int pair = c0 + threadIdx.x;
    int bucket = -1;
    if (pair < p1) {
      const int id = a.ids[pair];
      bucket = id < 0 ? a.E : id;
    }
    const unsigned same = __match_any_sync(0xffffffffu, bucket);
    const int rank = __popc(same & ((1u << lane) - 1u));
    if (bucket >= 0 && rank == 0) s.cnt[warp][bucket] = __popc(same);
    __syncthreads();
    for (int e = threadIdx.x; e < nb; e += MR_THREADS) {
      int run = s.base[e];
#pragma unroll
      for (int w = 0; w < MR_WARPS; w++) {
        const int t = s.cnt[w][e];
        s.cnt[w][e] = run;
        run += t;
      }
      s.base[e] = run;
    }
    __syncthreads();
    if (bucket >= 0) {
      const int pos = s.cnt[warp][bucket] + rank, in = pos - s.first[bucket];
      const int c = s.total[bucket], each = mr_item_rows(c), i = in / each;
      a.pairs[pos] = pair;
      a.where[pair] = bucket == a.E ? make_int2(-1, 0)
                                    : make_int2(s.pad[bucket] + i * mr_ceil16(each),
                                                (in - i * each) | mr_ceil16(min(each, c - i * each)) << 16);
    }
    __syncthreads();
  }
}

// The same for at most 128 pairs in one block (every bucket is one item): each pair counts the ones that go before it.
constexpr int MR_FEW = 128;
__device__ __forceinline__ void mr_place_few(const RouteArgs& a, RouteSmem& s) {
  const int n = a.M * a.top_k, p = threadIdx.x;
  const int* bucket = s.cnt[0];   // [MR_FEW], every pair's
  int* size = s.cnt[0] + MR_FEW;  // of the bucket that begins with pair q (0: it does not begin one)
  int less = 0, same = 0, before = 0, b = 0;
  if (p < n) {
    b = bucket[p];
    for (int q = 0; q < n; q++) {
      const int t = bucket[q];
      less += t < b;
      same += t == b;
      before += t == b && q < p;
    }
    a.pairs[less + before] = p;
    size[p] = before == 0 ? same : 0;
  }
  for (int e = threadIdx.x; e < a.E + 2; e += MR_THREADS) {
    int c = 0;
    for (int q = 0; q < n; q++) c += bucket[q] < e;
    a.offsets[e] = c;
  }
  const int items = __syncthreads_count(p < n && before == 0);
  if (p < n) {
    int item = 0, pad = 0;
    for (int q = 0; q < n; q++) {
      const int t = size[q];
      if (t && bucket[q] < b) {
        item++;
        pad += mr_ceil16(t);
      }
    }
    if (before == 0)
      reinterpret_cast<int4*>(a.plan + MOE_PLAN_HEADER)[item] = make_int4(b, less, same, pad);
    a.where[p] = b == a.E ? make_int2(-1, 0) : make_int2(pad, before | mr_ceil16(same) << 16);
  }
  if (p == 0) {
    mr_header(a, items);
  }
}

// Selection and counting; with ONE the block holds every row and places the pairs too.
template <int EL, bool PACK, bool ONE>
__global__ void __launch_bounds__(MR_THREADS) moe_select_kernel(RouteArgs a) {
  __shared__ RouteSmem s;
  const int nb = a.E + 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool few = ONE && a.M * a.top_k <= MR_FEW;
  if (!few) {
    for (int e = threadIdx.x; e < nb; e += MR_THREADS) {
      s.total[e] = 0;
      s.base[e] = 0;
    }
    __syncthreads();
  }
  pdl_wait();
  pdl_trigger();
  const int r0 = blockIdx.x * a.rows_per_block, r1 = min(a.M, r0 + a.rows_per_block);
  for (int row = r0 + warp; row < r1; row += MR_WARPS) {
    const int id = mr_row<EL, PACK>(a, row, lane);
    if (lane < a.top_k) {
      const int bucket = id < 0 ? a.E : id;
      if (few)
        s.cnt[0][row * a.top_k + lane] = bucket;
      else
        atomicAdd(&s.total[bucket], 1);
    }
  }
  __syncthreads();
  if constexpr (ONE) {
    if (few)
      mr_place_few(a, s);
    else
      mr_place(a, s);
  } else {
    for (int e = threadIdx.x; e < nb; e += MR_THREADS) a.counts[(size_t)e * a.blocks + blockIdx.x] = s.total[e];
  }
}

__global__ void __launch_bounds__(MR_THREADS) moe_place_kernel(RouteArgs a) {
  __shared__ RouteSmem s;
  const int nb = a.E + 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_trigger();
  // a warp per bucket, four at a time: the blocks' counts, all and the earlier blocks', every load in flight at once
  for (int e0 = warp; e0 < nb; e0 += 4 * MR_WARPS) {
    int c[4][(MOE_ROUTE_BLOCKS + 31) / 32];
#pragma unroll
    for (int u = 0; u < 4; u++)
#pragma unroll
      for (int i = 0; i < (MOE_ROUTE_BLOCKS + 31) / 32; i++) {
        const int e = e0 + u * MR_WARPS, b = i * 32 + lane;
        c[u][i] = e < nb && b < a.blocks ? a.counts[(size_t)e * a.blocks + b] : 0;
      }
#pragma unroll
    for (int u = 0; u < 4; u++) {
      int all = 0, earlier = 0;
#pragma unroll
      for (int i = 0; i < (MOE_ROUTE_BLOCKS + 31) / 32; i++) {
        all += c[u][i];
        earlier += i * 32 + lane < (int)blockIdx.x ? c[u][i] : 0;
      }
      all = __reduce_add_sync(0xffffffffu, all);
      earlier = __reduce_add_sync(0xffffffffu, earlier);
      if (lane == 0 && e0 + u * MR_WARPS < nb) {
        s.total[e0 + u * MR_WARPS] = all;
        s.base[e0 + u * MR_WARPS] = earlier;
      }
    }
  }
  __syncthreads();
  mr_place(a, s);
}

template <int EL, bool PACK>
static int mr_launch_as(const RouteArgs& a, cudaStream_t st) {
  if (a.blocks <= 1)
    return launch("moe_select_kernel", moe_select_kernel<EL, PACK, true>, dim3(1), dim3(MR_THREADS), 0, st, a);
  const int rc =
      launch("moe_select_kernel", moe_select_kernel<EL, PACK, false>, dim3(a.blocks), dim3(MR_THREADS), 0, st, a);
  if (rc) return rc;
  return launch("moe_place_kernel", moe_place_kernel, dim3(a.blocks), dim3(MR_THREADS), 0, st, a);
}

template <int EL>
static int mr_launch(const RouteArgs& a, cudaStream_t st) {
  return !a.f32 && !a.bias ? mr_launch_as<EL, true>(a, st) : mr_launch_as<EL, false>(a, st);
}

}  // namespace im

using namespace im;

static bool moe_sizes_ok(int64_t M, int64_t E, int64_t top_k) {
  return M >= 0 && M <= MOE_MAX_ROWS && E >= 1 && E <= MOE_MAX_EXPERTS && top_k >= 1 && top_k <= MOE_MAX_TOP_K &&
         top_k <= E;
}

extern "C" size_t im_moe_plan_bytes(int64_t M, int64_t E, int64_t top_k) {
  return moe_sizes_ok(M, E, top_k) ? moe_plan(M, E, top_k).bytes : 0;
}

extern "C" int im_moe_route(const void* logits, int logits_f32, int64_t M, int64_t E, int64_t ld, const float* bias,
                            int64_t top_k, int scoring, int normalise, float scale, int32_t* ids, float* weights,
                            int32_t* offsets, int32_t* pairs, void* plan, size_t plan_bytes, void* stream) {
  return im_moe_route_ex(logits, logits_f32, M, E, ld, bias, top_k, scoring, normalise, scale, ids, weights, offsets,
                         pairs, plan, plan_bytes, nullptr, stream);
}

extern "C" int im_moe_route_ex(const void* logits, int logits_f32, int64_t M, int64_t E, int64_t ld, const float* bias,
                               int64_t top_k, int scoring, int normalise, float scale, int32_t* ids, float* weights,
                               int32_t* offsets, int32_t* pairs, void* plan, size_t plan_bytes, int32_t* error,
                               void* stream) {
  clear_error();
  IM_REQUIRE(M >= 0 && E >= 1 && top_k >= 1 && top_k <= E, IM_INVALID,
             "im_moe_route: bad sizes M=%lld E=%lld top_k=%lld", (long long)M, (long long)E, (long long)top_k);
  IM_REQUIRE(moe_sizes_ok(M, E, top_k), IM_UNSUPPORTED,
             "im_moe_route: at most %lld rows, %d experts and %d places a row (M=%lld E=%lld top_k=%lld)",
             (long long)MOE_MAX_ROWS, MOE_MAX_EXPERTS, MOE_MAX_TOP_K, (long long)M, (long long)E, (long long)top_k);
  const int on_score = scoring & IM_MOE_BIAS_ON_SCORE;
  scoring &= ~IM_MOE_BIAS_ON_SCORE;
  IM_REQUIRE(scoring == IM_MOE_SOFTMAX || scoring == IM_MOE_SIGMOID, IM_INVALID, "im_moe_route: bad scoring");
  IM_REQUIRE(!on_score || bias, IM_INVALID, "im_moe_route: a bias on the scores needs bias");
  IM_REQUIRE(offsets && plan, IM_INVALID, "im_moe_route: null pointer");
  IM_REQUIRE(M == 0 || (logits && ids && weights && pairs), IM_INVALID, "im_moe_route: null pointer");
  IM_REQUIRE(ld >= E, IM_INVALID, "im_moe_route: row stride %lld below %lld experts", (long long)ld, (long long)E);
  IM_REQUIRE(aligned(logits, logits_f32 ? 4 : 2) && aligned(plan, 16) && aligned(error, 4), IM_INVALID,
             "im_moe_route: misaligned logits, plan or error word");
  const MoePlan p = moe_plan(M, E, top_k);
  IM_REQUIRE(plan_bytes >= p.bytes, IM_INVALID, "im_moe_route: plan of %zu bytes needed, %zu given", p.bytes,
             plan_bytes);
  RouteArgs a = {};
  a.logits = logits;
  a.bias = bias;
  a.ids = ids;
  a.weights = weights;
  a.offsets = offsets;
  a.pairs = pairs;
  a.plan = reinterpret_cast<int*>(plan);
  a.where = reinterpret_cast<int2*>(a.plan + p.where);
  a.counts = a.plan + p.counts;
  a.error = error;
  a.f32 = logits_f32;
  a.scoring = scoring;
  a.on_score = on_score;
  a.normalise = normalise;
  a.scale = scale;
  a.M = (int)M;
  a.E = (int)E;
  a.top_k = (int)top_k;
  a.rows_per_block = (int)p.rows_per_block;
  a.blocks = (int)p.blocks;
  a.ld = ld;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (E <= 32) return mr_launch<1>(a, st);
  if (E <= 64) return mr_launch<2>(a, st);
  if (E <= 128) return mr_launch<4>(a, st);
  if (E <= 256) return mr_launch<8>(a, st);
  return mr_launch<16>(a, st);
}
