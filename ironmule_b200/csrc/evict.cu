// Eviction from a paged cache by accumulated attention weight.
//
// A row is one kv head of one sequence in one layer, with its own slots, weights and positions. Of n slots a budget
// stays: slots are ordered by (protected, weight, lower slot first), protected being the first `sinks` positions and the
// last `recent` ones, and the first min(n, budget) = n' of that order are kept. A kept slot behind n' moves to a dropped
// slot before it, the i-th to the i-th: as many rows of K and V move as the cut leaves behind it, and none is both read
// and written, so the move is in place and in parallel. Attention over slots does not mind their order; positions say
// which token a slot holds.
//
// The order is that of one 32-bit key a slot: the weight's bits made monotone, NaN lowest, protected slots highest. The
// n'-th largest key is found digit by digit (8 bits a pass over the row's keys), the slots that share it are kept from
// the lowest slot on.
//
// Bound: HBM; weights and positions read once, n' of each written, 4 rows of head_dim values a moved slot.
#include "common.cuh"

namespace im {

constexpr int EV_THREADS = 1024;
constexpr int EV_WARPS = EV_THREADS / 32;

struct EvictArgs {
  char* k;
  char* v;
  long long layer_bytes;  // of k and v
  long long pages;
  const int* page_table;
  long long max_pages;
  const int* lengths;
  const int* seen;
  const float* weights;
  float* weights_out;
  const int* pos;
  int* pos_out;
  int* lengths_out;
  int seqs, hkv;
  long long cap;
  int row_bytes;  // a slot's of one head
  long long budget, recent, sinks;
  int* moves;  // [rows]
  int* holes;  // [rows][most]
  int* movers;
  long long most;
};

__device__ __forceinline__ int ev_length(const EvictArgs& a, int s) {
  const long long n = a.lengths[s];
  return (int)max(0ll, min(n, min(a.cap, a.max_pages * 16)));
}

__device__ __forceinline__ uint32_t ev_key(float w, int pos, long long sinks, long long recent_from) {
  if (pos < sinks || pos >= recent_from) return 0xffffffffu;
  if (w != w) return 0u;
  const uint32_t b = __float_as_uint(w + 0.0f);  // -0 as +0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// One block a row: which slots stay, and the pairs (hole, mover).
__global__ void __launch_bounds__(EV_THREADS) evict_select_kernel(EvictArgs a) {
  __shared__ unsigned hist[256];
  __shared__ unsigned s_digit, s_left;
  __shared__ int s_ties[EV_WARPS], s_holes[EV_WARPS], s_movers[EV_WARPS];
  pdl_wait();
  pdl_trigger();
  const long long row = blockIdx.x;  // (layer, sequence, head)
  const int seq = (int)(row / a.hkv % a.seqs);
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int n = ev_length(a, seq);
  const int left = (int)min((long long)n, a.budget);
  if (t == 0 && row < (long long)a.seqs * a.hkv && row % a.hkv == 0) a.lengths_out[seq] = left;
  const float* w = a.weights + row * a.cap;
  const int* pos = a.pos + row * a.cap;
  float* wo = a.weights_out + row * a.cap;
  int* po = a.pos_out + row * a.cap;
  if (n <= left || left == 0) {
    if (t == 0) a.moves[row] = 0;
    for (int s = t; s < left; s += EV_THREADS) wo[s] = w[s], po[s] = pos[s];
    return;
  }
  const long long recent_from = (long long)a.seen[seq] - a.recent;
  auto key = [&](int s) { return ev_key(w[s], pos[s], a.sinks, recent_from); };
  // the left-th largest key, and how many of those equal to it stay
  uint32_t prefix = 0, mask = 0;
  unsigned need = (unsigned)left;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = t; i < 256; i += EV_THREADS) hist[i] = 0;
    __syncthreads();
    for (int s = t; s < n; s += EV_THREADS) {
      const uint32_t k = key(s);
      if ((k & mask) == prefix) atomicAdd(&hist[k >> shift & 255], 1u);
    }
    __syncthreads();
    if (t == 0) {
      unsigned above = 0;
      int d = 255;
      for (; d > 0 && above + hist[d] < need; d--) above += hist[d];
      s_digit = d, s_left = need - above;
    }
    __syncthreads();
    prefix |= s_digit << shift, mask |= 255u << shift, need = s_left;
    __syncthreads();
  }
  const uint32_t border = prefix;
  // each warp walks a run of slots in order; counts before it come from the warps before
  const int span = ((n + EV_WARPS - 1) / EV_WARPS + 31) / 32 * 32;
  const int lo = min(n, warp * span), hi = min(n, lo + span);
  int ties = 0;
  for (int s0 = lo; s0 < hi; s0 += 32)
    ties += __popc(__ballot_sync(0xffffffffu, s0 + lane < hi && key(s0 + lane) == border));
  if (lane == 0) s_ties[warp] = ties;
  __syncthreads();
  int ties_before = 0;
  for (int i = 0; i < warp; i++) ties_before += s_ties[i];
  for (int pass = 0; pass < 2; pass++) {
    int run = ties_before, holes = 0, movers = 0;
    if (pass)
      for (int i = 0; i < warp; i++) holes += s_holes[i], movers += s_movers[i];
    for (int s0 = lo; s0 < hi; s0 += 32) {
      const int s = s0 + lane;
      const uint32_t k = s < hi ? key(s) : 0u;
      const unsigned tie = __ballot_sync(0xffffffffu, s < hi && k == border);
      const unsigned before = (1u << lane) - 1;
      const bool kept = s < hi && (k > border || (k == border && run + __popc(tie & before) < (int)need));
      run += __popc(tie);
      const unsigned hole = __ballot_sync(0xffffffffu, s < hi && s < left && !kept);
      const unsigned mover = __ballot_sync(0xffffffffu, kept && s >= left);
      if (pass) {
        if (hole >> lane & 1) a.holes[row * a.most + holes + __popc(hole & before)] = s;
        if (mover >> lane & 1) a.movers[row * a.most + movers + __popc(mover & before)] = s;
        if (kept && s < left) wo[s] = w[s], po[s] = pos[s];
      }
      holes += __popc(hole), movers += __popc(mover);
    }
    if (!pass) {
      if (lane == 0) s_holes[warp] = holes, s_movers[warp] = movers;
      __syncthreads();
    } else if (warp == EV_WARPS - 1 && lane == 0) {
      a.moves[row] = holes;
    }
  }
}

// A slot's K, V, weight and position to its new place: BYTES a lane, a warp for each pair of slots.
template <int BYTES>
__global__ void __launch_bounds__(256) evict_move_kernel(EvictArgs a) {
  pdl_wait();
  pdl_trigger();
  const long long row = blockIdx.x;
  const int head = (int)(row % a.hkv), seq = (int)(row / a.hkv % a.seqs);
  const long long layer = row / a.hkv / a.seqs;
  const int count = a.moves[row];
  const int lane = threadIdx.x & 31;
  const int* table = a.page_table + seq * a.max_pages;
  for (int i = blockIdx.y * 8 + threadIdx.x / 32; i < count; i += gridDim.y * 8) {
    const int to = a.holes[row * a.most + i], from = a.movers[row * a.most + i];
    if (lane == 0) {
      a.weights_out[row * a.cap + to] = a.weights[row * a.cap + from];
      a.pos_out[row * a.cap + to] = a.pos[row * a.cap + from];
    }
    const long long to_page = table[to / 16], from_page = table[from / 16];
    if (to_page < 0 || to_page >= a.pages || from_page < 0 || from_page >= a.pages) continue;
    const long long dst = layer * a.layer_bytes + ((to_page * a.hkv + head) * 16 + to % 16) * a.row_bytes;
    const long long src = layer * a.layer_bytes + ((from_page * a.hkv + head) * 16 + from % 16) * a.row_bytes;
    for (int at = lane * BYTES; at < a.row_bytes; at += 32 * BYTES) {
      if (BYTES == 16) {
        const uint4 x = *(const uint4*)(a.k + src + at), y = *(const uint4*)(a.v + src + at);
        *(uint4*)(a.k + dst + at) = x;
        *(uint4*)(a.v + dst + at) = y;
      } else {
        const char x = a.k[src + at], y = a.v[src + at];
        a.k[dst + at] = x;
        a.v[dst + at] = y;
      }
    }
  }
}

static long long evict_most(int64_t cap, int64_t budget) { return budget < cap - budget ? budget : cap - budget; }

}  // namespace im

using namespace im;

extern "C" size_t im_cache_evict_workspace_bytes(int64_t layers, int64_t S, int64_t Hkv, int64_t cap, int64_t budget) {
  if (layers < 1 || S < 1 || Hkv < 1 || cap < 1 || budget < 0 || layers * S * Hkv >= (1ll << 31)) return 0;
  const long long rows = layers * S * Hkv, most = evict_most(cap, budget);
  return (size_t)(rows * 4 + (most > 0 ? 2 * rows * most * 4 : 0));
}

extern "C" int im_cache_evict(void* k_cache, void* v_cache, int64_t layers, int64_t layer_bytes, int64_t pages,
                              const int32_t* page_table, int64_t max_pages, const int32_t* lengths, const int32_t* seen,
                              const float* weights, float* weights_out, const int32_t* slot_pos, int32_t* pos_out,
                              int32_t* lengths_out, int64_t S, int64_t Hkv, int64_t cap, int64_t row_bytes,
                              int64_t budget, int64_t recent, int64_t sinks, void* workspace, size_t workspace_bytes,
                              void* stream) {
  clear_error();
  IM_REQUIRE(layers >= 0 && S >= 0 && Hkv >= 1 && cap >= 1 && row_bytes >= 1 && pages >= 0 && max_pages >= 0 &&
                 budget >= 0 && recent >= 0 && sinks >= 0 && layer_bytes >= 0,
             IM_INVALID, "im_cache_evict: bad sizes");
  IM_REQUIRE(recent <= budget && sinks <= budget - recent, IM_INVALID,
             "im_cache_evict: %lld recent and %lld first slots do not fit a budget of %lld", (long long)recent,
             (long long)sinks, (long long)budget);
  if (layers == 0 || S == 0) return IM_OK;
  IM_REQUIRE(k_cache && v_cache && page_table && lengths && seen && weights && weights_out && slot_pos && pos_out &&
                 lengths_out,
             IM_INVALID, "im_cache_evict: null pointer");
  const size_t need = im_cache_evict_workspace_bytes(layers, S, Hkv, cap, budget);
  IM_REQUIRE(need > 0 && cap < (1ll << 30) && row_bytes < (1 << 20) && budget < (1ll << 31), IM_UNSUPPORTED,
             "im_cache_evict: too large");
  IM_REQUIRE(workspace && aligned(workspace, 16) && workspace_bytes >= need, IM_INVALID,
             "im_cache_evict: a workspace of %zu bytes needed, %zu given", need, workspace_bytes);
  const long long rows = layers * S * Hkv, most = evict_most(cap, budget);
  EvictArgs a = {(char*)k_cache, (char*)v_cache, layer_bytes, pages, page_table, max_pages, lengths, seen,
                 weights, weights_out, slot_pos, pos_out, lengths_out, (int)S, (int)Hkv, cap, (int)row_bytes,
                 budget, recent, sinks, (int*)workspace, nullptr, nullptr, most};
  a.holes = a.moves + rows, a.movers = a.holes + (most > 0 ? rows * most : 0);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int rc = launch("evict_select_kernel", evict_select_kernel, dim3((unsigned)rows), dim3(EV_THREADS), 0, st, a);
  if (rc != IM_OK || most <= 0) return rc;
  const long long chunks = (most + 63) / 64;
  const dim3 grid((unsigned)rows, (unsigned)(chunks < 1024 ? chunks : 1024));
  if (row_bytes % 16 == 0 && aligned(k_cache, 16) && aligned(v_cache, 16) && layer_bytes % 16 == 0)
    return launch("evict_move_kernel", evict_move_kernel<16>, grid, dim3(256), 0, st, a);
  return launch("evict_move_kernel", evict_move_kernel<1>, grid, dim3(256), 0, st, a);
}
