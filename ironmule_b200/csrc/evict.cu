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
// n'-th largest key is found digit by digit (8 bits a pass over the row's keys, which lie in shared memory), the slots that
// share it are kept from the lowest slot on; the search ends early where all of a digit's slots stay.
//
// Bound: HBM; weights and positions read once, n' of each written, 4 rows of head_dim values a moved slot. A short row is
// one block's, a long one a cluster's of up to 16, each with a run of its slots, which share counts through distributed
// shared memory.
#include <cooperative_groups.h>

#include "common.cuh"

namespace im {

namespace cg = cooperative_groups;

constexpr int EV_CLUSTER = 16;
constexpr int EV_RUN = 16384;       // slots of a block before a row takes another, up to EV_CLUSTER blocks
constexpr int EV_MOST = 49152;      // slots whose keys a block can hold
constexpr int EV_MOVE_THREADS = 256;

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

// Sums x over the block's warps before this one, and over all (warps <= 32); every thread gets both.
template <int WARPS>
__device__ __forceinline__ int2 ev_before(int x, int* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();
  if (lane == 0) scratch[warp] = x;
  __syncthreads();
  int v = lane < WARPS ? scratch[lane] : 0, before = lane < warp ? v : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v += __shfl_xor_sync(0xffffffffu, v, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  return make_int2(before, v);
}

// Which slots of a row stay, and the pairs (hole, mover). A cluster a row, a run of `run` slots a block, whose warps
// each walk a part of it in order.
template <int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 2) evict_select_kernel(EvictArgs a) {
  constexpr int THREADS = WARPS * 32;
  extern __shared__ uint32_t keys[];
  __shared__ unsigned hist[2][256];  // by turns: a block may count its next digit while others still read this one
  __shared__ unsigned s_digit, s_need, s_all;
  __shared__ int scratch[32];
  __shared__ int3 shared_counts;  // this block's ties, holes, movers, for the others
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = cluster.num_blocks(), rank = cluster.block_rank();
  pdl_wait();
  pdl_trigger();
  const long long row = blockIdx.x / ranks;  // (layer, sequence, head)
  const int seq = (int)(row / a.hkv % a.seqs);
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int n = ev_length(a, seq);
  const int left = (int)min((long long)n, a.budget);
  // lengths_out may be lengths: it is written here only where nothing is ever cut, else by the second kernel
  if (a.most <= 0 && t == 0 && rank == 0 && row < (long long)a.seqs * a.hkv && row % a.hkv == 0) a.lengths_out[seq] = left;
  const float* w = a.weights + row * a.cap;
  const int* pos = a.pos + row * a.cap;
  float* wo = a.weights_out + row * a.cap;
  int* po = a.pos_out + row * a.cap;
  if (n <= left || left == 0) {  // the whole cluster
    if (t == 0 && rank == 0) a.moves[row] = 0;
    for (int s = rank * THREADS + t; s < left; s += ranks * THREADS) wo[s] = w[s], po[s] = pos[s];
    return;
  }
  const long long recent_from = (long long)a.seen[seq] - a.recent;
  const int run = ((n + ranks - 1) / ranks + 31) / 32 * 32;
  const int begin = min(n, rank * run), count = min(n, begin + run) - begin;
#pragma unroll 4
  for (int s = t; s < count; s += THREADS) keys[s] = ev_key(w[begin + s], pos[begin + s], a.sinks, recent_from);
  for (int i = t; i < 512; i += THREADS) hist[0][i] = 0;
  __syncthreads();
  // the left-th largest key, and how many of those that share its digits stay
  uint32_t border = 0, mask = 0;
  unsigned need = (unsigned)left;
  bool all = false;  // all of them stay
  for (int shift = 24; shift >= 0 && !all; shift -= 8) {
    unsigned* h = hist[shift >> 3 & 1];
    for (int s = t; s < count; s += THREADS) {
      const uint32_t k = keys[s];
      if ((k & mask) == border) atomicAdd(&h[k >> shift & 255], 1u);
    }
    if (ranks > 1) cluster.sync();
    else __syncthreads();
    if (warp == 0) {  // eight digits a lane, from the highest down
      unsigned c[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int d = 255 - lane * 8 - i;
        c[i] = 0;
        if (ranks == 1) c[i] = h[d];
        else
          for (int r = 0; r < ranks; r++) c[i] += *cluster.map_shared_rank(&h[d], r);
        sum += c[i];
      }
      unsigned above = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned x = __shfl_up_sync(0xffffffffu, above, o);
        if (lane >= o) above += x;
      }
      above -= sum;
      if (above < need && need <= above + sum) {  // one lane
#pragma unroll
        for (int i = 0; i < 8; i++) {
          if (above < need && need <= above + c[i]) {
            s_digit = 255 - lane * 8 - i, s_need = need - above, s_all = c[i] == need - above;
          }
          above += c[i];
        }
      }
    }
    // the other counts are clear before the next digit: nobody reads them since the cluster met
    for (int i = t; i < 256; i += THREADS) hist[(shift >> 3 & 1) ^ 1][i] = 0;
    __syncthreads();
    border |= s_digit << shift, mask |= 255u << shift, need = s_need, all = s_all != 0;
    __syncthreads();
  }
  // keys of the same digits as the border's: all stay, or the first `need` in slot order
  const int part = ((count + WARPS - 1) / WARPS + 31) / 32 * 32;
  const int lo = min(count, warp * part), hi = min(count, lo + part);
  const unsigned under = (1u << lane) - 1;
  int ties = 0;
  if (!all) {
    for (int s0 = lo; s0 < hi; s0 += 32)
      ties += __popc(__ballot_sync(0xffffffffu, s0 + lane < hi && keys[s0 + lane] == border));
    const int2 x = ev_before<WARPS>(ties, scratch);
    ties = x.x;
    if (ranks > 1) {
      if (t == 0) shared_counts.x = x.y;
      cluster.sync();
      for (int r = 0; r < rank; r++) ties += cluster.map_shared_rank(&shared_counts, r)->x;
    }
  }
  int holes = 0, movers = 0;
  const int ties_first = ties;
  for (int pass = 0; pass < 2; pass++) {
    ties = ties_first;
    for (int s0 = lo; s0 < hi; s0 += 32) {
      const int at = s0 + lane, s = begin + at;
      const uint32_t k = at < hi ? keys[at] : 0u;
      bool kept;
      if (all) {
        kept = at < hi && (k & mask) >= border;
      } else {
        const unsigned tie = __ballot_sync(0xffffffffu, at < hi && k == border);
        kept = at < hi && (k > border || (k == border && ties + __popc(tie & under) < (int)need));
        ties += __popc(tie);
      }
      const unsigned hole = __ballot_sync(0xffffffffu, at < hi && s < left && !kept);
      const unsigned mover = __ballot_sync(0xffffffffu, kept && s >= left);
      if (pass) {
        if (hole >> lane & 1) a.holes[row * a.most + holes + __popc(hole & under)] = s;
        if (mover >> lane & 1) a.movers[row * a.most + movers + __popc(mover & under)] = s;
        if (kept && s < left) wo[s] = w[s], po[s] = pos[s];
      }
      holes += __popc(hole), movers += __popc(mover);
    }
    if (pass) break;
    const int2 h = ev_before<WARPS>(holes, scratch), v = ev_before<WARPS>(movers, scratch);
    holes = h.x, movers = v.x;
    int total = h.y;
    if (ranks > 1) {
      if (t == 0) shared_counts.y = h.y, shared_counts.z = v.y;
      cluster.sync();
      total = 0;
      for (int r = 0; r < ranks; r++) {
        const int3 c = *cluster.map_shared_rank(&shared_counts, r);
        if (r < rank) holes += c.y, movers += c.z;
        total += c.y;
      }
      cluster.sync();  // nobody leaves while its counts are read
    }
    if (t == 0 && rank == 0) a.moves[row] = total;
  }
}

// A slot's K, V, weight and position to its new place. A warp takes 32 moves: each lane finds one move's places, then the
// warp copies their rows, BYTES a lane, K's and V's chunks of a move side by side.
template <int BYTES>
__global__ void __launch_bounds__(EV_MOVE_THREADS, 3) evict_move_kernel(EvictArgs a) {
  pdl_wait();
  pdl_trigger();
  const long long row = blockIdx.x;
  const int head = (int)(row % a.hkv), seq = (int)(row / a.hkv % a.seqs);
  const int count = a.moves[row];
  const int lane = threadIdx.x & 31;
  if (blockIdx.y == 0 && threadIdx.x == 0 && row < (long long)a.seqs * a.hkv && head == 0)
    a.lengths_out[seq] = (int)min((long long)ev_length(a, seq), a.budget);
  const int* table = a.page_table + seq * a.max_pages;
  const long long layer = row / a.hkv / a.seqs * a.layer_bytes;
  const int chunks = a.row_bytes / BYTES;  // of K, and of V
  for (int i0 = (blockIdx.y * (EV_MOVE_THREADS / 32) + threadIdx.x / 32) * 32; i0 < count;
       i0 += gridDim.y * EV_MOVE_THREADS) {
    const int moves = min(32, count - i0);
    long long dst = 0, src = -1;
    if (lane < moves) {
      const int to = a.holes[row * a.most + i0 + lane], from = a.movers[row * a.most + i0 + lane];
      const long long to_page = table[to / 16], from_page = table[from / 16];
      a.weights_out[row * a.cap + to] = a.weights[row * a.cap + from];
      a.pos_out[row * a.cap + to] = a.pos[row * a.cap + from];
      if (to_page >= 0 && to_page < a.pages && from_page >= 0 && from_page < a.pages) {
        dst = layer + ((to_page * a.hkv + head) * 16 + to % 16) * a.row_bytes;
        src = layer + ((from_page * a.hkv + head) * 16 + from % 16) * a.row_bytes;
      }
    }
    const int work = moves * 2 * chunks;
    constexpr int BATCH = BYTES == 16 ? 8 : 4;  // loads in flight a lane
    for (int c0 = 0; c0 < work; c0 += 32 * BATCH) {
      uint4 x[BATCH];
      char* to[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; i++) {
        const int c = c0 + i * 32 + lane;
        const int move = c / (2 * chunks), part = c - move * 2 * chunks;
        const long long from = __shfl_sync(0xffffffffu, src, move & 31);
        const long long there = __shfl_sync(0xffffffffu, dst, move & 31);
        to[i] = nullptr;
        if (c < work && from >= 0) {
          const bool is_k = part < chunks;
          const long long off = (long long)(is_k ? part : part - chunks) * BYTES;
          char* cache = is_k ? a.k : a.v;
          to[i] = cache + there + off;
          if (BYTES == 16) x[i] = *(const uint4*)(cache + from + off);
          else x[i].x = *(const unsigned char*)(cache + from + off);
        }
      }
#pragma unroll
      for (int i = 0; i < BATCH; i++) {
        if (to[i]) {
          if (BYTES == 16) *(uint4*)to[i] = x[i];
          else *(unsigned char*)to[i] = (unsigned char)x[i].x;
        }
      }
    }
  }
}

template <int WARPS>
int launch_evict_select(const EvictArgs& a, long long rows, int ranks, cudaStream_t st) {
  const long long run = ((a.cap + ranks - 1) / ranks + 31) / 32 * 32;
  const int smem = (int)(run * 4);
  cudaError_t e = cudaFuncSetAttribute(evict_select_kernel<WARPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess && ranks > 8)
    e = cudaFuncSetAttribute(evict_select_kernel<WARPS>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) {
    set_error("evict_select_kernel: %s", cudaGetErrorString(e));
    return IM_CUDA_ERROR;
  }
  return launch_cluster("evict_select_kernel", evict_select_kernel<WARPS>, dim3((unsigned)(rows * ranks)),
                        dim3(WARPS * 32), ranks, smem, st, a);
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
  IM_REQUIRE(need > 0 && cap <= (int64_t)EV_CLUSTER * EV_MOST && row_bytes < (1 << 20), IM_UNSUPPORTED,
             "im_cache_evict: rows of %lld slots (up to %d), or too many of them", (long long)cap, EV_CLUSTER * EV_MOST);
  IM_REQUIRE(workspace && aligned(workspace, 16) && workspace_bytes >= need, IM_INVALID,
             "im_cache_evict: a workspace of %zu bytes needed, %zu given", need, workspace_bytes);
  const long long rows = layers * S * Hkv, most = evict_most(cap, budget);
  EvictArgs a = {(char*)k_cache, (char*)v_cache, layer_bytes, pages, page_table, max_pages, lengths, seen,
                 weights, weights_out, slot_pos, pos_out, lengths_out, (int)S, (int)Hkv, cap, (int)row_bytes,
                 budget, recent, sinks, (int*)workspace, nullptr, nullptr, most};
  a.holes = a.moves + rows, a.movers = a.holes + (most > 0 ? rows * most : 0);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  // blocks a row: one up to EV_RUN slots, more for longer rows (and so few rows that the device has room for them)
  int ranks = 1;
  while (ranks < EV_CLUSTER && (cap > (int64_t)ranks * EV_MOST || (cap > (int64_t)ranks * EV_RUN && rows * ranks < 296)))
    ranks *= 2;
  const int rc = cap <= 4096 ? launch_evict_select<8>(a, rows, ranks, st) : launch_evict_select<16>(a, rows, ranks, st);
  if (rc != IM_OK || most <= 0) return rc;
  const long long chunks = (most + EV_MOVE_THREADS - 1) / EV_MOVE_THREADS;
  const dim3 grid((unsigned)rows, (unsigned)(chunks < 1024 ? chunks : 1024));
  if (row_bytes % 16 == 0 && aligned(k_cache, 16) && aligned(v_cache, 16) && layer_bytes % 16 == 0)
    return launch("evict_move_kernel", evict_move_kernel<16>, grid, dim3(EV_MOVE_THREADS), 0, st, a);
  return launch("evict_move_kernel", evict_move_kernel<1>, grid, dim3(EV_MOVE_THREADS), 0, st, a);
}
