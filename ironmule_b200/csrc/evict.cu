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
// n'-th largest key is found digit by digit (8 bits a pass over the row's keys, which stay in registers), the slots that
// share it are kept from the lowest slot on; the search ends early where all of a digit's slots stay.
//
// Bound: HBM; weights and positions read once, n' of each written, 4 rows of head_dim values a moved slot. A row is one
// block's up to 16384 slots, and that block moves its slots too where they are few; else the pairs go through the workspace
// to a second kernel that spreads them over the device. Longer rows are a cluster's of up to 16 blocks, which share counts
// through distributed shared memory. 288 rows of 8192 slots of 2 x 256 bytes cut to 2048 take 102 us: 20 of selection, bound by
// instructions, and 80 of moves at 5.8 TB/s; 288 rows of 2064 cut by 16 slots 13.8 us.
#include <cooperative_groups.h>

#include "common.cuh"

namespace im {

namespace cg = cooperative_groups;

constexpr int EV_CLUSTER = 16;
constexpr int EV_RUN = 16384;  // slots of a block at most
constexpr int EV_MOVE_THREADS = 256;
constexpr int EV_HERE = 1024;  // moves of a row that its own block makes at most

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
  int moves_here;  // the first kernel moves the slots too
  int chunk_shift;  // log2 of a move's chunks (K's and V's), -1: no power of two
  int lengths_here;  // and writes lengths_out, which is not lengths
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
  const uint32_t b = __float_as_uint(w + 0.0f);  // -0 as +0
  const uint32_t k = w != w ? 0u : b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
  return pos < sinks || pos >= recent_from ? 0xffffffffu : k;
}

// Where a digit is counted: the eight that a lane reads lie 32 apart.
__device__ __forceinline__ int ev_bin(int digit) { return (digit & 7) * 32 + (digit >> 3); }

// Sums of x over the block's warps before this one, and over all; x is the same in a warp's lanes.
template <int WARPS>
__device__ __forceinline__ int2 ev_before(int x, int* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
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

// Up to 32 moves of one row by a warp: each lane has one move's slots; the warp then copies their rows together, BYTES a
// lane, K's and V's chunks of a move side by side, four loads in flight a lane (with eight, at half the
// warps an SM, a prompt's cut took 111 us in the place of 102).
template <int BYTES>
__device__ __forceinline__ void ev_move(const EvictArgs& a, long long row, const int* table, int moves, int to,
                                        int from) {
  const int head = (int)(row % a.hkv), lane = threadIdx.x & 31;
  const long long layer = row / a.hkv / a.seqs * a.layer_bytes;
  const int chunks = a.row_bytes / BYTES;  // of K, and of V
  long long dst = 0, src = -1;
  if (lane < moves) {
    const long long to_page = table[to / 16], from_page = table[from / 16];
    const bool on = to_page >= 0 && to_page < a.pages && from_page >= 0 && from_page < a.pages;
    // a slot whose page is none of the cache's neither moves nor is moved to: the hole keeps its token, so that position and
    // weight stay those of what the slot holds
    const int at = on ? from : to;
    a.weights_out[row * a.cap + to] = a.weights[row * a.cap + at];
    a.pos_out[row * a.cap + to] = a.pos[row * a.cap + at];
    if (on) {
      dst = layer + ((to_page * a.hkv + head) * 16 + to % 16) * a.row_bytes;
      src = layer + ((from_page * a.hkv + head) * 16 + from % 16) * a.row_bytes;
    }
  }
  constexpr int BATCH = 4;
  const int work = moves * 2 * chunks;
  for (int c0 = 0; c0 < work; c0 += 32 * BATCH) {
    uint4 x[BATCH];
    char* at[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; i++) {
      const int c = c0 + i * 32 + lane;
      const int move = a.chunk_shift >= 0 ? c >> a.chunk_shift : c / (2 * chunks), part = c - move * 2 * chunks;
      const long long here = __shfl_sync(0xffffffffu, src, move & 31);
      const long long there = __shfl_sync(0xffffffffu, dst, move & 31);
      at[i] = nullptr;
      if (c < work && here >= 0) {
        const bool is_k = part < chunks;
        const long long off = (long long)(is_k ? part : part - chunks) * BYTES;
        char* cache = is_k ? a.k : a.v;
        at[i] = cache + there + off;
        if (BYTES == 16) x[i] = *(const uint4*)(cache + here + off);
        else x[i].x = *(const unsigned char*)(cache + here + off);
      }
    }
#pragma unroll
    for (int i = 0; i < BATCH; i++) {
      if (at[i]) {
        if (BYTES == 16) *(uint4*)at[i] = x[i];
        else *(unsigned char*)at[i] = (unsigned char)x[i].x;
      }
    }
  }
}

// Which slots of a row stay, the pairs (hole, mover), and the moves where they are not left to the second kernel. A cluster
// a row; a warp has up to 32 * ITEMS slots in order, its lanes' keys in registers.
template <int THREADS, int ITEMS, int BLOCKS, int BYTES>
__global__ void __launch_bounds__(THREADS, BLOCKS) evict_select_kernel(EvictArgs a) {
  constexpr int WARPS = THREADS / 32;
  extern __shared__ int pairs[];     // where the moves are made here: holes, movers, the sequence's pages
  __shared__ unsigned hist[2][256];  // by turns: a block may count its next digit while others still read this one
  __shared__ unsigned s_digit[2], s_need[2], s_all[2];
  __shared__ int scratch[2][32];
  __shared__ unsigned merged[256];           // a cluster's counts of the digit
  __shared__ int3 shared_counts;             // this block's ties, holes, movers, for the others
  __shared__ int3 all_counts[EV_CLUSTER];    // theirs
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = cluster.num_blocks(), rank = cluster.block_rank();
  pdl_wait();
  pdl_trigger();
  const long long row = blockIdx.x / ranks;  // (layer, sequence, head)
  const int seq = (int)(row / a.hkv % a.seqs);
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int n = ev_length(a, seq);
  const int left = (int)min((long long)n, a.budget);
  if (a.lengths_here && t == 0 && rank == 0 && row < (long long)a.seqs * a.hkv && row % a.hkv == 0)
    a.lengths_out[seq] = left;
  const float* w = a.weights + row * a.cap;
  const int* pos = a.pos + row * a.cap;
  float* wo = a.weights_out + row * a.cap;
  int* po = a.pos_out + row * a.cap;
  if (n <= left || left == 0) {  // the whole cluster
    if (!a.moves_here && t == 0 && rank == 0) a.moves[row] = 0;
    for (int s = rank * THREADS + t; s < left; s += ranks * THREADS) wo[s] = w[s], po[s] = pos[s];
    return;
  }
  const long long recent_from = (long long)a.seen[seq] - a.recent;
  const int items = (n + ranks * THREADS - 1) / (ranks * THREADS);  // at most ITEMS
  const int first = (rank * WARPS + warp) * 32 * items + lane;      // this lane's slots: 32 apart
  uint32_t key[ITEMS];
  {
    float wv[ITEMS];  // all on their way before the first is used
    int pv[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
      const int s = min(first + 32 * i, n - 1);
      wv[i] = 0.f, pv[i] = 0;
      if (i < items) wv[i] = w[s], pv[i] = pos[s];
    }
#pragma unroll
    for (int i = 0; i < ITEMS; i++) key[i] = ev_key(wv[i], pv[i], a.sinks, recent_from);
  }
  for (int i = t; i < 512; i += THREADS) hist[0][i] = 0;
  int* pages = pairs + 2 * a.most;
  if (a.moves_here)
    for (int i = t; i < (n + 15) / 16; i += THREADS) pages[i] = a.page_table[seq * a.max_pages + i];
  const int mine = first - lane < n ? min(items, (n - first + 31) / 32) : 0;  // slots of this lane (may be 0)
  __syncthreads();
  // the left-th largest key, and how many of those that share its digits stay
  uint32_t border = 0, mask = 0;
  unsigned need = (unsigned)left;
  bool all = false;  // all of them stay
  for (int shift = 24; shift >= 0 && !all; shift -= 8) {
    const int turn = shift >> 3 & 1;
    unsigned* h = hist[turn];
#pragma unroll
    for (int i = 0; i < ITEMS; i++)
      if (i < mine && (key[i] & mask) == border) atomicAdd(&h[ev_bin(key[i] >> shift & 255)], 1u);
    if (ranks > 1) {
      cluster.sync();
      for (int i = t; i < 256; i += THREADS) {
        unsigned sum = 0;
#pragma unroll 4
        for (int r = 0; r < ranks; r++) sum += *cluster.map_shared_rank(&h[i], r);
        merged[i] = sum;
      }
      h = merged;
    }
    __syncthreads();
    if (warp == 0) {  // eight digits a lane, from the highest down
      unsigned c[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        c[i] = h[ev_bin(255 - lane * 8 - i)];
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
          if (above < need && need <= above + c[i])
            s_digit[turn] = 255 - lane * 8 - i, s_need[turn] = need - above, s_all[turn] = c[i] == need - above;
          above += c[i];
        }
      }
    }
    // the other counts are clear before the next digit: nobody reads them since the blocks met
    for (int i = t; i < 256; i += THREADS) hist[turn ^ 1][i] = 0;
    __syncthreads();
    border |= s_digit[turn] << shift, mask |= 255u << shift, need = s_need[turn], all = s_all[turn] != 0;
  }
  // keys of the same digits as the border's: all stay, or the first `need` in slot order
  const unsigned under = (1u << lane) - 1;
  int ties = 0;
  if (!all) {
#pragma unroll
    for (int i = 0; i < ITEMS; i++) ties += __popc(__ballot_sync(0xffffffffu, i < mine && key[i] == border));
    const int2 x = ev_before<WARPS>(ties, scratch[0]);
    ties = x.x;
    if (ranks > 1) {
      if (t == 0) shared_counts.x = x.y;
      cluster.sync();
      if (t < ranks) all_counts[t].x = cluster.map_shared_rank(&shared_counts, t)->x;
      __syncthreads();
      for (int r = 0; r < rank; r++) ties += all_counts[r].x;
    }
  }
  unsigned kept = 0;  // of this lane's slots
  int holes = 0, movers = 0;
#pragma unroll
  for (int i = 0; i < ITEMS; i++) {
    bool k;
    if (all) {
      k = i < mine && (key[i] & mask) >= border;
    } else {
      const unsigned tie = __ballot_sync(0xffffffffu, i < mine && key[i] == border);
      k = i < mine && (key[i] > border || (key[i] == border && ties + __popc(tie & under) < (int)need));
      ties += __popc(tie);
    }
    const int s = first + 32 * i;
    if (k) kept |= 1u << i;
    holes += __popc(__ballot_sync(0xffffffffu, i < mine && s < left && !k));
    movers += __popc(__ballot_sync(0xffffffffu, k && s >= left));
  }
  const int2 both = ev_before<WARPS>(holes | movers << 16, scratch[1]);  // a block's are under 2^15 each
  holes = both.x & 0xffff, movers = both.x >> 16;
  int total = both.y & 0xffff;
  if (ranks > 1) {
    if (t == 0) shared_counts.y = total, shared_counts.z = both.y >> 16;
    cluster.sync();
    if (t < ranks) all_counts[t] = *cluster.map_shared_rank(&shared_counts, t);
    cluster.sync();  // nobody leaves while its counts are read
    total = 0;
    for (int r = 0; r < ranks; r++) {
      const int3 c = all_counts[r];
      if (r < rank) holes += c.y, movers += c.z;
      total += c.y;
    }
  }
  const bool copies = a.weights_out != a.weights || a.pos_out != a.pos;
  int* hole_list = a.moves_here ? pairs : a.holes + row * a.most;
  int* mover_list = a.moves_here ? pairs + a.most : a.movers + row * a.most;
#pragma unroll
  for (int i = 0; i < ITEMS; i++) {
    const int s = first + 32 * i;
    const bool k = kept >> i & 1;
    const unsigned hole = __ballot_sync(0xffffffffu, i < mine && s < left && !k);
    const unsigned mover = __ballot_sync(0xffffffffu, k && s >= left);
    if (hole >> lane & 1) hole_list[holes + __popc(hole & under)] = s;
    if (mover >> lane & 1) mover_list[movers + __popc(mover & under)] = s;
    if (k && s < left && copies) wo[s] = w[s], po[s] = pos[s];
    holes += __popc(hole), movers += __popc(mover);
  }
  if (!a.moves_here) {
    if (t == 0 && rank == 0) a.moves[row] = total;
    return;
  }
  __syncthreads();
  const int share = min(32, (total + WARPS - 1) / WARPS);  // moves of a warp at a time
  for (int i0 = warp * share; i0 < total; i0 += WARPS * share) {
    const int moves = min(share, total - i0);
    ev_move<BYTES>(a, row, pages, moves, lane < moves ? pairs[i0 + lane] : 0,
                   lane < moves ? pairs[a.most + i0 + lane] : 0);
  }
}

// The moves of all rows from the workspace, and the lengths, which nobody reads any more. Five blocks an SM: with the
// registers of six, a prompt's cut (288 rows, 2048 moves each) takes 106 us in the place of 102, with eight 114.
template <int BYTES>
__global__ void __launch_bounds__(EV_MOVE_THREADS, 5) evict_move_kernel(EvictArgs a) {
  pdl_wait();
  pdl_trigger();
  const long long row = blockIdx.x;
  const int seq = (int)(row / a.hkv % a.seqs), lane = threadIdx.x & 31;
  if (!a.lengths_here && blockIdx.y == 0 && threadIdx.x == 0 && row < (long long)a.seqs * a.hkv && row % a.hkv == 0)
    a.lengths_out[seq] = (int)min((long long)ev_length(a, seq), a.budget);
  if (a.moves_here) return;
  const int count = a.moves[row];
  for (int i0 = (blockIdx.y * (EV_MOVE_THREADS / 32) + threadIdx.x / 32) * 32; i0 < count;
       i0 += gridDim.y * EV_MOVE_THREADS) {
    const int moves = min(32, count - i0);
    ev_move<BYTES>(a, row, a.page_table + seq * a.max_pages, moves, lane < moves ? a.holes[row * a.most + i0 + lane] : 0,
                                        lane < moves ? a.movers[row * a.most + i0 + lane] : 0);
  }
}

template <int THREADS, int ITEMS, int BLOCKS, int BYTES>
int launch_evict_select(const EvictArgs& a, long long rows, int ranks, cudaStream_t st) {
  // at most EV_HERE moves and EV_RUN / 16 pages: 12 KB
  const int smem = a.moves_here ? (int)(2 * a.most + (a.cap + 15) / 16) * 4 : 0;
  const int rc = configure<evict_select_kernel<THREADS, ITEMS, BLOCKS, BYTES>>("evict_select_kernel", 0, true);
  if (rc != IM_OK) return rc;
  return launch_cluster("evict_select_kernel", evict_select_kernel<THREADS, ITEMS, BLOCKS, BYTES>,
                        dim3((unsigned)(rows * ranks)), dim3(THREADS), ranks, smem, st, a);
}

static long long evict_most(int64_t cap, int64_t budget) { return budget < cap - budget ? budget : cap - budget; }

// Whether a row's moves are made by its own block. Up to 777 moves a row of 624 rows: 20.0 us so, 22.6 by a second kernel; up
// to 2048 of 288 rows: 112 and 102 us. With fewer rows than SMs a row's moves are spread sooner.
static bool evict_here(long long rows, long long cap, long long most) {
  return cap <= EV_RUN && most <= (rows >= 148 ? EV_HERE : 128);
}

static bool evict_fits(int64_t layers, int64_t S, int64_t Hkv, int64_t cap) {
  return layers >= 1 && S >= 1 && Hkv >= 1 && cap >= 1 && cap <= EV_CLUSTER * EV_RUN && layers < (1 << 27) &&
         S < (1 << 27) && Hkv < (1 << 27) && layers * S < (1 << 27) && layers * S * Hkv < (1 << 27);
}

template <int BYTES>
int launch_evict(EvictArgs& a, long long rows, cudaStream_t st) {
  a.moves_here = evict_here(rows, a.cap, a.most);
  a.lengths_here = a.lengths_out != a.lengths;
  const int chunks = 2 * (a.row_bytes / BYTES);
  a.chunk_shift = (chunks & (chunks - 1)) == 0 ? __builtin_ctz(chunks) : -1;
  // blocks a row: as many as its slots need, and more where that leaves SMs idle, down to 2048 slots each (16 rows of 10409
  // slots: 21.5 us with one, 17.5 with four; 24 rows of 17203: 27.7 with two, 21.6 with four)
  int ranks = 1;
  while ((long long)ranks * EV_RUN < a.cap) ranks *= 2;
  while (!a.moves_here && ranks < EV_CLUSTER && rows * ranks * 2 <= 148 && a.cap >= ranks * 2 * 2048) ranks *= 2;
  const long long run = (a.cap + ranks - 1) / ranks;
  const int rc = run <= 2048   ? launch_evict_select<256, 8, 4, BYTES>(a, rows, ranks, st)
                 : run <= 4096 ? launch_evict_select<512, 8, 2, BYTES>(a, rows, ranks, st)
                 : run <= 8192 ? launch_evict_select<512, 16, 2, BYTES>(a, rows, ranks, st)
                               : launch_evict_select<1024, 16, 1, BYTES>(a, rows, ranks, st);
  if (rc != IM_OK || (a.moves_here && a.lengths_here)) return rc;
  const long long blocks = a.moves_here || a.most <= 0 ? 1 : (a.most + EV_MOVE_THREADS - 1) / EV_MOVE_THREADS;
  return launch("evict_move_kernel", evict_move_kernel<BYTES>,
                dim3((unsigned)rows, (unsigned)(blocks < 1024 ? blocks : 1024)), dim3(EV_MOVE_THREADS), 0, st, a);
}

}  // namespace im

using namespace im;

extern "C" size_t im_cache_evict_workspace_bytes(int64_t layers, int64_t S, int64_t Hkv, int64_t cap, int64_t budget) {
  if (!evict_fits(layers, S, Hkv, cap) || budget < 0) return 0;
  const long long rows = layers * S * Hkv, most = evict_most(cap, budget) > 0 ? evict_most(cap, budget) : 0;
  return evict_here(rows, cap, most) ? 0 : (size_t)(rows * 4 + 2 * rows * most * 4);
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
  IM_REQUIRE(aligned(page_table, 4) && aligned(lengths, 4) && aligned(seen, 4) && aligned(weights, 4) &&
                 aligned(weights_out, 4) && aligned(slot_pos, 4) && aligned(pos_out, 4) && aligned(lengths_out, 4),
             IM_INVALID, "im_cache_evict: misaligned pointer");
  IM_REQUIRE(evict_fits(layers, S, Hkv, cap) && row_bytes <= (1 << 16), IM_UNSUPPORTED,
             "im_cache_evict: rows of %lld slots (up to %d) of %lld bytes (up to 65536), or too many of them", (long long)cap,
             EV_CLUSTER * EV_RUN, (long long)row_bytes);
  const size_t need = im_cache_evict_workspace_bytes(layers, S, Hkv, cap, budget);
  IM_REQUIRE(need == 0 || (workspace && aligned(workspace, 16) && workspace_bytes >= need), IM_INVALID,
             "im_cache_evict: a workspace of %zu bytes needed, %zu given", need, workspace_bytes);
  IM_REQUIRE(lengths_out != seen, IM_INVALID, "im_cache_evict: lengths_out is seen");
  const long long rows = layers * S * Hkv, most = evict_most(cap, budget);
  EvictArgs a = {};
  a.k = (char*)k_cache, a.v = (char*)v_cache, a.layer_bytes = layer_bytes, a.pages = pages;
  a.page_table = page_table, a.max_pages = max_pages, a.lengths = lengths, a.seen = seen;
  a.weights = weights, a.weights_out = weights_out, a.pos = slot_pos, a.pos_out = pos_out, a.lengths_out = lengths_out;
  a.seqs = (int)S, a.hkv = (int)Hkv, a.cap = cap, a.row_bytes = (int)row_bytes;
  a.budget = budget, a.recent = recent, a.sinks = sinks;
  a.most = most > 0 ? most : 0, a.moves = (int*)workspace, a.holes = a.moves + rows, a.movers = a.holes + rows * a.most;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (row_bytes % 16 == 0 && aligned(k_cache, 16) && aligned(v_cache, 16) && layer_bytes % 16 == 0)
    return launch_evict<16>(a, rows, st);
  return launch_evict<1>(a, rows, st);
}
