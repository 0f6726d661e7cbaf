// Shared by the mixture-of-experts kernels: the routing plan that im_moe_route writes and the products read.
#pragma once

#include <cstddef>
#include <cstdint>

#include <cuda_runtime.h>

namespace im {

constexpr int MOE_MAX_EXPERTS = 512;
constexpr int MOE_MAX_TOP_K = 32;
constexpr int64_t MOE_MAX_ROWS = 1 << 22;
constexpr int MOE_ROUTE_BLOCKS = 296;   // blocks of the routing kernels at most (two per SM)
constexpr int MOE_ROUTE_ROWS = 64;      // rows that one block alone routes
constexpr int MOE_ITEM_ROWS = 128;      // rows of a work item at most (MMA N)
constexpr int MOE_PLAN_HEADER = 8;      // ints: [0] work items, [1] error word of the bounded waits, [2..3] the address
                                        // of the caller's own error word (0: none)

// Packed weights of an expert: 128-output blocks (rows past N are zero), each a run of 64-wide groups of
// MOE_BLOCK_BYTES = 4 tiles of 32 rows x (two 16-byte halves a row, [half][row]) of codes, then per tile 128 bytes of
// scales and biases: for g = 0..7 the bf16 scales of rows g, g + 8, g + 16, g + 24, then their biases. One copy brings
// a block's group; a thread reads its row's codes in two 16-byte loads without bank conflicts. After the E experts:
// float32 [E][padded rows], the largest |scale * q + bias| that a row's scales and biases allow; float32 [E][2], the
// largest 2-norm of an expert's rows with r & 16 == 0 (the gate rows of a gated product) and of the others (the up rows).
constexpr int MOE_BLOCK_BYTES = 4608;

// One work item (four ints): the expert, the first of its entries in the sorted pair list, their number, and the rows
// before it when every item is rounded up to 16. Items of expert E are places that chose none; their outputs are zero.
//
// Plan layout in ints: header | items | where each pair's row lies | per-block expert counts (the routing's own scratch).
// where[pair] = {the item's padded first row (-1: no expert), its row r in the item | the item's rows rounded up to 16
// << 16}.
struct MoePlan {
  int64_t max_items;   // bound on the items of any routing of these sizes
  int64_t blocks, rows_per_block;
  int64_t where;       // int offsets
  int64_t counts;
  size_t bytes;
};

MoePlan moe_plan(int64_t M, int64_t E, int64_t top_k);

struct MoeProduct {
  const unsigned char* wp;  // [E] packed matrices
  uint16_t* y;              // [M, top_k, N], or unused by the first product of a gated MLP
  const int* plan;
  const int* pairs;
  int M, E, top_k, N, K;
  int epilogue;             // IM_EPI_STORE, IM_EPI_SWIGLU, IM_EPI_GEGLU
  bool second;              // its rows are the gated activations that the first product left in the workspace
};

// Byte offsets in the products' workspace.
struct MoeSpace {
  size_t tiles, scale, xlog, next, hscale, total;
};
MoeSpace moe_space(const MoePlan& p, int64_t pairs, int64_t K, int64_t I);
// x [M, K], or [M, top_k, K] with by_pair, into the workspace's operand tiles.
int moe_prep_launch(const MoePlan& p, const MoeProduct& a, const uint16_t* x, int by_pair, const MoeSpace& s,
                    void* workspace, cudaStream_t st);
int moe_product_launch(const MoePlan& p, const MoeProduct& a, const MoeSpace& s, void* workspace, cudaStream_t st);

}  // namespace im
