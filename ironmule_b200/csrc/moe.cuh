// Shared by the mixture-of-experts kernels: the routing plan that im_moe_route writes and the products read.
#pragma once

#include <cstddef>
#include <cstdint>

#include <cuda_runtime.h>

namespace im {

constexpr int MOE_MAX_EXPERTS = 512;
constexpr int MOE_MAX_TOP_K = 32;
constexpr int64_t MOE_MAX_ROWS = 1 << 22;
constexpr int MOE_ROUTE_BLOCKS = 148;   // blocks of the routing kernels at most (one per SM)
constexpr int MOE_ROUTE_ROWS = 64;      // rows that one block alone routes
constexpr int MOE_TC_ROWS = 128;        // rows of a work item on the tensor-core kernel
constexpr int MOE_PLAN_HEADER = 8;      // ints: [0] work items, [1] error word of the bounded waits

// Packed weights of an expert: 128-output blocks (rows past N are zero), each a run of 64-wide groups of
// MOE_BLOCK_BYTES = 4 tiles of 32 rows x (two 16-byte halves a row, [half][row]) of codes, then per tile 128 bytes of
// scales and biases: for g = 0..7 the bf16 scales of rows g, g + 8, g + 16, g + 24, then their biases. One copy brings
// a block's group; a thread reads its row's codes in two 16-byte loads without bank conflicts, and a warp-MMA lane the
// 8 bytes of each of its four rows. After the E experts: float32 [E][padded rows], the
// largest |scale * q + bias| that a row's scales and biases allow; float32 [E][2], the largest over an expert's rows
// with r & 16 == 0 (the gate rows of a gated product) and over the others (the up rows).
constexpr int MOE_BLOCK_BYTES = 4608;

// One work item: `rows` consecutive entries of the sorted pair list, all of one expert (or, with expert == E, of the
// places that chose no expert, whose outputs are zero).
struct MoeItem {
  int expert, first, rows, padded;  // padded: the rows before it when every item is rounded up to 16
};

// Plan layout in ints: header | items | per-block expert counts (the routing's own scratch).
struct MoePlan {
  int64_t item_rows;   // most rows of an item; 8, 16, 32: the warp-MMA kernel, MOE_TC_ROWS: the tensor-core kernel
  int64_t max_items;   // bound on the items of any routing of these sizes
  int64_t blocks, rows_per_block;
  int64_t counts;      // int offset of the counts
  size_t bytes;
};

// path: IM_MOE_AUTO, IM_MOE_WARP, IM_MOE_TENSOR
MoePlan moe_plan(int64_t M, int64_t E, int64_t top_k, int path);

// Where a product's input and output rows are: by token (pair / top_k), by pair, or by position in the sorted list.
enum MoeRows { MOE_BY_TOKEN = 0, MOE_BY_PAIR = 1, MOE_SORTED = 2 };

struct MoeProduct {
  const unsigned char* wp;  // [E] matrices in packed units
  const uint16_t* x;
  uint16_t* y;
  const int* plan;
  const int* pairs;
  int M, E, top_k, N, K;
  int src, dst;   // MoeRows
  int epilogue;   // IM_EPI_STORE, IM_EPI_SWIGLU, IM_EPI_GEGLU
  int early;      // the plan was finished before the preceding launch began: items and weights may be read before
                  // the dependency wait
};

// Byte offsets in the workspace of the tensor-core path.
struct MoeTcSpace {
  size_t tiles, scale, xlog, next, hscale, total;
};
MoeTcSpace moe_tc_space(const MoePlan& p, int64_t pairs, int64_t K, int64_t I);
int moe_prep_launch(const MoePlan& p, const MoeProduct& a, const MoeTcSpace& s, void* workspace, cudaStream_t st);
int moe_tc_launch(const MoePlan& p, const MoeProduct& a, const MoeTcSpace& s, void* workspace, cudaStream_t st);
int moe_mma_launch(const MoePlan& p, const MoeProduct& a, cudaStream_t st);

}  // namespace im
