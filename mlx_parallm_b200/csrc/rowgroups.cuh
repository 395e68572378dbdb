// Rows of a batch grouped by an index of each (b200p_row_groups): what the kernels that work group by group read of the plan.
//   int32: [0] tiles, [1] rows in groups, [2] rows whose index is behind the last group, [3] rows of a tile at most
//          [4, 4 + M) rows in the order of their groups (the batch's order within a group), filled up to a multiple of 4
//          then per tile: group, first place in that order, rows, first place of the group
#pragma once
#include "common.cuh"

namespace b200p {

constexpr int RG_HEAD = 4;
constexpr int RG_GROUPS = 1024;                  // groups at most
constexpr int64_t RG_ROWS = 1 << 20;

static inline int64_t row_group_tiles(int64_t M, int64_t groups, int64_t tile) { return M / tile + (groups < M ? groups : M); }      // at most
static inline int64_t row_group_ints(int64_t M, int64_t groups, int64_t tile) { return RG_HEAD + (M + 3) / 4 * 4 + 4 * row_group_tiles(M, groups, tile); }

struct RowGroups {
  const int32_t* plan;
  int M;
  __device__ int tiles() const { return plan[0]; }
  __device__ const int32_t* order() const { return plan + RG_HEAD; }
  __device__ int4 tile(int i) const { return *reinterpret_cast<const int4*>(plan + RG_HEAD + (M + 3) / 4 * 4 + 4 * (int64_t)i); }
};

}  // namespace b200p
