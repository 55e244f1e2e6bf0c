// Rows sorted by group: what the kernels that sum over the rows of a group, or take a group's rows together, go by.
#pragma once

#include "smx_finetune.hpp"

namespace smx {

// key of a row in the sorted order: its group, or behind the groups: no group (-1), an index out of range
__device__ __forceinline__ int row_key(int index, int groups) { return (unsigned)index < (unsigned)groups ? index : (index == -1 ? groups : groups + 1); }

struct RowOrder {
    int* order;        // [rows]
    int* offsets;      // [groups + 2]; NULL: not asked for
    int* keys;         // [rows], sorted; NULL: not asked for
};
// Enqueues the sort; what it needs beside its results comes from the arena.
void sort_rows(Launches& launches, Arena& arena, const int* index, long rows, int groups, const RowOrder& to);

}  // namespace smx
