// Rows sorted by group: what the kernels that sum over the rows of a group, or take a group's rows together, go by.
#pragma once

#include "smx_finetune.hpp"

namespace smx {

// key of a row in the sorted order: its group, or behind the groups: no group (-1), an index out of range
__device__ __forceinline__ int row_key(int index, int groups) { return (unsigned)index < (unsigned)groups ? index : (index == -1 ? groups : groups + 1); }

// first place in sorted keys that holds `key` or more
__device__ __forceinline__ int first_place(const int* keys, int n, int key)
{
    int low = 0;
    while (n > 0) {
        const int half = n / 2;
        if (keys[low + half] < key) low += half + 1, n -= half + 1;
        else n = half;
    }
    return low;
}

struct RowOrder {
    int* order;        // [rows]
    int* offsets;      // [groups + 2]; NULL: not asked for
    int* keys;         // [rows], sorted; NULL: not asked for
};
// Whether the sort writes offsets without a launch for them.
bool sort_has_offsets(long rows, int groups);
// Memory that is filled with zeros beside the sort, which leaves most of the card idle.
struct Zeros {
    char* at = nullptr;      // a multiple of 2, as bytes is
    long bytes = 0;
};
// Enqueues the sort; what it needs beside its results comes from the arena.
void sort_rows(Launches& launches, Arena& arena, const int* index, long rows, int groups, const RowOrder& to, const Zeros& zeros = {});

// out[group][dim] = scale times the sum of the group's rows of in, and zeros where it has none; in `type`.  The rows' order in the
// sums is theirs.  sorted.order null: the rows are sorted here.
void add_rows(Launches& launches, Arena& arena, int type, const void* in, long in_stride, const int* index, long rows, int groups, int dim, RowOrder sorted, float scale, void* out);

}  // namespace smx
