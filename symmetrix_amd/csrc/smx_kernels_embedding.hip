// Rows of a table by index, scaled, and the table's gradient.
//
//   y_i = scale table[index_i],   dtable_t = scale sum over the rows with index t of dy_i
//
// Forward: neighbouring threads take neighbouring 16 bytes of a row, a thread four rows at a time.  Gradient: rows sorted by entry, then
// a wavefront for every entry and 1 KB of its row.
//
// Bound by memory.
#include "smx_groups.hpp"

#include <limits>

namespace smx {

namespace {

struct Lookup {
    const void* table;
    long table_stride;
    const int* index;
    void* y;
    long y_stride;
    long rows;
    int entries, dim, lanes;      // lanes: threads of a row, a power of two
    float scale;
};
constexpr int kLookupRows = 4;      // of a thread
template <typename T>
__global__ __launch_bounds__(256) void k_lookup(const Lookup p)
{
    constexpr int V = kRun<T>;
    const int at_once = 256 / p.lanes, mine = threadIdx.x / p.lanes, lane = threadIdx.x % p.lanes;
    const long row0 = (long)blockIdx.x * (kLookupRows * at_once) + mine;
    int t[kLookupRows];
#pragma unroll
    for (int u = 0; u < kLookupRows; ++u) t[u] = p.index[min(row0 + u * at_once, p.rows - 1)];
    for (int at = lane * V; at < p.dim; at += p.lanes * V) {
        float v[kLookupRows][V];
#pragma unroll
        for (int u = 0; u < kLookupRows; ++u) {
            const bool has = (unsigned)t[u] < (unsigned)p.entries;
            const float other = t[u] == -1 ? 0.0f : std::numeric_limits<float>::quiet_NaN();
            if (has) load_run<V>(static_cast<const T*>(p.table) + t[u] * p.table_stride + at, p.dim - at, v[u]);
#pragma unroll
            for (int j = 0; j < V; ++j) v[u][j] = has ? v[u][j] * p.scale : other;
        }
#pragma unroll
        for (int u = 0; u < kLookupRows; ++u)
            if (row0 + u * at_once < p.rows) store_run<V>(static_cast<T*>(p.y) + (row0 + u * at_once) * p.y_stride + at, p.dim - at, v[u]);
    }
}

struct Sums {
    const void* dy;
    long dy_stride;
    const int *order, *offsets;
    void* dtable;
    int entries, dim, slabs;
    float scale;
};
template <typename T>
__global__ __launch_bounds__(256) void k_entry_sums(const Sums p)
{
    constexpr int V = kRun<T>;
    const long item = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int t = (int)(item / p.slabs), at = (int)(item % p.slabs) * 64 * V + (threadIdx.x & 63) * V;
    if (t >= p.entries || at >= p.dim) return;
    const int begin = p.offsets[t], end = p.offsets[t + 1];
    float sum[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = 0.0f;
    for (int i = begin; i < end; ++i) {
        float v[V];
        load_run<V>(static_cast<const T*>(p.dy) + p.order[i] * p.dy_stride + at, p.dim - at, v);
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] += v[j];
    }
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] *= p.scale;
    store_run<V>(static_cast<T*>(p.dtable) + (long)t * p.dim + at, p.dim - at, sum);
}

// ---- host side

void check(long rows, int entries, int dim)
{
    refuse_unless(rows >= 0 && rows <= 1L << 28, "rows: 0 to 2^28");
    refuse_unless(entries >= 0 && entries <= SMX_MOST_ENTRIES, "entries: 0 to 2^24");
    refuse_unless(dim >= 1 && dim <= 1 << 20, "dim: 1 to 2^20");
}

struct Call : Launches {
    Arena arena;
    template <typename T>
    void backward(long rows, int entries, int dim, const T* dy, long dy_stride, const int* index, const int* order, const int* offsets, float scale, T* dtable)
    {
        constexpr int V = kRun<T>;
        if (!order) {
            const RowOrder sorted{arena.take<int>(rows), arena.take<int>(entries + 2L), nullptr};
            sort_rows(*this, arena, index, rows, entries, sorted);
            order = sorted.order;
            offsets = sorted.offsets;
        }
        const int slabs = (dim + 64 * V - 1) / (64 * V);
        start(k_entry_sums<T>, ((long)entries * slabs + 3) / 4, 1, 1, 256, 0, Sums{dy, dy_stride, order, offsets, dtable, entries, dim, slabs, scale});
    }
};
long workspace(int type, long rows, int entries, int dim)
{
    Call c{{nullptr, true}, {reinterpret_cast<char*>(256)}};
    with_type(type, [&](auto t) { c.backward<decltype(t)>(rows, entries, dim, nullptr, dim, nullptr, nullptr, nullptr, 1.0f, nullptr); });
    return c.arena.used;
}

}  // namespace

}  // namespace smx

using namespace smx;

extern "C" int smx_embedding_forward(int type, long rows, int entries, int dim, const void* d_table, long table_stride, const int* d_index, double scale, void* d_y,
                                     long y_stride, void* stream)
{
    return finetune_entry("smx_embedding_forward", [&] {
        (void)type_bytes(type);
        check(rows, entries, dim);
        if (rows == 0) return;
        refuse_unless(d_index && d_y && (d_table || entries == 0), "table, index and y must not be null");
        refuse_unless(table_stride >= dim && y_stride >= dim, "strides of table and y: at least dim");
        require_gfx950();
        Launches launches{static_cast<hipStream_t>(stream), false};
        with_type(type, [&](auto t) {
            using T = decltype(t);
            int lanes = 1;
            while (lanes < 256 && lanes * kRun<T> < dim) lanes *= 2;
            const long per_block = kLookupRows * (256 / lanes);
            Launches::in_slabs((rows + per_block - 1) / per_block, [&](long first, long some) {
                const long row = first * per_block;
                launches.start(k_lookup<T>, some, 1, 1, 256, 0,
                               Lookup{d_table, table_stride, d_index + row, static_cast<T*>(d_y) + row * y_stride, y_stride, rows - row, entries, dim, lanes, (float)scale});
            });
        });
        hip_ok(hipGetLastError(), "launch");
    });
}

extern "C" int smx_embedding_backward_workspace(int type, long rows, int entries, int dim, long* bytes)
{
    return finetune_entry("smx_embedding_backward_workspace", [&] {
        (void)type_bytes(type);
        check(rows, entries, dim);
        refuse_unless(bytes, "bytes must not be null");
        *bytes = entries ? workspace(type, rows, entries, dim) : 0;
    });
}

extern "C" int smx_embedding_backward(int type, long rows, int entries, int dim, const void* d_dy, long dy_stride, const int* d_index,
                                      const int* d_order, const int* d_offsets, double scale, void* d_dtable, void* d_workspace, long workspace_bytes, void* stream)
{
    return finetune_entry("smx_embedding_backward", [&] {
        (void)type_bytes(type);
        check(rows, entries, dim);
        if (entries == 0) return;
        refuse_unless(d_dtable && (rows == 0 || (d_dy && d_index)), "dy, index and dtable must not be null");
        refuse_unless(dy_stride >= dim, "the stride of dy: at least dim");
        refuse_unless((d_order == nullptr) == (d_offsets == nullptr) || rows == 0, "order and offsets: both or neither");
        if (rows == 0) d_order = d_offsets = nullptr;
        check_workspace(d_workspace, workspace_bytes, workspace(type, rows, entries, dim), "smx_embedding_backward_workspace");
        require_gfx950();
        Call c{{static_cast<hipStream_t>(stream), false}, {static_cast<char*>(d_workspace)}};
        with_type(type, [&](auto t) {
            using T = decltype(t);
            c.backward<T>(rows, entries, dim, static_cast<const T*>(d_dy), dy_stride, d_index, d_order, d_offsets, (float)scale, static_cast<T*>(d_dtable));
        });
        hip_ok(hipGetLastError(), "launch");
    });
}
