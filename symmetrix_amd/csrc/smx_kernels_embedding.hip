// Rows of a table by index, scaled, and the table's gradient.
//
//   y_i = scale table[index_i],   dtable_t = scale sum over the rows with index t of dy_i
//
// Forward: neighbouring threads take neighbouring 16 bytes of a row, a thread four rows at a time.  Gradient: rows sorted by entry, cut
// into pieces of equal length whatever their entries (an entry may have one row, or all), and a second launch for the entries that lie in
// several pieces and for those without a row.
//
// Bound by memory.  32 749 rows of 4 096 in bfloat16 looked up: 74 us, 5.9 TB/s of what has to move (81 a call; 91 with results by way of the caches).
#include "smx_groups.hpp"

#include <cmath>
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
constexpr long kMuch = 64L << 20;   // bytes of a result that are written past the caches
template <typename T, bool PAST>
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
            if (row0 + u * at_once < p.rows) {
                T* y = static_cast<T*>(p.y) + (row0 + u * at_once) * p.y_stride + at;
                if (PAST && p.dim - at >= V) store_past<V>(y, v[u]);
                else store_run<V>(y, p.dim - at, v[u]);
            }
    }
}

// ---- sums of rows by group

struct Sums {
    const void* in;
    long in_stride;
    const int *index, *order;
    const int* keys;           // sorted, or null: those of index
    int* offsets;              // written by blocks behind the pieces' where they are not there yet
    long rows;
    int groups, dim, slabs, piece;
    long pieces;
    float* partial;            // [piece][0: of a run of rows that began before the piece, 1: that goes on behind it][dim]
    float scale;
    void* out;
    bool by_piece;             // of k_join_pieces
    long first;                // which of all blocks the launch's first one is
};

// Pieces of sorted rows: a block's four wavefronts have a quarter of a piece each, and 1 KB of its rows.  A group's rows that lie in one
// piece are summed and stored; of a group that goes on in other pieces, a part.  Eight rows are under way at a time.
// 50 000 rows of 256, 89 entries, single precision: 10.5 us, 4.9 TB/s; 16 381 of 2 048, 32 000 entries in bfloat16: 18, 6 TB/s with the sums written.
template <typename T>
__global__ __launch_bounds__(256) void k_pieces(const Sums p)
{
    constexpr int V = kRun<T>, U = 8;
    __shared__ float head[4][64][V], tail[4][64][V];      // of a quarter: the run that began before it, the one that goes on behind it
    __shared__ int key_of[4][2];                          // their keys, or -1
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long blocks = p.pieces * p.slabs, block = p.first + blockIdx.x;
    if (block >= blocks) {      // (offsets)
        const int g = (int)(block - blocks) * 256 + threadIdx.x;
        if (g < p.groups + 2) p.offsets[g] = first_place(p.keys, (int)p.rows, g);
        return;
    }
    const long piece = block / p.slabs;
    const int at = (int)(block % p.slabs) * 64 * V + lane * V, quarter = p.piece / 4;
    const long begin = piece * p.piece + wave * quarter;
    const int count = (int)max(0L, min((long)quarter, p.rows - begin));
    const bool whole = at + V <= p.dim, some = at < p.dim;
    auto finish = [&](int key, float (&sum)[V]) {
        if (!some) return;
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] *= p.scale;
        store_run<V>(static_cast<T*>(p.out) + (long)key * p.dim + at, p.dim - at, sum);
    };
    int head_key = -1, tail_key = -1;
    if (count > 0) {
        auto key_at = [&](long i, int row) { return p.keys ? p.keys[i] : row_key(p.index[row], p.groups); };
        const int my_row = p.order[begin + min(lane, count - 1)];
        const int my_key = key_at(begin + min(lane, count - 1), my_row);
        const int before = begin > 0 ? key_at(begin - 1, p.keys ? 0 : p.order[begin - 1]) : -1;
        const int behind = begin + count < p.rows ? key_at(begin + count, p.keys ? 0 : p.order[begin + count]) : -1;
        const T* in = static_cast<const T*>(p.in) + at;
        float sum[V];
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] = 0.0f;
        int key = __builtin_amdgcn_readlane(my_key, 0);
        bool entered = key == before;
        auto flush = [&](bool leaves) {
            if (entered) {
                head_key = key;
#pragma unroll
                for (int j = 0; j < V; ++j) head[wave][lane][j] = sum[j];
            } else if (leaves) {
                tail_key = key;
#pragma unroll
                for (int j = 0; j < V; ++j) tail[wave][lane][j] = sum[j];
            } else finish(key, sum);
        };
#pragma unroll 1
        for (int i0 = 0; i0 < count && key < p.groups; i0 += U) {      // (what lies behind the groups belongs to none)
            typename Operand<T>::type x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long row = __builtin_amdgcn_readlane(my_row, min(i0 + u, count - 1));
                if (whole) x[u] = *reinterpret_cast<const typename Run<T, V>::loose*>(in + row * p.in_stride);
                else x[u] = load_operand(in + (some ? row * p.in_stride : 0), p.dim - at);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (i0 + u >= count || key >= p.groups) break;
                const int k = __builtin_amdgcn_readlane(my_key, i0 + u);
                if (k != key) {
                    flush(false);
#pragma unroll
                    for (int j = 0; j < V; ++j) sum[j] = 0.0f;
                    key = k;
                    entered = false;
                }
#pragma unroll
                for (int j = 0; j < V; ++j) sum[j] += (float)x[u][j];
            }
        }
        if (key < p.groups) {
            flush(key == behind);
            if (entered && key == behind) tail_key = key;      // (a run that fills the quarter and goes on: its sum is in head)
        }
    }
    if (lane == 0) {
        key_of[wave][0] = head_key;
        key_of[wave][1] = tail_key;
    }
    __syncthreads();
    if (wave > 0) return;
    // runs over several quarters, by the first wavefront
    float sum[V];
    int key = -1;
    bool entered = false;
    for (int w = 0; w < 4; ++w) {
        const int h = __builtin_amdgcn_readfirstlane(key_of[w][0]), t = __builtin_amdgcn_readfirstlane(key_of[w][1]);
        if (h >= 0) {
            if (key < 0) {
                entered = true;
#pragma unroll
                for (int j = 0; j < V; ++j) sum[j] = head[w][lane][j];
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) sum[j] += head[w][lane][j];
            }
            key = h;
            if (t == h) continue;
            if (entered) {
                if (some) store_run<V>(p.partial + 2 * piece * p.dim + at, p.dim - at, sum);
            } else finish(key, sum);
            key = -1;
        }
        if (t >= 0) {
            key = t;
            entered = false;
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] = tail[w][lane][j];
        }
    }
    if (key >= 0 && some) store_run<V>(p.partial + (2 * piece + (entered ? 0 : 1)) * p.dim + at, p.dim - at, sum);
}

// Groups whose rows lie in several pieces: the parts, in order, by 16 wavefronts for 1 KB of a group.  Of many groups (by_piece) a block looks
// at a piece, for the group that goes on behind it and began in it.  Groups without rows: zeros, where they are not there yet; of many
// groups by blocks behind the others, a wavefront up to 4 KB.  (16 381 rows of 32 000 entries, 2 048 in bfloat16, half of them of one
// entry: 56 us, and 203 with a wavefront for a group's parts.)
template <typename T>
__global__ __launch_bounds__(1024) void k_join_pieces(const Sums p)
{
    constexpr int V = kRun<T>, WAVES = 16, SLABS = 4;
    __shared__ float part[WAVES][64][V];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long item = p.first + blockIdx.x, joins = (p.by_piece ? p.pieces : (long)p.groups) * p.slabs;
    float sum[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = 0.0f;
    if (item >= joins) {
        const int each = (p.slabs + SLABS - 1) / SLABS;
        const long mine = (item - joins) * WAVES + wave, g = mine / each;
        if (g >= p.groups || p.offsets[g] != p.offsets[g + 1]) return;
#pragma unroll
        for (int s = 0; s < SLABS; ++s) {
            const int at = ((int)(mine % each) * SLABS + s) * 64 * V + lane * V;
            if (at < p.dim) store_run<V>(static_cast<T*>(p.out) + g * p.dim + at, p.dim - at, sum);
        }
        return;
    }
    const int which = (int)(item / p.slabs), at = (int)(item % p.slabs) * 64 * V + lane * V;
    int g = which;
    if (p.by_piece) {
        const long last = min((which + 1L) * p.piece, p.rows) - 1;
        g = p.keys ? p.keys[last] : row_key(p.index[p.order[last]], p.groups);
        if (g >= p.groups) return;
    }
    const int begin = p.offsets[g], end = p.offsets[g + 1];
    const int first = begin / p.piece, last = end > begin ? (end - 1) / p.piece : first;
    if (p.by_piece ? first != which || last == which : end > begin && first == last) return;      // (the same in all wavefronts)
    if (end == begin && wave > 0) return;
    const bool some = at < p.dim;
    if (end > begin) {
        if (some) {
            // (the first part lies in its piece's second place, the others in the first)
#pragma unroll 8
            for (int k = first + wave; k <= last; k += WAVES) {
                float v[V];
                load_run<V>(p.partial + (2L * k + (k == first ? 1 : 0)) * p.dim + at, p.dim - at, v);
#pragma unroll
                for (int j = 0; j < V; ++j) sum[j] += v[j];
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) part[wave][lane][j] = sum[j];
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int w = 1; w < WAVES; ++w)
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] += part[w][lane][j];
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] *= p.scale;
    }
    if (some) store_run<V>(static_cast<T*>(p.out) + (long)g * p.dim + at, p.dim - at, sum);
}

// Few rows: a wavefront for 1 KB of a group's sum looks through the index by itself.
template <typename T>
__global__ __launch_bounds__(256) void k_few_rows(const Sums p)
{
    constexpr int V = kRun<T>, U = 8;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long item = (p.first + blockIdx.x) * 4 + wave;
    if (item >= (long)p.groups * p.slabs) return;
    const int g = (int)(item / p.slabs), at = (int)(item % p.slabs) * 64 * V + lane * V;
    float sum[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = 0.0f;
    for (int i0 = 0; i0 < p.rows; i0 += 64) {
        unsigned long left = __ballot(i0 + lane < p.rows && p.index[min((long)i0 + lane, p.rows - 1)] == g);
        while (left) {
            float x[U][V];
            int n = 0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int bit = left ? __builtin_ctzl(left) : 64;
                left &= left - 1;
                n += bit < 64;
                const long row = i0 + min(bit, 63);
                if (bit < 64) load_run<V>(static_cast<const T*>(p.in) + row * p.in_stride + at, p.dim - at, x[u]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (u < n)
#pragma unroll
                    for (int j = 0; j < V; ++j) sum[j] += x[u][j];
        }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] *= p.scale;
    store_run<V>(static_cast<T*>(p.out) + (long)g * p.dim + at, p.dim - at, sum);
}

// ---- host side

void check(long rows, int entries, int dim)
{
    refuse_unless(rows >= 0 && rows <= 1L << 28, "rows: 0 to 2^28");
    refuse_unless(entries >= 0 && entries <= SMX_MOST_ENTRIES, "entries: 0 to 2^24");
    refuse_unless(dim >= 1 && dim <= 1 << 20, "dim: 1 to 2^20");
}

// (kernels multiply in single precision)
void check_scale(double scale)
{
    const float f = (float)scale;
    refuse_unless(scale == 0 || (std::isfinite(f) && std::fabs(f) >= std::numeric_limits<float>::min()), "scale: 0 or a normal number of single precision");
}

long workspace(int type, long rows, int entries, int dim)
{
    Launches dry{nullptr, true};
    Arena arena{reinterpret_cast<char*>(256)};
    add_rows(dry, arena, type, nullptr, dim, nullptr, rows, entries, dim, RowOrder{}, 1.0f, nullptr);
    return arena.used;
}

}  // namespace

// Rows up to which a wavefront looks through the index by itself.
constexpr int kMostFew = 128;

void add_rows(Launches& launches, Arena& arena, int type, const void* in, long in_stride, const int* index, long rows, int groups, int dim, RowOrder sorted, float scale, void* out)
{
    with_type(type, [&](auto t) {
        using T = decltype(t);
        constexpr int V = kRun<T>;
        Sums p{};
        p.in = in; p.in_stride = in_stride; p.index = index; p.rows = rows; p.groups = groups; p.dim = dim; p.scale = scale; p.out = out;
        p.slabs = (dim + 64 * V - 1) / (64 * V);
        const long entries = (long)groups * p.slabs;
        auto start = [&](auto kernel, long blocks, int threads) {
            Launches::in_slabs(blocks, [&](long first, long some) {
                p.first = first;
                launches.start(kernel, some, 1, 1, threads, 0, p);
            });
        };
        if (rows <= kMostFew) {
            start(k_few_rows<T>, (entries + 3) / 4, 256);
            return;
        }
        // pieces of 32 to 256 rows, until there are 16 wavefronts for every CU
        p.piece = 32;
        while (p.piece < 256 && rows * p.slabs / p.piece > 1024) p.piece *= 2;
        p.pieces = (rows + p.piece - 1) / p.piece;
        p.partial = arena.take<float>(2 * p.pieces * dim);
        // Of more groups than rows most have none: zeros everywhere, beside the sort, and sums over them.  (16 381 rows of 32 000 entries, 2 048 in
        // bfloat16, nothing in the caches: 62 us, with zeros by the last launch 72; everything there: 60 and 58.)
        const bool filled = !sorted.order && groups >= rows;
        p.by_piece = groups > 4096 || filled;
        long offset_blocks = 0;
        if (!sorted.order) {
            sorted = RowOrder{arena.take<int>(rows), arena.take<int>(groups + 2L), arena.take<int>(rows)};
            // (where the sort has them anyway it writes the offsets; otherwise they are looked for beside the pieces)
            const bool with_offsets = sort_has_offsets(rows, groups);
            sort_rows(launches, arena, index, rows, groups, RowOrder{sorted.order, with_offsets ? sorted.offsets : nullptr, sorted.keys},
                      filled ? Zeros{static_cast<char*>(out), (long)groups * dim * (long)sizeof(T)} : Zeros{});
            if (!with_offsets) offset_blocks = (groups + 2L + 255) / 256;
        }
        p.order = sorted.order; p.offsets = sorted.offsets; p.keys = sorted.keys;
        start(k_pieces<T>, p.pieces * p.slabs + offset_blocks, 256);
        const long zeros = p.by_piece && !filled ? ((p.slabs + 3) / 4 * (long)groups + 15) / 16 : 0;
        start(k_join_pieces<T>, (p.by_piece ? p.pieces : (long)groups) * p.slabs + zeros, 1024);
    });
}

}  // namespace smx

using namespace smx;

extern "C" int smx_embedding_forward(int type, long rows, int entries, int dim, const void* d_table, long table_stride, const int* d_index, double scale, void* d_y,
                                     long y_stride, void* stream)
{
    return finetune_entry("smx_embedding_forward", [&] {
        (void)type_bytes(type);
        check(rows, entries, dim);
        check_scale(scale);
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
                launches.start(rows * dim * (long)sizeof(T) >= kMuch ? k_lookup<T, true> : k_lookup<T, false>, some, 1, 1, 256, 0,
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
        check_scale(scale);
        if (entries == 0) return;
        refuse_unless(d_dtable && (rows == 0 || (d_dy && d_index)), "dy, index and dtable must not be null");
        refuse_unless(dy_stride >= dim, "the stride of dy: at least dim");
        refuse_unless((d_order == nullptr) == (d_offsets == nullptr) || rows == 0, "order and offsets: both or neither");
        if (rows == 0) d_order = d_offsets = nullptr;
        check_workspace(d_workspace, workspace_bytes, workspace(type, rows, entries, dim), "smx_embedding_backward_workspace");
        require_gfx950();
        Launches launches{static_cast<hipStream_t>(stream), false};
        Arena arena{static_cast<char*>(d_workspace)};
        add_rows(launches, arena, type, d_dy, dy_stride, d_index, rows, entries, dim, RowOrder{const_cast<int*>(d_order), const_cast<int*>(d_offsets), nullptr},
                 (float)scale, d_dtable);
        hip_ok(hipGetLastError(), "launch");
    });
}
