// Rows sorted by group, stable: a radix sort of (key, row) by digits of up to ten bits, the lowest first.
//
// A digit takes two launches: the digits of every block's rows are counted, and then every block places its rows behind those of
// smaller digits and those of earlier blocks, which it sums up from the counts by itself.  Inside a wavefront the rows of a digit find
// their places from the lanes that hold it too (a ballot for every bit), so nothing depends on the order in which blocks or
// atomics run.  Up to 4 096 rows stay in the LDS of one block, for all digits.
//
// Bound by latency: a few dependent loads and barriers a launch.  50 000 rows of 89 entries: 3.1 us to count, 6.6 to place; 3 000 rows in
// one block 4.7.
#include "smx_groups.hpp"

namespace smx {

namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kMostDigits = 1024;
constexpr int kSmallRows = 4096;      // of one block

// A launch's share of the zeros, by its blocks behind the sort's; past the caches, which the sums' rows need (16 381 rows of 32 000 entries, 2 048 in
// bfloat16: the gradient takes 62 us, 69 by way of the caches).
struct Filling {
    char* at;
    long bytes;
    int blocks;      // of the sort
};
__device__ __forceinline__ bool fills(const Filling& f)
{
    if ((int)blockIdx.x < f.blocks) return false;
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    char* const end = f.at + f.bytes;
    char* const from = f.at - (reinterpret_cast<size_t>(f.at) & 15);      // (pieces of 16 bytes at multiples of 16)
    const long pieces = (end - from + 15) / 16, each = (long)blockDim.x * 8;
    for (long at = (blockIdx.x - f.blocks) * each + threadIdx.x; at < pieces; at += (gridDim.x - f.blocks) * each)
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            char* const to = from + (at + u * (int)blockDim.x) * 16;
            if (to >= f.at && to + 16 <= end) __builtin_nontemporal_store(u32x4{0, 0, 0, 0}, reinterpret_cast<u32x4*>(to));
            else
                for (char* p = to; p < to + 16; p += 2)
                    if (p >= f.at && p < end) *reinterpret_cast<short*>(p) = 0;
        }
    return true;
}

struct Pass {
    const int* index;      // the first pass: indices of the rows; or
    const int* keys;       // keys and rows as the pass before left them
    const int* rows_in;
    int *keys_out, *rows_out;      // keys_out may be null
    int* offsets;                  // of the only pass, or null
    int* count;                    // [block][digit]
    int groups, shift, bits, blocks, rows_per_block;
    long rows;
    Filling zeros;
};
__device__ __forceinline__ int key_at(const Pass& p, long i) { return p.index ? row_key(p.index[i], p.groups) : p.keys[i]; }

// lanes of the wavefront that are alive and have this lane's digit
__device__ __forceinline__ unsigned long same_digit(int digit, bool live, int bits)
{
    unsigned long same = __ballot(live);
    for (int b = 0; b < bits; ++b) {
        const unsigned long set = __ballot(digit >> b & 1);
        same &= digit >> b & 1 ? set : ~set;
    }
    return same;
}
// A row's place among those of its digit that the wavefront has met so far, from next[] (the wavefront's own; its LDS operations are
// done in order, and the fences keep the compiler to it).
__device__ __forceinline__ int take_place(int* next, int digit, bool live, int bits, int lane)
{
    const unsigned long same = same_digit(digit, live, bits);
    const int before = __popcll(same & ((1ul << lane) - 1));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int first = live ? next[digit] : 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (live && before == 0) next[digit] = first + __popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    return first + before;
}

__global__ __launch_bounds__(kThreads) void k_sort_count(const Pass p)
{
    __shared__ int hist[kMostDigits];
    if (fills(p.zeros)) return;
    const int digits = 1 << p.bits;
    for (int d = threadIdx.x; d < digits; d += kThreads) hist[d] = 0;
    __syncthreads();
    const long begin = (long)blockIdx.x * p.rows_per_block, end = min(begin + p.rows_per_block, p.rows);
#pragma unroll 4
    for (long i = begin + threadIdx.x; i < end; i += kThreads) atomicAdd(&hist[key_at(p, i) >> p.shift & (digits - 1)], 1);
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += kThreads) p.count[(long)blockIdx.x * digits + d] = hist[d];
}

// exclusive sums over the block's threads of one number each; part: a number a wavefront
__device__ __forceinline__ int block_exclusive(int x, int* part, int& total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int sum = x;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int y = __shfl_up(sum, d, 64);
        if (lane >= d) sum += y;
    }
    __syncthreads();
    if (lane == 63) part[wave] = sum;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int w = 0; w < (int)(blockDim.x >> 6); ++w) {
        const int y = part[w];
        before += w < wave ? y : 0;
        total += y;
    }
    return before + sum - x;
}

__global__ __launch_bounds__(kThreads) void k_sort_place(const Pass p)
{
    __shared__ int next[kWaves][kMostDigits];      // at first the counts of the wavefronts' rows
    __shared__ int all[kMostDigits], before[kMostDigits];
    __shared__ int part[kWaves];
    if (fills(p.zeros)) return;
    const int digits = 1 << p.bits, mask = digits - 1, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int d = threadIdx.x; d < digits; d += kThreads) {
        all[d] = before[d] = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) next[w][d] = 0;
    }
    __syncthreads();
    // rows of a wavefront: neighbours
    const long per_wave = p.rows_per_block / kWaves;
    const long begin = (long)blockIdx.x * p.rows_per_block + wave * per_wave, end = min(begin + per_wave, p.rows);
#pragma unroll 4
    for (long i = begin + lane; i < end; i += 64) atomicAdd(&next[wave][key_at(p, i) >> p.shift & mask], 1);
    // counts of all blocks, and of those before this one: a digit's by several threads where there are more threads than digits
    const int at_once = min(digits, kThreads), parts = kThreads / at_once, mine = threadIdx.x / at_once;
    for (int d = threadIdx.x % at_once; d < digits; d += at_once) {
        int a = 0, b = 0;
#pragma unroll 8
        for (int k = mine; k < p.blocks; k += parts) {
            const int x = p.count[(long)k * digits + d];
            a += x;
            b += k < (int)blockIdx.x ? x : 0;
        }
        atomicAdd(&all[d], a);
        atomicAdd(&before[d], b);
    }
    __syncthreads();
    int base = 0;
    for (int d0 = 0; d0 < digits; d0 += kThreads) {
        const int d = d0 + threadIdx.x;
        int total;
        const int start = base + block_exclusive(d < digits ? all[d] : 0, part, total);
        if (d < digits) {
            if (p.offsets && blockIdx.x == 0 && d < p.groups + 2) p.offsets[d] = start;
            int at = start + before[d];
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const int c = next[w][d];
                next[w][d] = at;
                at += c;
            }
        }
        base += total;
    }
    __syncthreads();
    for (long i = begin; i < end; i += 64) {
        const bool live = i + lane < end;
        const int key = live ? key_at(p, i + lane) : 0;
        const int at = take_place(next[wave], key >> p.shift & mask, live, p.bits, lane);
        if (live) {
            p.rows_out[at] = p.index ? (int)(i + lane) : p.rows_in[i + lane];
            if (p.keys_out) p.keys_out[at] = key;
        }
    }
}

__global__ __launch_bounds__(256) void k_sort_offsets(const int* keys, int rows, int groups, int* offsets)
{
    const int g = blockIdx.x * 256 + threadIdx.x;
    if (g < groups + 2) offsets[g] = first_place(keys, rows, g);
}

__global__ __launch_bounds__(256) void k_no_rows(int* offsets, int n)
{
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < n) offsets[i] = 0;
}

// (offsets of more groups by one block would take longer than the sort)
constexpr int kMostInside = 4096;

// All digits in one block: a wavefront has neighbouring rows, 64 at a time, at first and after every digit.
struct SmallSort {
    const int* index;
    int rows, groups, key_bits, bits;
    int *order, *offsets, *keys;
    Filling zeros;
};
constexpr int kSmallWaves = 16, kSmallDigits = 512;
constexpr int small_lds(int rows) { return rows * 6 + kSmallWaves * kSmallDigits * 4; }
template <int PER>
__global__ __launch_bounds__(1024) void k_sort_small(const SmallSort p)
{
    extern __shared__ int small[];
    __shared__ int part[kSmallWaves];
    if (fills(p.zeros)) return;
    int(*next)[kSmallDigits] = reinterpret_cast<int(*)[kSmallDigits]>(small);
    int* key_of = small + kSmallWaves * kSmallDigits;
    unsigned short* row_of = reinterpret_cast<unsigned short*>(key_of + 1024 * PER);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, digits = 1 << p.bits;
    const int per_wave = ((p.rows + 1023) / 1024) * 64, begin = wave * per_wave, end = min(begin + per_wave, p.rows);
    int key[PER], row[PER], at[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        row[u] = min(begin + 64 * u + lane, p.rows - 1);
        key[u] = p.index[row[u]];
    }
#pragma unroll
    for (int u = 0; u < PER; ++u) key[u] = row_key(key[u], p.groups);
    for (int shift = 0; shift < p.key_bits; shift += p.bits) {
        const bool first = shift == 0, last = shift + p.bits >= p.key_bits;
        for (int d = threadIdx.x; d < kSmallWaves * digits; d += 1024) next[d >> p.bits][d & (digits - 1)] = 0;
        __syncthreads();
        if (!first)
#pragma unroll
            for (int u = 0; u < PER; ++u)
                if (begin + 64 * u + lane < end) {
                    key[u] = key_of[begin + 64 * u + lane];
                    row[u] = row_of[begin + 64 * u + lane];
                }
#pragma unroll
        for (int u = 0; u < PER; ++u)      // places inside the wavefront first
            if (begin + 64 * u < end) at[u] = take_place(next[wave], key[u] >> shift & (digits - 1), begin + 64 * u + lane < end, p.bits, lane);
        __syncthreads();
        int sum = 0, total;
        if ((int)threadIdx.x < digits)
#pragma unroll
            for (int w = 0; w < kSmallWaves; ++w) sum += next[w][threadIdx.x];
        int start = block_exclusive(sum, part, total);
        if ((int)threadIdx.x < digits) {
            if (p.offsets && first && last && (int)threadIdx.x < p.groups + 2) p.offsets[threadIdx.x] = start;
#pragma unroll
            for (int w = 0; w < kSmallWaves; ++w) {
                const int c = next[w][threadIdx.x];
                next[w][threadIdx.x] = start;
                start += c;
            }
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < PER; ++u)
            if (begin + 64 * u + lane < end) {
                const int to = next[wave][key[u] >> shift & (digits - 1)] + at[u];
                key_of[to] = key[u];
                row_of[to] = (unsigned short)row[u];
            }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < p.rows; i += 1024) {
        p.order[i] = row_of[i];
        if (p.keys) p.keys[i] = key_of[i];
    }
    if (p.offsets && p.key_bits > p.bits)
        for (int g = threadIdx.x; g < p.groups + 2; g += 1024) p.offsets[g] = first_place(key_of, p.rows, g);
}

}  // namespace

bool sort_has_offsets(long rows, int groups)
{
    return rows <= kSmallRows ? groups <= kMostInside : groups + 2L <= kMostDigits;
}

void sort_rows(Launches& launches, Arena& arena, const int* index, long rows, int groups, const RowOrder& to, const Zeros& zeros)
{
    // Zeros are shared by the launches of a sort, equally: of two passes they take 3.2, 6.4, 2.7 and 6.8 us without.
    auto share = [&](int which, int of, long blocks) {
        const long begin = zeros.bytes / 2 * which / of * 2, end = zeros.bytes / 2 * (which + 1) / of * 2;
        return Filling{zeros.at + begin, end - begin, (int)blocks};
    };
    auto filling_blocks = [](const Filling& f) { return std::min((f.bytes + (64 << 10) - 1) / (64 << 10), 2048L); };
    if (rows == 0) {
        if (to.offsets) launches.start(k_no_rows, ((long)groups + 2 + 255) / 256, 1, 1, 256, 0, to.offsets, groups + 2);
        return;
    }
    int key_bits = 1;
    while ((1L << key_bits) < (long)groups + 2) ++key_bits;
    int* keys = to.keys;
    auto offsets = [&] { launches.start(k_sort_offsets, ((long)groups + 2 + 255) / 256, 1, 1, 256, 0, (const int*)keys, (int)rows, groups, to.offsets); };
    if (rows <= kSmallRows) {
        const bool later = to.offsets && groups > kMostInside;
        if (later && !keys) keys = arena.take<int>(rows);
        const int passes = (key_bits + 8) / 9;
        const SmallSort p{index, (int)rows, groups, key_bits, (key_bits + passes - 1) / passes, to.order, later ? nullptr : to.offsets, keys, share(0, 1, 1)};
        auto go = [&](auto per) {
            constexpr int PER = decltype(per)::value, bytes = small_lds(1024 * PER);
            if (bytes > 48 * 1024 && !launches.dry)
                hip_ok(hipFuncSetAttribute(reinterpret_cast<const void*>(k_sort_small<PER>), hipFuncAttributeMaxDynamicSharedMemorySize, bytes), "LDS");
            launches.start(k_sort_small<PER>, 1 + filling_blocks(p.zeros), 1, 1, 1024, bytes, p);
        };
        if (rows <= 1024) go(Int<1>{});
        else go(Int<4>{});
        if (later) offsets();
        return;
    }
    const int passes = (key_bits + 9) / 10;
    Pass p{};
    p.groups = groups;
    p.rows = rows;
    // (every block reads the counts of all)
    p.rows_per_block = (int)std::max(1024L, up((rows + 255) / 256, kThreads));
    p.blocks = (int)((rows + p.rows_per_block - 1) / p.rows_per_block);
    p.count = arena.take<int>((long)p.blocks << ((key_bits + passes - 1) / passes));
    if (passes > 1 && !keys) keys = arena.take<int>(rows);
    int* other_keys[2] = {passes > 1 ? arena.take<int>(rows) : nullptr, nullptr};
    int* other_rows[2] = {passes > 1 ? arena.take<int>(rows) : nullptr, nullptr};
    if (passes > 2) other_keys[1] = arena.take<int>(rows), other_rows[1] = arena.take<int>(rows);
    for (int pass = 0, shift = 0; pass < passes; ++pass) {
        const bool last = pass == passes - 1;
        p.bits = (key_bits - shift + passes - pass - 1) / (passes - pass);
        p.shift = shift;
        p.index = pass == 0 ? index : nullptr;
        p.keys = pass == 0 ? nullptr : other_keys[(pass - 1) % 2];
        p.rows_in = pass == 0 ? nullptr : other_rows[(pass - 1) % 2];
        p.keys_out = last ? keys : other_keys[pass % 2];
        p.rows_out = last ? to.order : other_rows[pass % 2];
        p.offsets = passes == 1 ? to.offsets : nullptr;
        p.zeros = share(2 * pass, 2 * passes, p.blocks);
        launches.start(k_sort_count, p.blocks + filling_blocks(p.zeros), 1, 1, kThreads, 0, p);
        p.zeros = share(2 * pass + 1, 2 * passes, p.blocks);
        launches.start(k_sort_place, p.blocks + filling_blocks(p.zeros), 1, 1, kThreads, 0, p);
        shift += p.bits;
    }
    if (to.offsets && passes > 1) offsets();
}

namespace {

void check(long rows, int groups)
{
    refuse_unless(rows >= 0 && rows <= 1L << 28, "rows: 0 to 2^28");
    refuse_unless(groups >= 0 && groups <= SMX_MOST_ENTRIES, "num_groups: 0 to 2^24");
}

}  // namespace

}  // namespace smx

using namespace smx;

extern "C" int smx_group_rows_workspace(long rows, int num_groups, long* bytes)
{
    return finetune_entry("smx_group_rows_workspace", [&] {
        check(rows, num_groups);
        refuse_unless(bytes, "bytes must not be null");
        Launches dry{nullptr, true};
        Arena arena{reinterpret_cast<char*>(256)};
        sort_rows(dry, arena, nullptr, rows, num_groups, RowOrder{nullptr, reinterpret_cast<int*>(4), nullptr});
        *bytes = arena.used;
    });
}

extern "C" int smx_group_rows(long rows, int num_groups, const int* d_index, int* d_order, int* d_offsets, void* d_workspace, long workspace_bytes, void* stream)
{
    return finetune_entry("smx_group_rows", [&] {
        check(rows, num_groups);
        refuse_unless(d_offsets && (rows == 0 || (d_index && d_order)), "index, order and offsets must not be null");
        long need = 0;
        if (smx_group_rows_workspace(rows, num_groups, &need) != SMX_OK) throw Refusal(SMX_EINVAL, "sizes");
        check_workspace(d_workspace, workspace_bytes, need, "smx_group_rows_workspace");
        require_gfx950();
        Launches launches{static_cast<hipStream_t>(stream), false};
        Arena arena{static_cast<char*>(d_workspace)};
        sort_rows(launches, arena, d_index, rows, num_groups, RowOrder{d_order, d_offsets, nullptr});
        hip_ok(hipGetLastError(), "launch");
    });
}
