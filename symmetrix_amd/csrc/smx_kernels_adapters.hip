// A shared projection with a low-rank adapter per row beside it, and its gradient.
//
//   y = W x + B_a h,  h = c_a A_a x
//   g = c_a B_a^T dy:   dx = W^T dy + A_a^T g,   dA_a = sum over the adapter's rows of g x^T,   dB_a = sum of dy h^T
//
// Forward: h of all rows (k_down), then one product that adds the adapters' part to its sums before they are rounded and stored
// (k_product16, k_product32 with k_add_mixed; long sums of few tiles in parts, k_join_splits; few rows: k_down_few, k_product_few).
// Gradient: h and g, the product with W^T, and for dA and dB the rows sorted by adapter (counted in k_prepare, placed beside k_down), sums
// over pieces of an adapter's rows (k_outer), and the sums of those (k_join).  k_prepare also lays out the operands that the products
// cannot take as they are: W^T, rows that are not aligned, single precision in its parts.
//
// What bounds it: 16-bit products of many rows the matrix instructions (8 179 rows, 4 096 x 4 096 in bfloat16: 250 us a call, 1.10
// PFLOP/s, of which k_down 27), few rows the bytes of W (16 rows of the same: 8.4 us for the product's 34 MB, 4.0 TB/s), single precision the six bf16 products a product is made of (50 000 rows, 256 -> 512: 111 us, 119 TFLOP/s).
//
// Rows are taken as they come in the first two: sixteen of them share a matrix instruction, and every adapter that occurs among them is
// gone through, its result kept by its own rows alone (a choice, not a product with zero: infinities and NaN of an adapter stay with
// its rows).
#include "smx_finetune.hpp"

#include <algorithm>
#include <limits>

namespace smx {

namespace {

typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
// sixteen terms of a sum in single precision: a lane holds four neighbouring ones
__device__ __forceinline__ f32x4 mma(f32x4 a, f32x4 b, f32x4 c)
{
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
}
// what a lane holds of an operand: 16 bytes
template <typename T>
struct Operand {
    typedef T type __attribute__((ext_vector_type(kRun<T>)));
};
template <typename T>
__device__ __forceinline__ typename Operand<T>::type load_operand(const T* p, long left)
{
    constexpr int V = kRun<T>;
    if (left >= V) return *reinterpret_cast<const typename Run<T, V>::loose*>(p);
    typename Operand<T>::type x;
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = j < left ? p[j] : (T)0.0f;
    return x;
}

// 16 rows of 64 bytes, 16 bytes a lane: from lane 4 n + g, where neighbouring lanes have asked for neighbouring bytes of row n, to lane
// 16 g + n, which has them in an operand.  (Asked for in the order of an operand, with every lane in another row than its neighbours, a
// load takes about 100 cycles instead of 16, caches or not.)
template <typename V>
__device__ __forceinline__ V to_operand(const V& x, int lane)
{
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    const int from = (4 * (lane & 15) + (lane >> 4)) * 4;
    const i32x4 u = __builtin_bit_cast(i32x4, x);
    i32x4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __builtin_amdgcn_ds_bpermute(from, u[j]);
    return __builtin_bit_cast(V, v);
}

// and back: what lane 16 g + n has of row n goes to lane 4 n + g
template <typename V>
__device__ __forceinline__ V from_operand(const V& x, int lane)
{
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    const int from = (16 * (lane & 3) + (lane >> 2)) * 4;
    const i32x4 u = __builtin_bit_cast(i32x4, x);
    i32x4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __builtin_amdgcn_ds_bpermute(from, u[j]);
    return __builtin_bit_cast(V, v);
}

__device__ __forceinline__ bool has_adapter(int a, int n) { return a >= 0 && a < n; }
__device__ __forceinline__ bool is_bad(int a, int n) { return a < -1 || a >= n; }

constexpr int kPiece = 32;           // terms of a sum that a step of a product takes
// Rows of the kernels for few rows (64 rows, 4 096 x 4 096 in bfloat16: 20 us, and 38 with the others).
constexpr int kMostFew = 64;

// ---- operands laid out anew: rows of a multiple of 32 numbers, zeros behind the last; single precision for products in three bf16 parts

constexpr float kSplitScale = 16777216.0f;      // 2^24: the parts of every number down to the smallest are normal numbers
template <int N>
__device__ __forceinline__ void split(const float (&x)[N], bf16 (&part)[3][N])
{
#pragma unroll
    for (int j = 0; j < N; j += 2) {
        f32x2 rest = {x[j], x[j + 1]};
#pragma unroll
        for (int s = 0; s < 3; ++s) {
            const bf16x2 h = __builtin_convertvector(rest, bf16x2);
            part[s][j] = h[0]; part[s][j + 1] = h[1];
            if (s < 2) rest -= __builtin_convertvector(h, f32x2);
        }
    }
}

struct Layout {
    const void* src;
    long src_each, src_row, src_k;      // strides of a matrix, a row and a number
    void* dst;
    long dst_each;                      // stride of a matrix
    int rows, k, k_padded, matrices;
    bool parts;    // single precision in three bf16 parts, in the order of k_product32
    int live;      // rows that there are; zeros behind them
};
// First part of number k of a row, in [128 rows][32 numbers][part][row][32]: what a block takes at a step lies as it goes into LDS, the
// four pieces of a row in an order that depends on the row, for the banks.
constexpr int kPartRows = 128;
__device__ __forceinline__ long split_place(int row, int k, int k_padded)
{
    const int r = row % kPartRows, piece = (k % kPiece / 8) ^ (r >> 1 & 3);
    return ((long)(row / kPartRows) * (k_padded / kPiece) + k / kPiece) * 3 * kPartRows * kPiece + r * kPiece + piece * 8 + k % 8;
}
inline __host__ __device__ long layout_blocks(const Layout& p) { return (long)((p.k_padded + 63) / 64) * ((p.rows + 63) / 64) * p.matrices; }
// a block takes 64 rows and 64 numbers of them
template <typename T>
__device__ __forceinline__ void lay_out(const Layout& p, long block, T (*tile)[65])
{
    const int across = (p.k_padded + 63) / 64, down = (p.rows + 63) / 64;
    const int k0 = (int)(block % across) * 64, row0 = (int)(block / across % down) * 64, matrix = (int)(block / across / down);
    const T* src = static_cast<const T*>(p.src) + matrix * p.src_each;
    T x[16];
    // (neighbouring threads where neighbouring numbers are)
    if (p.src_k == 1) {
        const int k = threadIdx.x & 63;
#pragma unroll
        for (int u = 0; u < 16; ++u) {
            const int r = (threadIdx.x >> 6) + 4 * u;
            x[u] = row0 + r < p.live && k0 + k < p.k ? src[(row0 + r) * p.src_row + k0 + k] : (T)0.0f;
        }
#pragma unroll
        for (int u = 0; u < 16; ++u) tile[(threadIdx.x >> 6) + 4 * u][k] = x[u];
    } else {
        const int r = threadIdx.x & 63;
#pragma unroll
        for (int u = 0; u < 16; ++u) {
            const int k = (threadIdx.x >> 6) + 4 * u;
            x[u] = row0 + r < p.live && k0 + k < p.k ? src[(row0 + r) * p.src_row + (k0 + k) * p.src_k] : (T)0.0f;
        }
#pragma unroll
        for (int u = 0; u < 16; ++u) tile[r][(threadIdx.x >> 6) + 4 * u] = x[u];
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        const int r = (threadIdx.x >> 5) + 8 * u, k = (threadIdx.x & 31) * 2;
        if (row0 + r >= p.rows || k0 + k >= p.k_padded) continue;
        if (std::is_same_v<T, float> && p.parts) {
            const float v[2] = {(float)tile[r][k] * kSplitScale, (float)tile[r][k + 1] * kSplitScale};
            bf16 part[3][2];
            split(v, part);
            bf16* to = static_cast<bf16*>(p.dst) + split_place(row0 + r, k0 + k, p.k_padded);
#pragma unroll
            for (int q = 0; q < 3; ++q) *reinterpret_cast<bf16x2*>(to + q * kPartRows * kPiece) = bf16x2{part[q][0], part[q][1]};
        } else {
            typedef T pair __attribute__((ext_vector_type(2)));
            *reinterpret_cast<pair*>(static_cast<T*>(p.dst) + matrix * p.dst_each + (long)(row0 + r) * p.k_padded + k0 + k) = pair{tile[r][k], tile[r][k + 1]};
        }
    }
}

// ---- rows sorted by adapter, in their order: places [start[a], start[a + 1]) of perm hold adapter a's; rows with no adapter, and with an
// index out of range, come last.  Pieces of at most `piece` rows of one adapter: [first[a], first[a + 1]).

struct Groups {
    const int* index;
    int adapters, blocks, rows_per_block, piece;
    long rows;
    int* count;              // [block][key]: rows of a block
    int *start, *first;      // [adapters + 1]
    int* perm;
};
__device__ __forceinline__ int key_of(int a, int n) { return has_adapter(a, n) ? a : (a == -1 ? n : n + 1); }
constexpr int kMostKeys = SMX_ADAPTER_MAX_COUNT + 2;

__device__ __forceinline__ void count_rows(const Groups& p, int block, int* hist)
{
    const int keys = p.adapters + 2;
    for (int k = threadIdx.x; k < keys; k += 256) hist[k] = 0;
    __syncthreads();
    const long begin = (long)block * p.rows_per_block, end = min(begin + p.rows_per_block, p.rows);
    for (long i = begin + threadIdx.x; i < end; i += 256) atomicAdd(&hist[key_of(p.index[i], p.adapters)], 1);
    __syncthreads();
    for (int k = threadIdx.x; k < keys; k += 256) p.count[(long)block * keys + k] = hist[k];
}
__device__ __forceinline__ int wave_exclusive(int x, int lane, int& total)
{
    int sum = x;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int y = __shfl_up(sum, d, 64);
        if (lane >= d) sum += y;
    }
    total = __shfl(sum, 63, 64);
    return sum - x;
}
// One wavefront places the rows of a block.
__device__ __forceinline__ void place_rows(const Groups& p, int block, int lane, int* base)
{
    const int keys = p.adapters + 2;
    int rows = 0, pieces = 0;
    for (int k0 = 0; k0 < keys; k0 += 64) {
        const int k = min(k0 + lane, keys - 1);
        int all = 0, before = 0;
#pragma unroll 8
        for (int b = 0; b < p.blocks; ++b) {
            const int x = p.count[(long)b * keys + k];
            all += x;
            before += b < block ? x : 0;
        }
        if (k0 + lane >= keys) all = 0;
        int row_total, piece_total;
        const int row_before = rows + wave_exclusive(all, lane, row_total);
        const int piece_before = pieces + wave_exclusive(k0 + lane < p.adapters ? (all + p.piece - 1) / p.piece : 0, lane, piece_total);
        if (k0 + lane < keys) base[k0 + lane] = row_before + before;
        if (block == 0 && k0 + lane <= p.adapters) {
            p.start[k0 + lane] = row_before;
            p.first[k0 + lane] = piece_before;
        }
        rows += row_total;
        pieces += piece_total;
    }
    const long begin = (long)block * p.rows_per_block, end = min(begin + p.rows_per_block, p.rows);
    for (long i = begin; i < end; i += 64) {
        const bool live = i + lane < end;
        const int key = live ? key_of(p.index[i + lane], p.adapters) : keys;
        unsigned long same = __ballot(live);
        for (int bit = 0; (1 << bit) <= keys; ++bit) {
            const unsigned long set = __ballot(key >> bit & 1);
            same &= key >> bit & 1 ? set : ~set;
        }
        const int before = __popcll(same & ((1ul << lane) - 1));
        // (the wavefront's own LDS operations, which are done in order; the fences keep the compiler to it)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const int at = live ? base[key] + before : 0;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (live) {
            p.perm[at] = (int)(i + lane);
            if (before == 0) base[key] = at + __popcll(same);
        }
    }
}

// What the other kernels need beforehand: two layouts, and the rows of every adapter counted.
struct Prepare {
    Layout layout[2];
    long blocks[2];
    Groups groups;
    long first;      // which of all blocks the launch's first one is
};
template <typename T>
__global__ __launch_bounds__(256) void k_prepare(const Prepare p)
{
    __shared__ union {
        T tile[64][65];
        int hist[kMostKeys];
    } lds;
    long block = p.first + blockIdx.x;
    if (block < p.blocks[0]) {
        lay_out<T>(p.layout[0], block, lds.tile);
        return;
    }
    block -= p.blocks[0];
    if (block < p.blocks[1]) {
        lay_out<T>(p.layout[1], block, lds.tile);
        return;
    }
    count_rows(p.groups, (int)(block - p.blocks[1]), lds.hist);
}

// ---- h[row][r] = c_a sum over k of in[row][k] F_a(r, k); zero for r from the rank on and for rows without an adapter

struct Down {
    const void* in;
    long in_stride;
    const void* F;
    long f_each, f_row;      // strides of an adapter and of an r
    const float* scale;
    const int* index;
    int adapters, rank, padded, k;      // padded: of h's rows, a multiple of 16
    long rows;
    float* h;
};
// one or two of them, and beside them the rows placed by adapter
struct Downs {
    Down down[2];
    int blocks[2];
    Groups groups;
    int first;      // as in Prepare
};

// A block takes 16 MT rows; its wavefronts have 128 bytes of a row by turns, and their sums are added in order.  The next 128 bytes are under
// way during the sums of these.  Bound by the latency of loads, with few wavefronts on a CU: 67 MB of rows in 27 us (8 179 rows of 4 096
// numbers in bfloat16, 24 adapters of rank 32), 51 MB in 13 (50 000 rows of 256 in single precision, 4.0 TB/s).
template <typename T, int RT, int MT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_down(const Downs both)
{
    constexpr int V = kRun<T>, UNIT = 8 * V;
    typedef typename Operand<T>::type frag;
    __shared__ union {
        f32x4 part[WAVES][MT * RT][64];
        int base[kMostKeys];
    } lds;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    int block = both.first + blockIdx.x;
    if (block >= both.blocks[0] + both.blocks[1]) {
        if (wave == 0) place_rows(both.groups, block - both.blocks[0] - both.blocks[1], lane, lds.base);
        return;
    }
    const bool second = block >= both.blocks[0];
    if (second) block -= both.blocks[0];
    const Down& p = both.down[second];
    // the blocks of a die (every eighth) take neighbouring rows, whose factors its L2 holds: rows of one adapter mostly are neighbours
    block = block % 8 * (both.blocks[second] / 8) + block / 8;
    if ((long)block * 16 * MT >= p.rows) return;
    long row[MT];
    int a[MT];
    bool good[MT];
    unsigned left[MT];
    const T* in[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const long at = ((long)block * MT + i) * 16 + n;
        row[i] = min(at, p.rows - 1);
        a[i] = p.index[row[i]];
        good[i] = at < p.rows && has_adapter(a[i], p.adapters);
        left[i] = (unsigned)__ballot(good[i]) & 0xffffu;
        in[i] = static_cast<const T*>(p.in) + min(((long)block * MT + i) * 16 + lane / 4, p.rows - 1) * p.in_stride + (lane & 3) * V;
        if (at < p.rows && !good[i] && wave == 0)
#pragma unroll
            for (int q = 0; q < RT; ++q)
                if (16 * q < p.padded) *reinterpret_cast<f32x4*>(p.h + row[i] * p.padded + 16 * q + 4 * g) = f32x4{0, 0, 0, 0};
    }
    // the sums of rows with up to ADAPTERS adapters in one sweep over their numbers
    auto sweep = [&](auto adapters, const int (&cur)[2]) {
        constexpr int ADAPTERS = decltype(adapters)::value;
        f32x4 acc[ADAPTERS][MT][RT];
        const T* F[ADAPTERS][RT];
#pragma unroll
        for (int c = 0; c < ADAPTERS; ++c) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int q = 0; q < RT; ++q) acc[c][i][q] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int q = 0; q < RT; ++q) F[c][q] = static_cast<const T*>(p.F) + cur[c] * p.f_each + (long)min(16 * q + lane / 4, p.rank - 1) * p.f_row + (lane & 3) * V;
        }
        const int full = p.k / UNIT;
        struct Unit {
            frag x[MT][2], f[ADAPTERS][RT][2];
        };
        auto fetch = [&](int u, Unit& v) {
            const long k = (long)min(u, full - 1) * UNIT;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
#pragma unroll
                for (int i = 0; i < MT; ++i) v.x[i][half] = *reinterpret_cast<const typename Run<T, V>::loose*>(in[i] + k + half * (UNIT / 2));
#pragma unroll
                for (int c = 0; c < ADAPTERS; ++c)
#pragma unroll
                    for (int q = 0; q < RT; ++q) v.f[c][q][half] = *reinterpret_cast<const typename Run<T, V>::loose*>(F[c][q] + k + half * (UNIT / 2));
            }
            asm volatile("" ::: "memory");      // (asked for here, not where they are used)
        };
        auto sums = [&](const Unit& v) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                frag x[MT];
#pragma unroll
                for (int i = 0; i < MT; ++i) x[i] = to_operand(v.x[i][half], lane);
#pragma unroll
                for (int c = 0; c < ADAPTERS; ++c)
#pragma unroll
                    for (int q = 0; q < RT; ++q) {
                        const frag f = to_operand(v.f[c][q][half], lane);
#pragma unroll
                        for (int i = 0; i < MT; ++i) acc[c][i][q] = mma(f, x[i], acc[c][i][q]);
                    }
            }
        };
        int u = wave;
        if (u < full) {
            Unit even, odd;
            fetch(u, even);
#pragma unroll 1
            for (;;) {
                fetch(u + WAVES, odd);
                sums(even);
                if ((u += WAVES) >= full) break;
                fetch(u + WAVES, even);
                sums(odd);
                if ((u += WAVES) >= full) break;
            }
        }
        if (u == full && p.k % UNIT) {      // (the end of the rows, for one wavefront)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int k = full * UNIT + half * (UNIT / 2), rest = p.k - k - (lane & 3) * V;
                frag x[MT];
#pragma unroll
                for (int i = 0; i < MT; ++i) x[i] = to_operand(load_operand(in[i] + k, rest), lane);
#pragma unroll
                for (int c = 0; c < ADAPTERS; ++c)
#pragma unroll
                    for (int q = 0; q < RT; ++q) {
                        const frag f = to_operand(load_operand(F[c][q] + k, rest), lane);
#pragma unroll
                        for (int i = 0; i < MT; ++i) acc[c][i][q] = mma(f, x[i], acc[c][i][q]);
                    }
            }
        }
#pragma unroll
        for (int c = 0; c < ADAPTERS; ++c) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int q = 0; q < RT; ++q) lds.part[wave][i * RT + q][lane] = acc[c][i][q];
            __syncthreads();
            const float scale = p.scale ? p.scale[cur[c]] : 1.0f;
#pragma unroll
            for (int at = 0; at < MT * RT; ++at) {
                if (at % WAVES != wave) continue;
                const int i = at / RT, q = at % RT;
                f32x4 sum = lds.part[0][at][lane];
#pragma unroll
                for (int w = 1; w < WAVES; ++w) sum += lds.part[w][at][lane];
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[j] = 16 * q + 4 * g + j < p.rank ? sum[j] * scale : 0.0f;
                if (good[i] && a[i] == cur[c] && 16 * q < p.padded) *reinterpret_cast<f32x4*>(p.h + row[i] * p.padded + 16 * q + 4 * g) = sum;
            }
            __syncthreads();
        }
    };
    auto next = [&] {
        int cur = -1;
#pragma unroll
        for (int i = 0; i < MT; ++i)
            if (cur < 0 && left[i]) cur = __builtin_amdgcn_readlane(a[i], __builtin_ctz(left[i]));
#pragma unroll
        for (int i = 0; i < MT; ++i) left[i] &= ~(unsigned)__ballot(good[i] && a[i] == cur);
        return cur;
    };
    // (two at a time: the blocks in which one adapter's rows end and another's begin would be the last ones otherwise)
    for (int cur[2] = {next(), 0}; cur[0] >= 0; cur[0] = next()) {
        cur[1] = next();
        if (cur[1] >= 0) sweep(std::integral_constant<int, 2>{}, cur);
        else sweep(std::integral_constant<int, 1>{}, cur);
    }
}

// Few rows: a wavefront per number of h.  (16 rows of 4 096 numbers: 3.6 us, a chain of a load, a sum and a store.)
template <typename T>
__global__ __launch_bounds__(256) void k_down_few(const Down p)
{
    constexpr int V = kRun<T>;
    const long row = blockIdx.x;
    const int lane = threadIdx.x & 63, r = blockIdx.y * 4 + (threadIdx.x >> 6), a = p.index[row];
    float sum = 0.0f;
    if (has_adapter(a, p.adapters) && r < p.rank) {
        const T* in = static_cast<const T*>(p.in) + row * p.in_stride + lane * V;
        const T* F = static_cast<const T*>(p.F) + a * p.f_each + (long)r * p.f_row + lane * V;
        const int full = p.k / (64 * V) * (64 * V);
#pragma unroll 4
        for (int k = 0; k < full; k += 64 * V) {
            const typename Operand<T>::type x = *reinterpret_cast<const typename Run<T, V>::loose*>(in + k), f = *reinterpret_cast<const typename Run<T, V>::loose*>(F + k);
#pragma unroll
            for (int j = 0; j < V; ++j) sum = fmaf((float)x[j], (float)f[j], sum);
        }
        if (full < p.k) {
            float x[V], f[V];
            load_run<V>(in + full, p.k - full - lane * V, x);
            load_run<V>(F + full, p.k - full - lane * V, f);
#pragma unroll
            for (int j = 0; j < V; ++j) sum = fmaf(x[j], f[j], sum);
        }
        sum = group_sum<64>(sum) * (p.scale ? p.scale[a] : 1.0f);
    }
    if (lane == 0 && r < p.padded) p.h[row * p.padded + r] = sum;
}

// ---- out[row][col] = sum over k of in[row][k] W(col, k) + sum over r of h[row][r] F_a(col, r); NaN where the index is out of range

struct Product {
    const void* in;
    long in_stride;
    const void* W;               // laid out: rows (columns of the result) w_stride apart, of a multiple of 32 numbers; or three bf16 parts
    long w_stride;
    const void* W0;              // as the caller has it
    long w0_col, w0_k;
    const void* F;
    long f_each, f_col, f_r;
    bool f_runs;
    const float* h;
    const int* index;
    int adapters, rank, padded, k, k_padded, cols;
    long rows;
    void* out;
    long out_stride;
    int row_tiles, col_tiles;
    int splits, split_steps;      // of the sum over k: parts, and steps of each; from two parts on sums go to partial[split][row][col]
    float* partial;
};

// Block -> tile: the blocks of a die (every eighth) take neighbouring tiles, four row tiles high, so that they share rows in its L2.
__device__ __forceinline__ bool tile_of(const Product& p, int& rt, int& ct)
{
    const int tiles = p.row_tiles * p.col_tiles, per = (tiles + 7) / 8, at = blockIdx.x % 8 * per + blockIdx.x / 8;
    if (at >= tiles || (int)blockIdx.x / 8 >= per) return false;
    const int band = at / (4 * p.col_tiles), high = min(4, p.row_tiles - 4 * band), in_band = at - band * 4 * p.col_tiles;
    rt = band * 4 + in_band % high;
    ct = in_band / high;
    return true;
}

// Lane (n, g) holds of tile (i, t) row i * 16 + n and four columns: in single precision 16 t + 4 g + 0..3; in 16 bits 8 g + 4 (t % 2) + 0..3 of
// the 32 columns of two tiles, so that a lane has eight neighbours of them to store.
template <typename T>
__device__ __forceinline__ int column_of(int t, int m) { return std::is_same_v<T, float> ? 16 * t + m : 32 * (t >> 1) + 8 * (m >> 2) + 4 * (t & 1) + (m & 3); }

// The product of a factor's columns and rows of h, 32 r at a time, for 16-bit types: on the bf16 instructions, h in two
// bf16 parts (what is left out is below 2^-16 of a product; the result is rounded to 2^-9 or 2^-11), and numbers of float16 in two, which
// hold them exactly.
template <typename T>
struct AdapterProduct {
    static constexpr int CHUNK = 32, F_PARTS = std::is_same_v<T, f16> ? 2 : 1;
    struct Factor {
        bf16x8 part[F_PARTS];
    };
    // Whether an infinity or NaN, or what rounds to one, was among a lane's numbers.
    struct Odd {
        float none = 0.0f;      // NaN then,
        unsigned bits = 0;      // or the sign's place of a half set
        __device__ __forceinline__ bool any() const { return __any(none != none || bits & 0x80008000u); }
    };
    __device__ static __forceinline__ void parts_of(const float (&x)[8], bf16x8 (&part)[2], float& none)
    {
        constexpr float most = std::numeric_limits<float>::max();
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const f32x2 v = {x[j], x[j + 1]};
            const bf16x2 h = __builtin_convertvector(v, bf16x2);
            f32x2 rest = v - __builtin_convertvector(h, f32x2);
            none = fmaf(rest[0], 0.0f, none);
            none = fmaf(rest[1], 0.0f, none);
            if (!(fabsf(rest[0]) <= most)) rest[0] = 0.0f;      // (infinities are their first part)
            if (!(fabsf(rest[1]) <= most)) rest[1] = 0.0f;
            const bf16x2 l = __builtin_convertvector(rest, bf16x2);
            part[0][j] = h[0]; part[0][j + 1] = h[1];
            part[1][j] = l[0]; part[1][j + 1] = l[1];
        }
    }
    // F(col, r) = base[col * f_col + r * f_r] for the columns of a tile, r = r0 + 8 g + 0..7; eight numbers at a time where they are side by side
    // and the rank is a multiple of eight.  (No branch depends on the lane, here and below: what is behind the rank is read from its end and
    // put to zero.)
    __device__ static __forceinline__ Factor factor(const Product& p, const T* base, int col0, int t, int r0, int lane, Odd& odd)
    {
        typename Operand<T>::type v;
        if (p.f_runs) {
            const int r = r0 + 8 * (lane & 3);
            v = *reinterpret_cast<const typename Run<T, 8>::loose*>(base + min(col0 + column_of<T>(t, lane >> 2), p.cols - 1) * p.f_col + min(r, p.rank - 8));
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = r < p.rank ? v[j] : (T)0.0f;
            v = to_operand(v, lane);
        } else {
            const int r = r0 + 8 * (lane >> 4);
            const T* from = base + min(col0 + column_of<T>(t, lane & 15), p.cols - 1) * p.f_col;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const T x = from[min(r + j, p.rank - 1) * p.f_r];
                v[j] = r + j < p.rank ? x : (T)0.0f;
            }
        }
        // (an exponent of ones carries into the sign's place)
        typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
        const u32x4 u = (__builtin_bit_cast(u32x4, v) & 0x7fff7fffu) + (std::is_same_v<T, f16> ? 0x04000400u : 0x00800080u);
        odd.bits |= u[0] | u[1] | u[2] | u[3];
        Factor f;
        if constexpr (F_PARTS == 1) f.part[0] = v;
        else {
            float x[8], none = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = (float)v[j];
            parts_of(x, f.part, none);
        }
        return f;
    }
    struct Row {
        bf16x8 part[2];
    };
    // h of the rows of a tile
    __device__ static __forceinline__ Row row(const Product& p, long row0, int r0, int lane, Odd& odd)
    {
        const int r = r0 + 8 * (lane & 3);
        const f32x4* from = reinterpret_cast<const f32x4*>(p.h + min(row0 + lane / 4, p.rows - 1) * p.padded + min(r, p.padded - 8));
        f32x4 u = from[0], v = from[1];
        if (r >= p.padded) u = v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        u = to_operand(u, lane);
        v = to_operand(v, lane);
        const float x[8] = {u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]};
        Row both;
        parts_of(x, both.part, odd.none);
        return both;
    }
    __device__ static __forceinline__ f32x4 run(const Factor& f, const Row& h, f32x4 c)
    {
        c = mma(f.part[0], h.part[1], c);
        if constexpr (F_PARTS == 2) c = mma(f.part[1], h.part[0], c);
        return mma(f.part[0], h.part[0], c);
    }
};
// In single precision for NM tiles of rows that all belong to adapter a, sixteen r at a time: lane g has four of them, or where the rest of the
// rank is 8 or 4, so that half or three quarters would be zeros, two or one, for as many instructions.
__device__ __forceinline__ f32x4 deal(f32x4 x, int e, int lane)
{
    if (e == 4) return to_operand(x, lane);
    const int n = lane & 15, g = lane >> 4, from = (4 * n + (e == 2 ? g >> 1 : 0)) * 4;
    f32x4 y;
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = __int_as_float(__builtin_amdgcn_ds_bpermute(from, __float_as_int(x[j])));
    if (e == 2) return g & 1 ? f32x4{y[2], y[3], 0.0f, 0.0f} : f32x4{y[0], y[1], 0.0f, 0.0f};
    return f32x4{g & 2 ? (g & 1 ? y[3] : y[2]) : (g & 1 ? y[1] : y[0]), 0.0f, 0.0f, 0.0f};
}
template <int NM, int NT>
__device__ __forceinline__ void add_adapter(const Product& p, int lane, long row0, int col0, int a, f32x4 (&acc)[NM][NT])
{
    const int n = lane & 15, g = lane >> 4;
    const float* F = static_cast<const float*>(p.F) + a * p.f_each;
    const bool runs = p.f_r == 1 && p.rank % 4 == 0;
#pragma unroll 1
    for (int r0 = 0; r0 < p.rank; r0 += 16) {
        const int e = p.rank - r0 == 4 ? 1 : (p.rank - r0 == 8 ? 2 : 4), r = r0 + 4 * (lane & 3);
        f32x4 h[NM], f[NT];
#pragma unroll
        for (int i = 0; i < NM; ++i) h[i] = *reinterpret_cast<const f32x4*>(p.h + min(row0 + 16 * i + lane / 4, p.rows - 1) * p.padded + r);
        if (runs) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
                f[t] = *reinterpret_cast<const Run<float, 4>::loose*>(F + min(col0 + 16 * t + lane / 4, p.cols - 1) * p.f_col + min(r, p.rank - 4));
        } else {      // (the instructions' own order)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) f[t][j] = F[min(col0 + 16 * t + n, p.cols - 1) * p.f_col + min(r0 + e * g + j, p.rank - 1) * p.f_r];
        }
#pragma unroll
        for (int i = 0; i < NM; ++i) h[i] = deal(h[i], e, lane);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if (runs) {
                if (r >= p.rank) f[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                f[t] = deal(f[t], e, lane);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) f[t][j] = r0 + e * g + j < p.rank ? f[t][j] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < NM; ++i) {
                acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(f[t][0], h[i][0], acc[i][t], 0, 0, 0);
                if (e >= 2) acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(f[t][1], h[i][1], acc[i][t], 0, 0, 0);
                if (e == 4) {
                    acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(f[t][2], h[i][2], acc[i][t], 0, 0, 0);
                    acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(f[t][3], h[i][3], acc[i][t], 0, 0, 0);
                }
            }
        }
    }
}
// The adapter of all rows of NM tiles (-1: all have none; -2: they differ).  A row behind the last one has the last one's.
template <int NM>
__device__ __forceinline__ int one_adapter(const Product& p, int lane, long row0)
{
    int a[NM];
#pragma unroll
    for (int i = 0; i < NM; ++i) a[i] = p.index[min(row0 + 16 * i + (lane & 15), p.rows - 1)];
    const int first = __builtin_amdgcn_readfirstlane(a[0]);
    bool same = true;
#pragma unroll
    for (int i = 0; i < NM; ++i) same = same && a[i] == first;
    return __all(same) ? (has_adapter(first, p.adapters) ? first : -1) : -2;
}

// Adds the adapters' part to sums of NM tiles of 16 rows and NT of 16 columns.  For every tile of rows one adapter after the other of
// those that occur in it; a factor that is held as a whole stays for the next tile of rows.  The answer is whether an infinity or NaN was
// among the factors or h.
template <typename T, int NM, int NT>
__device__ __forceinline__ bool add_adapters(const Product& p, int lane, long row0, int col0, f32x4 (&acc)[NM][NT])
{
    typedef AdapterProduct<T> Op;
    const int n = lane & 15;
    __builtin_amdgcn_sched_barrier(0);
    typename Op::Odd odd;
    int a = p.index[min(row0 + n, p.rows - 1)];
    typename Op::Row first = Op::row(p, row0, 0, lane, odd);
    int held = -1;
    typename Op::Factor f[NT];
#pragma unroll
    for (int i = 0; i < NM; ++i) {
        const bool good = row0 + 16 * i + n < p.rows && has_adapter(a, p.adapters);
        unsigned left = (unsigned)__ballot(good) & 0xffffu;
        while (left) {
            const int cur = __builtin_amdgcn_readlane(a, __builtin_ctz(left));
            const bool mine = good && a == cur;
            const unsigned whose = (unsigned)__ballot(mine) & 0xffffu;
            left &= ~whose;
            for (int r0 = 0; r0 < p.rank; r0 += Op::CHUNK) {
                const typename Op::Row hr = r0 == 0 ? first : Op::row(p, row0 + 16 * i, r0, lane, odd);
                if (cur != held || r0 > 0) {
#pragma unroll
                    for (int t = 0; t < NT; ++t)
                        f[t] = Op::factor(p, static_cast<const T*>(p.F) + cur * p.f_each, col0, t, r0, lane, odd);
                    held = p.rank <= Op::CHUNK ? cur : -1;
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const f32x4 sum = Op::run(f[t], hr, f32x4{0, 0, 0, 0});
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][t][j] += mine ? sum[j] : 0.0f;
                }
            }
        }
        if (i + 1 < NM) {
            a = p.index[min(row0 + 16 * (i + 1) + n, p.rows - 1)];
            first = Op::row(p, row0 + 16 * (i + 1), 0, lane, odd);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    return odd.any();
}
template <typename T, int NM, int NT>
__device__ __forceinline__ void store_tiles(const Product& p, int lane, long row0, int col0, const f32x4 (&acc)[NM][NT])
{
    // (64 bytes of a row by four neighbouring lanes)
    constexpr int STEP = std::is_same_v<T, float> ? 1 : 2, N = 4 * STEP;
#pragma unroll
    for (int i = 0; i < NM; ++i) {
        const long row = row0 + 16 * i + lane / 4;
        const bool live = row < p.rows;
        T* out = static_cast<T*>(p.out) + row * p.out_stride;
#pragma unroll
        for (int t = 0; t < NT; t += STEP) {
            typename Run<T, N>::type v;
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = (T)acc[i][t + j / 4][j % 4];
            v = from_operand(v, lane);
            const int col = col0 + 16 * t + N * (lane & 3);
            if (!live) continue;
            if (p.cols - col >= N) *reinterpret_cast<typename Run<T, N>::loose*>(out + col) = v;
            else {
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (col + j < p.cols) out[col + j] = v[j];
            }
        }
        if (__builtin_expect(live && is_bad(p.index[row], p.adapters), 0))
            for (int c = col0 + (lane & 3); c < min(col0 + 16 * NT, p.cols); c += 4) out[c] = (T)std::numeric_limits<float>::quiet_NaN();
    }
}

// Results that are not finite, formed again with the adapters' part in single precision: an infinity times the second part of another
// number, which has any sign or is zero, is not what it is times the number.  (From what is stored, so that the sums need not be kept.)
template <typename T, int NM, int NT>
__device__ __forceinline__ void form_again(const Product& p, int lane, long row0, int col0)
{
    typedef typename Operand<T>::type frag;
    const int n = lane & 15, g = lane >> 4;
    __threadfence_block();
#pragma unroll 1
    for (int i = 0; i < NM * NT; ++i) {
        const long at = row0 + i / NT * 16 + n, row = min(at, p.rows - 1);
        const int t = i % NT, a = p.index[row], col = col0 + column_of<T>(t, 4 * g);
        const T* x = static_cast<const T*>(p.in) + row * p.in_stride + 8 * g;
        const T* w = static_cast<const T*>(p.W) + min(col0 + column_of<T>(t, n), p.cols - 1) * p.w_stride + 8 * g;
        f32x4 sum{0, 0, 0, 0};
#pragma unroll 1
        for (int k = 0; k < p.k_padded; k += kPiece) sum = mma(*reinterpret_cast<const frag*>(w + k), *reinterpret_cast<const frag*>(x + k), sum);
        if (at >= p.rows || !has_adapter(a, p.adapters)) continue;
        const float* h = p.h + row * p.padded;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            T* out = static_cast<T*>(p.out) + row * p.out_stride + col + j;
            if (col + j >= p.cols || fabsf((float)*out) <= std::numeric_limits<float>::max()) continue;
            const T* F = static_cast<const T*>(p.F) + a * p.f_each + (col + j) * p.f_col;
            float part = 0.0f;
#pragma unroll 1
            for (int r = 0; r < p.rank; ++r) part = fmaf(h[r], (float)F[r * p.f_r], part);
            *out = (T)(sum[j] + part);
        }
    }
}

// the sums of a part of k
template <typename T, int NM, int NT>
__device__ __forceinline__ void store_partial(const Product& p, int lane, long row0, int col0, const f32x4 (&acc)[NM][NT])
{
#pragma unroll
    for (int i = 0; i < NM; ++i) {
        const long row = row0 + 16 * i + (lane & 15);
        if (row >= p.rows) continue;
        float* out = p.partial + ((long)blockIdx.y * p.rows + row) * p.cols;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int col = col0 + column_of<T>(t, 4 * (lane >> 4));
            const float v[4] = {acc[i][t][0], acc[i][t][1], acc[i][t][2], acc[i][t][3]};
            store_run<4>(out + col, p.cols - col, v);
        }
    }
}

// 16-bit types.  Tiles of 64 terms come straight from memory into LDS, STAGES of them under way; WM x WN wavefronts share the tile.
// A load brings eight rows of 128 bytes; the 16-byte pieces of a row lie in an order that depends on the row, so that lanes that read
// together meet different banks.  A step of 32 terms has its operands fetched during the step before.
// Bound by the matrix instructions: 8 179 rows, 4 096 x 4 096 in bfloat16, rank 32: 240 to 265 us with the adapters' part, 1.03 to 1.14 PFLOP/s;
// 4 091 rows, 2 048 x 2 048 in float16: 46 us, 0.75.  Tiles of 256 x 256 need half the bytes of 128 x 128 ones for a product but leave CUs without
// work where there are few: the first 268 us, and 316 in tiles of 128 x 128; the second (128 of the large tiles) 63, and 46.
template <typename T, int BM, int BN, int WM, int WN, int STAGES>
__global__ __launch_bounds__(64 * WM * WN, 2) void k_product16(const Product p)
{
    constexpr int WAVES = WM * WN, NM = BM / WM / 16, NT = BN / WN / 16, PER = (BM + BN) / 8 / WAVES, STAGE = (BM + BN) * 128;
    static_assert((BM + BN) / 8 % WAVES == 0, "loads of a wavefront");
    typedef typename Operand<T>::type frag;
    extern __shared__ __align__(16) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    int rt, ct;
    if (!tile_of(p, rt, ct)) return;
    const long row0 = (long)rt * BM;
    const int col0 = ct * BN;
    constexpr bool SPLIT = BM == 64;      // (parts of long sums: of the small tiles alone)
    const int first = SPLIT ? blockIdx.y * p.split_steps : 0;      // (a multiple of two steps)
    const char* x_base = static_cast<const char*>(p.in) + 2 * (row0 * p.in_stride + first * kPiece);
    const char* w_base = static_cast<const char*>(p.W) + 2 * ((long)col0 * p.w_stride + first * kPiece);
    unsigned from[PER];
    unsigned second = 0;      // loads whose piece is in the second half of its row's 128 bytes
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        const int chunk = wave + u * WAVES;
        int piece;
        if (chunk < BM / 8) {
            const int r = chunk * 8 + lane / 8;
            piece = (lane & 7) ^ (r & 7);
            from[u] = (unsigned)(2 * min((long)r, p.rows - 1 - row0) * p.in_stride) + 16 * piece;
        } else {
            const int r = (chunk - BM / 8) * 8 + lane / 8;
            piece = (lane & 7) ^ ((r & 3) | (r >> 3 & 1) << 2);
            from[u] = (unsigned)(2 * min(r, p.cols - 1 - col0) * p.w_stride) + 16 * piece;
        }
        second |= (unsigned)(piece >> 2) << u;
    }
    const unsigned lds0 = lds_address(lds);
    const int all = p.k_padded / kPiece, steps = SPLIT ? min(all - first, p.split_steps) : all, stages = (steps + 1) / 2;
    auto request = [&](int s) {
        const unsigned to = lds0 + s % STAGES * STAGE + wave * 1024;
#pragma unroll
        for (int u = 0; u < PER; ++u)
            load_into_lds((wave + u * WAVES < BM / 8 ? x_base : w_base) + (long)s * 128, from[u], to + u * WAVES * 1024);
    };
    auto request_half = [&](int s) {      // of rows that end in the middle: the first half twice
        const unsigned to = lds0 + s % STAGES * STAGE + wave * 1024;
#pragma unroll
        for (int u = 0; u < PER; ++u)
            load_into_lds((wave + u * WAVES < BM / 8 ? x_base : w_base) + (long)s * 128, from[u] - (second >> u & 1) * 64, to + u * WAVES * 1024);
    };
    auto request_last = [&](int s) {
        if (2 * s + 1 == steps) request_half(s);
        else request(s);
    };
    f32x4 acc[NM][NT];
#pragma unroll
    for (int i = 0; i < NM; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[i][t] = f32x4{0, 0, 0, 0};
    const int wm = wave / WN, wn = wave % WN;
    const unsigned char* xs[2];
    const unsigned char* ws[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        xs[h] = lds + (wm * NM * 16 + n) * 128 + 16 * ((4 * h + g) ^ (n & 7));
        ws[h] = lds + (BM + wn * NT * 16 + column_of<T>(0, n)) * 128 + 16 * ((4 * h + g) ^ ((n & 3) | (n >> 2 & 1) << 2));
    }
    struct Frags {
        frag x[NM], w[NT];
    };
    auto fetch = [&](int s, int h, Frags& f) {
        const int at = s % STAGES * STAGE;
#pragma unroll
        for (int t = 0; t < NT; ++t) f.w[t] = *reinterpret_cast<const frag*>(ws[h] + at + column_of<T>(t, 0) * 128);
#pragma unroll
        for (int i = 0; i < NM; ++i) f.x[i] = *reinterpret_cast<const frag*>(xs[h] + at + i * 2048);
    };
    auto sums = [&](const Frags& now) {
#pragma unroll
        for (int i = 0; i < NM; ++i)
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[i][t] = mma(now.w[t], now.x[i], acc[i][t]);
    };
    auto woven = [&] {      // sums and the fetches beside them, by turns
#pragma unroll
        for (int i = 0; i < NM + NT; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, NM * NT / (NM + NT), 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, NM * NT - NM * NT / (NM + NT) * (NM + NT), 0);
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int s = 0; s < STAGES; ++s)
        if (s < stages) request_last(s);
    if (STAGES <= stages) wait_loads<(STAGES - 1) * PER>();
    else wait_loads<0>();
    barrier_only();
    Frags f[2];
    fetch(0, 0, f[0]);
    int s = 0;
#pragma unroll 1
    for (; s + STAGES + 1 < stages; ++s) {
        fetch(s, 1, f[1]);
        sums(f[0]);
        woven();
        wait_loads<(STAGES - 2) * PER>();
        barrier_only();      // the next tiles are there, and everybody has read these
        request(s + STAGES);
        fetch(s + 1, 0, f[0]);
        sums(f[1]);
        woven();
    }
#pragma unroll 1
    for (; s < stages; ++s) {      // the last request, and none
        if (2 * s + 1 < steps) fetch(s, 1, f[1]);
        sums(f[0]);
        if (s + 1 < stages) {
            wait_loads<0>();
            barrier_only();
            if (s + STAGES < stages) request_last(s + STAGES);
            fetch(s + 1, 0, f[0]);
        }
        if (2 * s + 1 < steps) sums(f[1]);
    }
    const long row_w = row0 + wm * NM * 16;
    const int col_w = col0 + wn * NT * 16;
    if constexpr (SPLIT)
        if (p.splits > 1) {
            store_partial<T, NM, NT>(p, lane, row_w, col_w, acc);
            return;
        }
    const bool odd = add_adapters<T, NM, NT>(p, lane, row_w, col_w, acc);
    store_tiles<T, NM, NT>(p, lane, row_w, col_w, acc);
    if (__builtin_expect(odd, 0)) form_again<T, NM, NT>(p, lane, row_w, col_w);
}

// Single precision on the bf16 matrix instructions: both operands in three parts, exactly, of whose products the six largest are formed
// (what is left out is below 1.002 2^-24 of a product), small ones first.  Numbers are brought up by 2^24 first, so that the parts of
// small ones are normal numbers; sums that are not finite for it, or are not at all, are formed again in single precision.
// A wavefront has 16 NM rows of its own, which it reads and splits in registers, a step of 32 terms ahead; W's parts, split beforehand, lie
// in memory as they go into LDS, where the four wavefronts share them.
// Six bf16 products a product: 50 000 rows, 256 -> 512 in 80 us, 164 TFLOP/s of single precision, 0.98 PFLOP/s of the instructions; the splits
// beside them and the short sums (eight steps, then 128 x 128 numbers to store) keep it from more.  The 154 TFLOP/s that a large product on the
// single-precision instructions reaches would be 85 us.
template <int NM, int NT>
__global__ __launch_bounds__(256, NM == 1 ? 4 : 3) void k_product32(const Product p)
{
    constexpr int BM = 64 * NM, BN = 16 * NT, STAGE = 3 * BN * 64, PER = STAGE / 4096;
    constexpr bool SPLIT = NM == 1;      // (parts of long sums: of the small tiles alone)
    __shared__ __align__(16) unsigned char lds[2 * STAGE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    int rt, ct;
    if (!tile_of(p, rt, ct)) return;
    const long row0 = (long)rt * BM + wave * 16 * NM;
    const int col0 = ct * BN, all = p.k_padded / kPiece, first = SPLIT ? blockIdx.y * p.split_steps : 0, steps = SPLIT ? min(all - first, p.split_steps) : all;
    const int begin = first * kPiece, rest = p.k - begin;      // numbers of a row from this part on
    const float* from[NM];
#pragma unroll
    for (int i = 0; i < NM; ++i) from[i] = static_cast<const float*>(p.in) + min(row0 + 16 * i + n, p.rows - 1) * p.in_stride + begin;
    const char* w_base = static_cast<const char*>(p.W) + ((long)(col0 / kPartRows) * all + first) * (3 * kPartRows * 64) + col0 % kPartRows * 64;
    const unsigned lds0 = lds_address(lds) + wave * PER * 1024;
    f32x4 raw[NM][2];
    auto request = [&](int s) {
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            const int chunk = wave * PER + u, part = chunk / NT;
            load_into_lds(w_base + (long)s * (3 * kPartRows * 64) + part * kPartRows * 64 + chunk % NT * 1024, lane * 16, lds0 + s % 2 * STAGE + u * 1024);
        }
        const int k = s * kPiece + 8 * g;
        if ((s + 1) * kPiece <= rest) {
#pragma unroll
            for (int i = 0; i < NM; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) raw[i][h] = *reinterpret_cast<const Run<float, 4>::loose*>(from[i] + k + 4 * h);
        } else {
#pragma unroll
            for (int i = 0; i < NM; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float x = from[i][min(k + j, rest - 1)];
                    raw[i][j / 4][j % 4] = k + j < rest ? x : 0.0f;
                }
        }
        asm volatile("" ::: "memory");      // (asked for here, not where they are used)
    };
    f32x4 acc[NM][NT];
#pragma unroll
    for (int i = 0; i < NM; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[i][t] = f32x4{0, 0, 0, 0};
    const unsigned char* ws = lds + n * 64 + 16 * (g ^ (n >> 1 & 3));
    request(0);
#pragma unroll 1
    for (int s = 0; s < steps; ++s) {
        bf16x8 x[NM][3];
#pragma unroll
        for (int i = 0; i < NM; ++i) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = raw[i][j / 4][j % 4] * kSplitScale;
            bf16 part[3][8];
            split(v, part);
#pragma unroll
            for (int q = 0; q < 3; ++q)
#pragma unroll
                for (int j = 0; j < 8; ++j) x[i][q][j] = part[q][j];
        }
        wait_loads<0>();
        barrier_only();      // this step's parts are there, and everybody has read those of the step before
        if (s + 1 < steps) request(s + 1);
        const unsigned char* at = ws + s % 2 * STAGE;
        // two tiles of columns at a time, the operands of the next two under way
        bf16x8 w[2][2][3];
        auto fetch = [&](int t) {
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int q = 0; q < 3; ++q) w[t / 2 % 2][c][q] = *reinterpret_cast<const bf16x8*>(at + q * BN * 64 + (t + c) * 1024);
        };
        fetch(0);
        __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
        for (int t = 0; t < NT; t += 2) {
            if (t + 2 < NT) fetch(t + 2);
            constexpr int ix[6] = {2, 0, 1, 1, 0, 0}, iw[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
            for (int o = 0; o < 6; ++o)
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int i = 0; i < NM; ++i) acc[i][t + c] = mma(w[t / 2 % 2][c][iw[o]], x[i][ix[o]], acc[i][t + c]);
            if (t + 2 < NT) __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 12 * NM, 0);
        }
    }
    constexpr float kBack = 1.0f / (kSplitScale * kSplitScale);
#pragma unroll
    for (int i = 0; i < NM; ++i) {
        float none[4] = {0.0f, 0.0f, 0.0f, 0.0f};      // NaN if a sum is not finite
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                none[j] = fmaf(acc[i][t][j], 0.0f, none[j]);
                acc[i][t][j] *= kBack;
            }
        const float any = (none[0] + none[1]) + (none[2] + none[3]);
        if (__builtin_expect(__any(any != any), 0)) {
            const float* row = static_cast<const float*>(p.in) + min(row0 + 16 * i + n, p.rows - 1) * p.in_stride;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll 1
                for (int j = 0; j < 4; ++j) {
                    const float* wc = static_cast<const float*>(p.W0) + min(col0 + 16 * t + 4 * g + j, p.cols - 1) * p.w0_col;
                    float sum = 0.0f;
                    for (int k = begin; k < min(p.k, begin + steps * kPiece); ++k) sum = fmaf(row[k], wc[k * p.w0_k], sum);
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        if (c == j && !(fabsf(acc[i][t][c]) <= std::numeric_limits<float>::max())) acc[i][t][c] = sum;
                }
        }
    }
    if constexpr (SPLIT)
        if (p.splits > 1) {
            store_partial<float, NM, NT>(p, lane, row0, col0, acc);
            return;
        }
    const int one = one_adapter<NM>(p, lane, row0);
    if (one >= 0) add_adapter<NM, NT>(p, lane, row0, col0, one, acc);
    store_tiles<float, NM, NT>(p, lane, row0, col0, acc);
}

// Where the rows of a wavefront of k_product32 have different adapters, their part is added here, to the stored sums: a block takes
// eight of the `group` rows of one, a lane a column.  (A launch of its own: the registers for it would cost k_product32 a
// block on every CU, and the few tiles that are mixed where requests are runs of rows would be its last ones: 95 us against 80 and 8,
// 50 000 rows of 256 numbers, 512 columns, 12 adapters of rank 8.)
__global__ __launch_bounds__(256) void k_add_mixed(const Product p, int group)
{
    const int lane = threadIdx.x & 63;
    const long row0 = (long)blockIdx.x * group;
    const int mine = p.index[min(row0 + lane % group, p.rows - 1)];
    if (__all(mine == __builtin_amdgcn_readfirstlane(mine))) return;
    const int col = blockIdx.y * 256 + threadIdx.x;
    if (col >= p.cols) return;
    const bool runs = p.f_r == 1 && p.rank % 4 == 0;
    float* out = static_cast<float*>(p.out) + col;
    const float* F0 = static_cast<const float*>(p.F) + col * p.f_col;
    {
        const int i0 = 8 * blockIdx.z;
        float y[8], sum[8];
        const float* F[8];
        const float* h[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const long row = min(row0 + i0 + u, p.rows - 1);
            const int a = __builtin_amdgcn_readlane(mine, i0 + u);
            F[u] = F0 + (has_adapter(a, p.adapters) ? a : 0) * p.f_each;
            h[u] = p.h + row * p.padded;
            y[u] = out[row * p.out_stride];
            sum[u] = 0.0f;
        }
#pragma unroll 1
        for (int r = 0; r < p.rank; r += 4) {
            f32x4 f[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                if (runs) f[u] = *reinterpret_cast<const Run<float, 4>::loose*>(F[u] + r);
                else {
#pragma unroll
                    for (int q = 0; q < 4; ++q) f[u][q] = F[u][min(r + q, p.rank - 1) * p.f_r];
                }
            }
#pragma unroll
            for (int u = 0; u < 8; ++u)
#pragma unroll
                for (int q = 0; q < 4; ++q) sum[u] = r + q < p.rank ? fmaf(h[u][r + q], f[u][q], sum[u]) : sum[u];
        }
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (row0 + i0 + u < p.rows && has_adapter(__builtin_amdgcn_readlane(mine, i0 + u), p.adapters)) out[(row0 + i0 + u) * p.out_stride] = y[u] + sum[u];
    }
}

// The parts of a product split along k, in order, with the adapters' part: a thread has a column of a row.
template <typename T>
__global__ __launch_bounds__(256) void k_join_splits(const Product p)
{
    const long row = blockIdx.x;
    const int col = blockIdx.y * 256 + threadIdx.x, a = p.index[row];
    if (col >= p.cols) return;
    float sum = 0.0f;
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) sum += p.partial[((long)s * p.rows + row) * p.cols + col];
    if (has_adapter(a, p.adapters)) {
        const T* F = static_cast<const T*>(p.F) + a * p.f_each + col * p.f_col;
        const float* h = p.h + row * p.padded;
        float part = 0.0f;
        if (p.f_runs) {
            for (int r = 0; r < p.rank; r += 8) {
                float f[8];
                load_run<8>(F + r, 8, f);
#pragma unroll
                for (int j = 0; j < 8; ++j) part = fmaf(h[r + j], f[j], part);
            }
        } else {
#pragma unroll 8
            for (int r = 0; r < p.rank; ++r) part = fmaf(h[r], (float)F[r * p.f_r], part);
        }
        sum += part;
    }
    static_cast<T*>(p.out)[row * p.out_stride + col] = is_bad(a, p.adapters) ? (T)std::numeric_limits<float>::quiet_NaN() : (T)sum;
}

// Few rows: a block takes 16 columns and all rows; eight wavefronts have 128 bytes of W's rows by turns, four units of them under way.
// Bound by W's bytes: 16 rows, 4 096 x 4 096 in bfloat16: 8.4 us, 4.0 TB/s.
template <typename T, int MT>
__global__ __launch_bounds__(512) void k_product_few(const Product p)
{
    constexpr int V = kRun<T>, UNIT = 8 * V;
    typedef typename Operand<T>::type frag;
    __shared__ f32x4 part[8][MT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col0 = blockIdx.x * 16, mine = (lane & 3) * V;
    const T* W = static_cast<const T*>(p.W0) + (long)min(col0 + lane / 4, p.cols - 1) * p.w0_col + mine;
    const T* in[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) in[i] = static_cast<const T*>(p.in) + min(16L * i + lane / 4, p.rows - 1) * p.in_stride + mine;
    f32x4 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = f32x4{0, 0, 0, 0};
    struct Unit {
        frag w[2], x[MT][2];
    };
    const int full = p.k / UNIT;
    auto fetch = [&](int u, Unit& v) {
        const long k = (long)min(u, full - 1) * UNIT;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            v.w[half] = *reinterpret_cast<const typename Run<T, V>::loose*>(W + k + half * (UNIT / 2));
#pragma unroll
            for (int i = 0; i < MT; ++i) v.x[i][half] = *reinterpret_cast<const typename Run<T, V>::loose*>(in[i] + k + half * (UNIT / 2));
        }
        asm volatile("" ::: "memory");      // (asked for here, not where they are used)
    };
    auto sums = [&](const Unit& v) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const frag w = to_operand(v.w[half], lane);
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[i] = mma(w, to_operand(v.x[i][half], lane), acc[i]);
        }
    };
    int u = wave;
    if (u < full) {
        Unit unit[4];
#pragma unroll
        for (int q = 0; q < 3; ++q) fetch(u + 8 * q, unit[q]);
#pragma unroll 1
        for (;;) {
            bool done = false;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (done) continue;
                fetch(u + 24, unit[(q + 3) % 4]);
                sums(unit[q]);
                done = (u += 8) >= full;
            }
            if (done) break;
        }
    }
    if (wave == full % 8 && p.k % UNIT) {      // (the end of the rows)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int k = full * UNIT + half * (UNIT / 2);
            const frag w = to_operand(load_operand(W + k, p.k - k - mine), lane);
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[i] = mma(w, to_operand(load_operand(in[i] + k, p.k - k - mine), lane), acc[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) part[wave][i][lane] = acc[i];
    __syncthreads();
    for (int at = threadIdx.x; at < MT * 256; at += 512) {
        const int row = at / 16, c = at % 16, col = col0 + c;
        if (row >= p.rows || col >= p.cols) continue;
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) sum += part[w][row / 16][c / 4 * 16 + row % 16][c % 4];
        const int a = p.index[row];
        if (has_adapter(a, p.adapters)) {
            const T* F = static_cast<const T*>(p.F) + a * p.f_each + (long)col * p.f_col;
            const float* h = p.h + (long)row * p.padded;
            float both = 0.0f;
            for (int r = 0; r < p.rank; r += 8) {
                float f[8];
                load_run<8>(F + r, p.rank - r, f);
#pragma unroll
                for (int j = 0; j < 8; ++j) both = fmaf(h[r + j], f[j], both);
            }
            sum += both;
        }
        static_cast<T*>(p.out)[(long)row * p.out_stride + col] = is_bad(a, p.adapters) ? (T)std::numeric_limits<float>::quiet_NaN() : (T)sum;
    }
}

// ---- sums over rows of h[row][r] in[row][col], by pieces of an adapter's rows

struct Outer {
    const void* in;
    long in_stride;
    const float* h;
    const int *start, *first, *perm;
    int adapters, rank, padded, cols, piece;
    float* partial;      // [piece][rank][cols]
    void* out;
    long out_each, out_r, out_col;
};
struct Outers {
    Outer outer[2];
    int blocks[2];      // of columns
};
// A block takes a piece, 64 r at most, and 64 V columns; a wavefront 16 V of them, four rows at a time, in single precision whatever the
// type.  Rows are read once for each 64 r; with the rows' indirection, bound by the latency of loads: 18 us for 4 091 rows of 2 048 and
// 2 048 numbers in float16, 14 for 20 011 of 256 and 512 in single precision (61 MB, 4.3 TB/s).
template <typename T, int RT>
__global__ __launch_bounds__(256) void k_outer(const Outers both)
{
    constexpr int V = kRun<T>, U = 4;
    const bool second = (int)blockIdx.y >= both.blocks[0];
    const Outer& p = both.outer[second];
    const int slab = second ? blockIdx.y - both.blocks[0] : blockIdx.y;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4, item = blockIdx.x;
    if (item >= p.first[p.adapters]) return;
    int low = 0, high = p.adapters;
    while (high - low > 1) {
        const int mid = (low + high) / 2;
        if (p.first[mid] <= item) low = mid;
        else high = mid;
    }
    const int begin = p.start[low] + (item - p.first[low]) * p.piece, end = min(begin + p.piece, p.start[low + 1]);
    const int col = (slab * 4 + wave) * 16 * V + V * n, r0 = blockIdx.z * 64;
    if ((slab * 4 + wave) * 16 * V >= p.cols) return;
    const T* in = static_cast<const T*>(p.in) + col;
    const float* h = p.h + r0 + n;
    const bool whole = (slab * 4 + wave + 1) * 16 * V <= p.cols;
    f32x4 acc[RT][V];
#pragma unroll
    for (int q = 0; q < RT; ++q)
#pragma unroll
        for (int t = 0; t < V; ++t) acc[q][t] = f32x4{0, 0, 0, 0};
    for (int at = begin; at < end; at += 64) {
        const int mine = p.perm[min(at + lane, end - 1)];      // the rows of the next 64
#pragma unroll 1
        for (int i0 = 0; i0 < min(64, end - at); i0 += 4 * U) {
            typename Operand<T>::type x[U];
            float hv[U][RT];
            bool live[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + 4 * u + g;
                live[u] = at + i < end;
                const long row = __shfl(mine, i, 64);
                if (whole) x[u] = *reinterpret_cast<const typename Run<T, V>::loose*>(in + row * p.in_stride);
                else x[u] = load_operand(in + row * p.in_stride, p.cols - col);
#pragma unroll
                for (int q = 0; q < RT; ++q) hv[u][q] = r0 + 16 * q + n < p.rank ? h[row * p.padded + 16 * q] : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int t = 0; t < V; ++t) {
                    const float v = live[u] ? (float)x[u][t] : 0.0f;
#pragma unroll
                    for (int q = 0; q < RT; ++q) acc[q][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(live[u] ? hv[u][q] : 0.0f, v, acc[q][t], 0, 0, 0);
                }
        }
    }
    float* out = p.partial + (long)item * p.rank * p.cols + col;
#pragma unroll
    for (int q = 0; q < RT; ++q)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = r0 + 16 * q + 4 * g + j;
            float v[V];
#pragma unroll
            for (int t = 0; t < V; ++t) v[t] = acc[q][t][j];
            if (r < p.rank) store_run<V>(out + (long)r * p.cols, p.cols - col, v);
        }
}
// The pieces of an adapter, in order: a block takes 64 numbers, four threads each.
template <typename T>
__global__ __launch_bounds__(256) void k_join(const Outers both)
{
    __shared__ float part[4][64];
    const Outer& p = both.outer[blockIdx.z];
    const int a = blockIdx.y, each = p.rank * p.cols, lane = threadIdx.x & 63, q = threadIdx.x >> 6, e = blockIdx.x * 64 + lane;
    if ((int)blockIdx.x * 64 >= each) return;
    float sum = 0.0f;
    if (e < each) {
        const float* from = p.partial + e;
        const int last = p.first[a + 1];
#pragma unroll 4
        for (int i = p.first[a] + q; i < last; i += 4) sum += from[(long)i * each];
    }
    part[q][lane] = sum;
    __syncthreads();
    if (q == 0 && e < each) {
        sum = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
        const int r = e / p.cols, col = e % p.cols;
        static_cast<T*>(p.out)[a * p.out_each + r * p.out_r + col * p.out_col] = (T)sum;
    }
}

// ---- host side

void check(const smx_adapted_linear* p)
{
    refuse_unless(p, "the description must not be null");
    (void)type_bytes(p->type);
    refuse_unless(p->rows >= 0 && p->rows <= 1L << 28, "rows: 0 to 2^28");
    refuse_unless(p->d_in >= 1 && p->d_out >= 1 && p->d_in <= (1 << 20) && p->d_out <= (1 << 20), "d_in and d_out: 1 to 2^20");
    refuse_unless(p->rank >= 1 && p->rank <= SMX_ADAPTER_MAX_RANK, "rank: 1 to 128");
    refuse_unless(p->num_adapters >= 0 && p->num_adapters <= SMX_ADAPTER_MAX_COUNT, "num_adapters: 0 to 4096");
    refuse_unless(p->x_stride >= p->d_in && p->weight_stride >= p->d_in, "strides of x and weight: at least d_in");
    refuse_unless(p->weight && (p->num_adapters == 0 || (p->A && p->B)), "weight, A and B must not be null");
    refuse_unless(p->rows == 0 || (p->x && p->index), "x and index must not be null");
}

long up(long x, long m) { return (x + m - 1) / m * m; }

// Parts of the workspace, 256 bytes aligned; counts them first and gives addresses when there is one.
struct Arena {
    char* base;
    long used = 0;
    template <typename P>
    P* take(long count)
    {
        P* at = base ? reinterpret_cast<P*>(base + used) : nullptr;
        used += up(count * (long)sizeof(P), 256);
        return at;
    }
};

// rows that direct loads into LDS can take as they are
// (the offsets inside a tile have 32 bits)
bool as_it_is(const void* p, long stride, long k) { return (reinterpret_cast<size_t>(p) & 15) == 0 && stride % 8 == 0 && stride <= 1 << 22 && k % kPiece == 0; }

template <int N>
using Int = std::integral_constant<int, N>;

struct Call {
    const smx_adapted_linear& p;
    hipStream_t s;
    Arena arena;
    const bool dry;      // nothing is launched, the workspace is counted, and the sizes of the launches are looked at
    const int padded;
    Prepare prepare{};
    Downs downs{};
    int num_layouts = 0, num_downs = 0;
    Call(const smx_adapted_linear& p_, void* base, hipStream_t s_, bool dry_)
        : p(p_), s(s_), arena{static_cast<char*>(base)}, dry(dry_), padded((int)up(p_.rank, 16)) {}

    // Every launch, also of a call that counts its workspace and launches nothing: sizes that a launch does not take are refused there,
    // before the call has enqueued anything.
    template <typename... P, typename... A>
    void start(void (*kernel)(P...), long x, long y, long z, int threads, unsigned lds, const A&... args)
    {
        refuse_unless(x >= 1 && y >= 1 && z >= 1, "a launch of no blocks");
        refuse_unless(x * threads < 1L << 32 && y <= 65535 && z <= 65535, "more blocks than a launch takes");
        if (!dry) hipLaunchKernelGGL(kernel, dim3((unsigned)x, (unsigned)y, (unsigned)z), dim3(threads), lds, s, args...);
    }

    // fn(first, some): as many blocks at a time as a launch takes of 1 024 threads
    template <typename Fn>
    static void in_slabs(long blocks, Fn&& fn)
    {
        constexpr long most = 1L << 21;
        for (long first = 0; first < blocks; first += most) fn(first, std::min(blocks - first, most));
    }

    template <typename T>
    void lay_out(const void* src, long src_each, long src_row, long src_k, void* dst, bool parts, long rows, int k, int matrices)
    {
        const int k_padded = (int)up(k, kPiece);
        if (num_layouts == 2) flush_layouts<T>();
        const long padded_rows = parts ? up(rows, kPartRows) : rows;
        const Layout l{src, src_each, src_row, src_k, dst, padded_rows * k_padded, (int)padded_rows, k, k_padded, matrices, parts, (int)rows};
        prepare.blocks[num_layouts] = layout_blocks(l);
        prepare.layout[num_layouts++] = l;
    }
    // launches what is laid out, and the count of rows if it is due
    template <typename T>
    void flush_layouts(bool count = false)
    {
        const long blocks = prepare.blocks[0] + prepare.blocks[1] + (count ? prepare.groups.blocks : 0);
        in_slabs(blocks, [&](long first, long some) {
            prepare.first = first;
            start(k_prepare<T>, some, 1, 1, 256, 0, prepare);
        });
        prepare.blocks[0] = prepare.blocks[1] = 0;
        num_layouts = 0;
    }

    template <typename T>
    void down(const T* in, long in_stride, const T* F, long f_each, long f_row, int k, float* h)
    {
        downs.down[num_downs++] = Down{in, in_stride, F, f_each, f_row, p.scale, p.index, p.num_adapters, p.rank, padded, k, p.rows, h};
    }
    template <typename T>
    void flush_downs(bool place)
    {
        auto go = [&](auto rt, auto mt, auto waves) {
            constexpr int RT = decltype(rt)::value, MT = decltype(mt)::value, WAVES = decltype(waves)::value;
            for (int i = 0; i < num_downs; ++i) downs.blocks[i] = (int)up((p.rows + 16 * MT - 1) / (16 * MT), 8);
            const long blocks = (long)downs.blocks[0] + downs.blocks[1] + (place ? downs.groups.blocks : 0);
            in_slabs(blocks, [&](long first, long some) {
                downs.first = (int)first;
                start(k_down<T, RT, MT, WAVES>, some, 1, 1, 64 * WAVES, 0, downs);
            });
        };
        // Wavefronts of a block share its sums.  Few blocks leave most of the chip without work, so they get more wavefronts: 8 where the
        // sums are long (4 091 rows of 2 048 and 2 048 in f16: 12.1 us with 8 of 32 rows, 13.6 with 16 of 16 rows), and below 4 096 rows in
        // all 16 of 16 rows each (1 840 rows of 2 207 in single precision: 21 us, and 48 with 4; 300 of 4 096 in bfloat16: 15 and 23).
        const bool long_rows = downs.down[0].k >= 1024, few_blocks = p.rows / 16 * num_downs < 4096, very_few = p.rows / 32 * num_downs < 128 && downs.down[0].k >= 256;
        if (padded == 16) very_few ? go(Int<1>{}, Int<1>{}, Int<16>{}) : few_blocks && long_rows ? go(Int<1>{}, Int<2>{}, Int<8>{}) : go(Int<1>{}, Int<2>{}, Int<4>{});
        else if (padded == 32) very_few ? go(Int<2>{}, Int<1>{}, Int<16>{}) : few_blocks && long_rows ? go(Int<2>{}, Int<2>{}, Int<8>{}) : go(Int<2>{}, Int<2>{}, Int<4>{});
        else if (padded <= 64) few_blocks && long_rows ? go(Int<4>{}, Int<1>{}, Int<8>{}) : go(Int<4>{}, Int<2>{}, Int<4>{});
        else go(Int<8>{}, Int<1>{}, Int<4>{});
    }

    // out[rows][cols] = in W^T + adapters' part; W(col, k) = W[col * w_col + k * w_k], F(col, r) = F[a][col * f_col + r * f_r].
    // First what has to be laid out for it, then the product itself.
    template <typename T>
    Product product(const T* in, long in_stride, const T* W, long w_col, long w_k, const T* F, long f_each, long f_col, long f_r, const float* h, int k, int cols, T* out,
                    long out_stride, bool few)
    {
        Product q{};
        q.in = in; q.in_stride = in_stride; q.W0 = W; q.w0_col = w_col; q.w0_k = w_k; q.F = F; q.f_each = f_each; q.f_col = f_col; q.f_r = f_r; q.f_runs = f_r == 1 && p.rank % 8 == 0; q.h = h;
        q.index = p.index; q.adapters = p.num_adapters; q.rank = p.rank; q.padded = padded; q.k = k; q.k_padded = (int)up(k, kPiece); q.cols = cols;
        q.rows = p.rows; q.out = out; q.out_stride = out_stride;
        q.splits = 1;
        q.split_steps = q.k_padded / kPiece + 1;
        if (few) return q;
        // Few tiles and long sums: the sums in parts of at least eight steps, until there are two blocks for every CU.  (40 tiles of 128 steps in
        // bfloat16: 12 us with the joining, 23 without parts; 176 tiles of 64 steps: 18 and 15.)
        const long few_tiles = (p.rows + 63) / 64 * ((cols + 63) / 64);
        const int steps = q.k_padded / kPiece;
        if (few_tiles <= 128 && steps >= 16) {
            q.split_steps = (int)std::max(8L, up((steps * few_tiles + 511) / 512, 2));
            q.splits = (steps + q.split_steps - 1) / q.split_steps;
            if (q.splits > 1) q.partial = arena.take<float>(q.splits * p.rows * cols);
        }
        if constexpr (std::is_same_v<T, float>) {
            bf16* parts = arena.take<bf16>(3 * up(cols, kPartRows) * q.k_padded);
            lay_out<float>(W, 0, w_col, w_k, parts, true, cols, k, 1);
            q.W = parts;
        } else {
            q.W = W; q.w_stride = w_col;
            if (!(w_k == 1 && as_it_is(W, w_col, k))) {
                T* laid = arena.take<T>((long)cols * q.k_padded);
                lay_out<T>(W, 0, w_col, w_k, laid, false, cols, k, 1);
                q.W = laid; q.w_stride = q.k_padded;
            }
            if (!as_it_is(in, in_stride, k)) {
                T* laid = arena.take<T>(p.rows * q.k_padded);
                lay_out<T>(in, 0, in_stride, 1, laid, false, p.rows, k, 1);
                q.in = laid; q.in_stride = q.k_padded;
            }
        }
        return q;
    }
    template <typename T>
    void launch(Product q, bool few)
    {
        if (few) {
            auto go = [&](auto mt) { start(k_product_few<T, decltype(mt)::value>, (q.cols + 15) / 16, 1, 1, 512, 0, q); };
            if (p.rows <= 16) go(Int<1>{});
            else if (p.rows <= 32) go(Int<2>{});
            else go(Int<4>{});
            return;
        }
        auto tiles = [&](int tile_rows, int tile_cols) {
            q.row_tiles = (int)((q.rows + tile_rows - 1) / tile_rows);
            q.col_tiles = (q.cols + tile_cols - 1) / tile_cols;
            return (long)q.row_tiles * q.col_tiles;
        };
        auto blocks = [&] { return up((long)q.row_tiles * q.col_tiles, 8); };
        // Tiles that run at once are done at about the same time: where those of the last such round are few, their rows get a launch of
        // smaller tiles: 8 500 rows, 4 096 x 4 096 in bfloat16, 544 tiles of 256 x 256: 256 + 32 us, and 326 in one launch.  (What is left for it
        // is in q then; the answer is whether there is anything.)  Where not one row of tiles fits into the full rounds all stay in one launch:
        // 200 rows, 1 024 -> 65 792: 79 us, and 89 in smaller tiles; 100 rows to 70 000: 79 and 52.
        auto rounds = [&](int tile_rows, int tile_cols, long at_once, auto&& go) {
            const long all = tiles(tile_rows, tile_cols), over = all % at_once;
            const long full_rows = over > 0 && over <= at_once / 2 ? (all - over) / q.col_tiles * tile_rows : 0, main_rows = full_rows > 0 ? full_rows : q.rows;
            const Product whole = q;
            q.rows = main_rows;
            tiles(tile_rows, tile_cols);
            go();
            q = whole;
            q.rows -= main_rows;
            q.in = static_cast<const T*>(q.in) + main_rows * q.in_stride;
            q.out = static_cast<T*>(q.out) + main_rows * q.out_stride;
            q.h += main_rows * q.padded;
            q.index += main_rows;
            return q.rows > 0;
        };
        auto join = [&] { start(k_join_splits<T>, q.rows, (q.cols + 255) / 256, 1, 256, 0, q); };
        if constexpr (std::is_same_v<T, float>) {
            if (q.splits > 1) {
                tiles(64, 64);
                start(k_product32<1, 4>, blocks(), q.splits, 1, 256, 0, q);
                join();
                return;
            }
            // (large tiles from one for every CU on: 4 090 rows, 1 024 x 1 024: 56 us, and 60 in small ones; 1 500 rows: 50, and 29)
            const bool wide = tiles(128, 128) >= 256;
            if (wide) start(k_product32<2, 8>, blocks(), 1, 1, 256, 0, q);
            else {
                tiles(64, 64);
                start(k_product32<1, 4>, blocks(), 1, 1, 256, 0, q);
            }
            const int group = wide ? 32 : 16;
            if (p.num_adapters) start(k_add_mixed, (q.rows + group - 1) / group, (q.cols + 255) / 256, group / 8, 256, 0, q, group);
        } else {
            auto go = [&](auto bm, auto bn, auto wm, auto wn, auto stages) {
                constexpr int BM = decltype(bm)::value, BN = decltype(bn)::value, WM = decltype(wm)::value, WN = decltype(wn)::value, S = decltype(stages)::value;
                constexpr int bytes = S * (BM + BN) * 128;
                if (bytes > 64 * 1024 && !dry)
                    hip_ok(hipFuncSetAttribute(reinterpret_cast<const void*>(&k_product16<T, BM, BN, WM, WN, S>), hipFuncAttributeMaxDynamicSharedMemorySize, bytes), "LDS");
                start(k_product16<T, BM, BN, WM, WN, S>, blocks(), q.splits, 1, 64 * WM * WN, bytes, q);
            };
            if (q.splits > 1) {
                tiles(64, 64);
                go(Int<64>{}, Int<64>{}, Int<2>{}, Int<2>{}, Int<3>{});
                join();
                return;
            }
            // Tiles as large as keep three quarters of the CUs busy (figures at k_product16; 512 tiles of 128 x 128: 46 us, and 67 in tiles of
            // 64 x 64; 96 of them: 23, and 14).
            if (tiles(256, 256) >= 192 && !rounds(256, 256, 256, [&] { go(Int<256>{}, Int<256>{}, Int<2>{}, Int<4>{}, Int<2>{}); })) return;
            if (tiles(128, 128) >= 192 && !rounds(128, 128, 512, [&] { go(Int<128>{}, Int<128>{}, Int<2>{}, Int<2>{}, Int<2>{}); })) return;
            tiles(64, 64);
            go(Int<64>{}, Int<64>{}, Int<2>{}, Int<2>{}, Int<3>{});
        }
    }

    template <typename T>
    void forward(T* y, long y_stride)
    {
        const bool few = p.rows <= kMostFew;
        const T *x = static_cast<const T*>(p.x), *W = static_cast<const T*>(p.weight), *A = static_cast<const T*>(p.A), *B = static_cast<const T*>(p.B);
        float* h = arena.take<float>(p.rows * padded);
        const Product q = product(x, p.x_stride, W, p.weight_stride, 1, B, (long)p.rank * p.d_out, p.rank, 1, h, p.d_in, p.d_out, y, y_stride, few);
        flush_layouts<T>();
        down(x, p.x_stride, A, (long)p.rank * p.d_in, p.d_in, p.d_in, h);
        if (!few) flush_downs<T>(false);
        else start(k_down_few<T>, p.rows, padded / 4, 1, 256, 0, downs.down[0]);
        launch<T>(q, few);
    }

    template <typename T>
    void backward(const T* dy, long dy_stride, T* dx, long dx_stride, T* dA, T* dB)
    {
        const T *x = static_cast<const T*>(p.x), *W = static_cast<const T*>(p.weight), *A = static_cast<const T*>(p.A), *B = static_cast<const T*>(p.B);
        const long each_a = (long)p.rank * p.d_in, each_b = (long)p.rank * p.d_out;
        const int n = p.num_adapters;
        const bool rows = p.rows > 0, want_x = rows && (dx || dry), want_a = n > 0 && (dA || dry), want_b = n > 0 && (dB || dry), sums = want_a || want_b;
        float *h = arena.take<float>(want_b ? p.rows * padded : 0), *g = arena.take<float>(want_x || want_a ? p.rows * padded : 0);
        Groups& groups = prepare.groups;
        long most = 0;
        float *partial_a = nullptr, *partial_b = nullptr;
        if (sums) {
            groups.index = p.index; groups.adapters = n; groups.rows = p.rows;
            // (a block that places rows reads the counts of all blocks)
            const long most_blocks = std::max(1, std::min(256, 16384 / (n + 2)));
            groups.rows_per_block = (int)std::max(256L, up((p.rows + most_blocks - 1) / most_blocks, 64));
            groups.blocks = (int)std::max(1L, (p.rows + groups.rows_per_block - 1) / groups.rows_per_block);
            groups.piece = (int)std::max(64L, up((p.rows + 511) / 512, 64));
            groups.count = arena.take<int>((long)(n + 2) * groups.blocks);
            groups.start = arena.take<int>(n + 1);
            groups.first = arena.take<int>(n + 1);
            groups.perm = arena.take<int>(p.rows);
            most = std::min<long>(p.rows, p.rows / groups.piece + n);      // pieces: of an adapter's rows, one that is not full
            if (want_a) partial_a = arena.take<float>(most * each_a);
            if (want_b) partial_b = arena.take<float>(most * each_b);
            downs.groups = groups;
        }
        Product q{};
        // B_a^T, so that sums over d_out run along rows
        const int k_padded = (int)up(p.d_out, kPiece);
        T* Bt = nullptr;
        if (want_x || (want_a && rows)) {
            Bt = arena.take<T>((long)n * p.rank * k_padded);
            if (n) lay_out<T>(B, each_b, 1, p.rank, Bt, false, p.rank, p.d_out, n);
            down(dy, dy_stride, Bt, (long)p.rank * k_padded, k_padded, p.d_out, g);
        }
        if (want_b && rows) down(x, p.x_stride, A, each_a, p.d_in, p.d_in, h);
        if (want_x) q = product(dy, dy_stride, W, 1, p.weight_stride, A, each_a, 1, p.d_in, g, p.d_out, p.d_in, dx, dx_stride, false);
        flush_layouts<T>(sums);
        flush_downs<T>(sums);
        if (want_x) launch<T>(q, false);
        if (!sums) return;
        Outers both{};
        Outer o{};
        o.start = groups.start; o.first = groups.first; o.perm = groups.perm; o.adapters = n; o.rank = p.rank; o.padded = padded; o.piece = groups.piece;
        int num = 0, across = 0, widest = 0;
        auto add = [&](const T* in, long in_stride, const float* factor, int cols, float* partial, T* out, long each, long out_r, long out_col) {
            o.in = in; o.in_stride = in_stride; o.h = factor; o.cols = cols; o.partial = partial; o.out = out; o.out_each = each; o.out_r = out_r; o.out_col = out_col;
            both.blocks[num] = (cols + 64 * kRun<T> - 1) / (64 * kRun<T>);
            across += both.blocks[num];
            widest = std::max(widest, cols);
            both.outer[num++] = o;
        };
        if (want_a) add(x, p.x_stride, g, p.d_in, partial_a, dA, each_a, p.d_in, 1);
        if (want_b) add(dy, dy_stride, h, p.d_out, partial_b, dB, each_b, 1, p.rank);
        if (rows) {
            auto go = [&](auto kernel) { start(kernel, most, across, (p.rank + 63) / 64, 256, 0, both); };
            if (padded == 16) go(k_outer<T, 1>);
            else if (padded == 32) go(k_outer<T, 2>);
            else go(k_outer<T, 4>);
        }
        start(k_join<T>, ((long)p.rank * widest + 63) / 64, n, num, 256, 0, both);
    }
};

long workspace(const smx_adapted_linear* p, bool backward)
{
    // (as if nothing could be taken as it is: what the pointers' alignment says does not change the size)
    smx_adapted_linear q = *p;
    q.x = q.weight = reinterpret_cast<const void*>(2);
    Call c(q, nullptr, nullptr, true);
    with_type(p->type, [&](auto t) {
        using T = decltype(t);
        if (backward) c.backward<T>(reinterpret_cast<const T*>(2), q.d_out, nullptr, q.d_in, nullptr, nullptr);
        else if (p->rows > 0) c.forward<T>(nullptr, q.d_out);
    });
    return c.arena.used;
}
void check_workspace(const void* at, long bytes, long need)
{
    refuse_unless(need == 0 || (at && bytes >= need), "the workspace is smaller than smx_adapted_linear_workspace says");
    refuse_unless((reinterpret_cast<size_t>(at) & 255) == 0, "the workspace: an address that is a multiple of 256");
}

}  // namespace

}  // namespace smx

using namespace smx;

extern "C" int smx_adapted_linear_workspace(const smx_adapted_linear* p, int backward, long* bytes)
{
    return finetune_entry("smx_adapted_linear_workspace", [&] {
        check(p);
        refuse_unless(bytes, "bytes must not be null");
        *bytes = workspace(p, backward != 0);
    });
}

extern "C" int smx_adapted_linear_forward(const smx_adapted_linear* p, void* d_y, long y_stride, void* d_workspace, long workspace_bytes, void* stream)
{
    return finetune_entry("smx_adapted_linear_forward", [&] {
        check(p);
        if (p->rows == 0) return;
        refuse_unless(d_y && y_stride >= p->d_out, "y must not be null, its stride at least d_out");
        check_workspace(d_workspace, workspace_bytes, workspace(p, false));
        require_gfx950();
        Call c(*p, d_workspace, static_cast<hipStream_t>(stream), false);
        with_type(p->type, [&](auto t) { c.forward<decltype(t)>(static_cast<decltype(t)*>(d_y), y_stride); });
        hip_ok(hipGetLastError(), "launch");
    });
}

extern "C" int smx_adapted_linear_backward(const smx_adapted_linear* p, const void* d_dy, long dy_stride, void* d_dx, long dx_stride, void* d_dA, void* d_dB,
                                           void* d_workspace, long workspace_bytes, void* stream)
{
    return finetune_entry("smx_adapted_linear_backward", [&] {
        check(p);
        refuse_unless(p->rows == 0 || (d_dy && dy_stride >= p->d_out), "dy must not be null, its stride at least d_out");
        refuse_unless(!d_dx || dx_stride >= p->d_in, "the stride of dx: at least d_in");
        if (!d_dx && !d_dA && !d_dB) return;
        check_workspace(d_workspace, workspace_bytes, workspace(p, true));
        require_gfx950();
        Call c(*p, d_workspace, static_cast<hipStream_t>(stream), false);
        with_type(p->type, [&](auto t) {
            using T = decltype(t);
            c.backward<T>(static_cast<const T*>(d_dy), dy_stride, static_cast<T*>(d_dx), dx_stride, static_cast<T*>(d_dA), static_cast<T*>(d_dB));
        });
        hip_ok(hipGetLastError(), "launch");
    });
}
