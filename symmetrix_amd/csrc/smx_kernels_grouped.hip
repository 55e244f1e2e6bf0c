// A product with a matrix of the row's own group, and its gradient.
//
//   y_i = W_g x_i + b_g,   dx_i = W_g^T dy_i,   dW_g = sum over the group's rows of dy_i x_i^T,   db_g = sum of dy_i
//
// Rows are taken in the order of their groups, by way of the sorted order: nothing is copied into it, a tile's rows are fetched from
// where they are and its results stored where they belong.  A tile has rows of one group.  How many tiles a group has is known on the
// device alone, so a launch has as many blocks as there can be tiles, and every block finds its own from the groups' offsets.
//
// Bound by the matrix instructions but for few rows, which are bound by the weights' bytes.  16-bit types, whole pieces of 16 bytes (k_direct):
// straight from memory into LDS; 16 381 rows of 16 groups, 4 096 -> 2 048 in bfloat16, 286 us a call with the sort, 0.96 PFLOP/s (the kernel alone, slowed by
// a profiler, 320 to 340; groups of the same even size 1.0 PFLOP/s, a library's product of that size 1.3 to 1.5).  Single precision and any alignment (k_staged): by way of registers;
// gradient of 50 000 rows of 12 groups, 256 -> 512: dx and dW 91 us each, 144 TFLOP/s (8 192 rows, 2 048 x 2 048: 190 to 210; a library's
// product 146).
#include "smx_groups.hpp"

#include <cmath>
#include <limits>

namespace smx {

namespace {

enum { FORWARD = 0, ROWS = 1, WEIGHTS = 2 };      // y, dx and dW

// C(m, c) = sum over k of A(m, k) B(k, c)
//   FORWARD, ROWS: m is a row of the tile's group, A a row of x or dy; B the group's weights, in which k or c runs along rows.
//   WEIGHTS: k is a row of the group, A(m, k) its number m of dy and B(k, c) its number c of x.
struct Product {
    const void* a;
    long a_stride;
    const void* b;
    long b_each, b_stride;
    const void* bias;          // [group][cols] or null
    const int *order, *offsets;
    int groups, k, m, cols;    // k: of FORWARD and ROWS, m: of WEIGHTS
    long rows;
    void* out;
    long out_stride;
    int row_tiles, col_tiles;  // row_tiles: of WEIGHTS
    int piece;                 // of WEIGHTS: rows of a group that a block sums at most
    float* partial;            // sums of groups of more than one piece [slot][m][cols]
    void* sums;                // of WEIGHTS: db [group][m], or null
    float* partial_sums;       // its parts [slot][m]
};

// Where a block's rows are: [begin, end) of the sorted order, group `group`; slot: of a piece of WEIGHTS, or -1.
struct Place {
    int group, begin, end, slot;
};
// Items are cut from the groups in order, `high` rows each; with ALL a group without rows has one too, and the last two groups (rows
// without a group) have none.  Every block works out for itself where they are: of up to 62 groups every wavefront, a lane a group; of more
// the block, a thread some neighbouring groups (20 000 rows of 1 024 groups, 256 x 256 in bfloat16: 43 us; every wavefront 64 groups at a time: 98).
__device__ __forceinline__ int wave_inclusive(int x, int lane)
{
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int y = __shfl_up(x, d, 64);
        if (lane >= d) x += y;
    }
    return x;
}
template <bool ALL>
struct Items {
    const Product& p;
    const int high, lane;
    int first = 0, count = -1, n = 0;      // of the lane's group: where its rows begin, how many they are, and its items
    int until;                             // items up to the lane's, or thread's, last
    int slots_until;                       // and of groups of several
    int total;                             // all items
    __device__ __forceinline__ bool few() const { return p.groups + 2 <= 64; }
    __device__ __forceinline__ int rows_of(int g, int& begin) const
    {
        begin = p.offsets[min(g, p.groups + 1)];
        const int end = g >= p.groups + 1 ? (int)p.rows : p.offsets[min(g, p.groups) + 1];
        return g < p.groups + (ALL ? 0 : 2) ? end - begin : -1;
    }
    __device__ __forceinline__ int items_of(int rows) const { return rows < 0 ? 0 : max((rows + high - 1) / high, ALL ? 1 : 0); }
    __device__ __forceinline__ int per_thread() const { return (p.groups + 2 + (int)blockDim.x - 1) / (int)blockDim.x; }
    // (part: two numbers a wavefront)
    __device__ __forceinline__ Items(const Product& p_, int high_, int lane_, int (*part)[2]) : p(p_), high(high_), lane(lane_)
    {
        if (few()) {
            count = rows_of(lane, first);
            n = items_of(count);
            until = wave_inclusive(n, lane);
            slots_until = ALL ? wave_inclusive(n > 1 ? n : 0, lane) : 0;
            total = __builtin_amdgcn_readlane(until, 63);
            return;
        }
        int slots = 0;
        const int g0 = threadIdx.x * per_thread(), wave = threadIdx.x >> 6;
#pragma unroll 4
        for (int g = g0; g < g0 + per_thread(); ++g) {
            int begin;
            const int k = items_of(rows_of(g, begin));
            n += k;
            slots += ALL && k > 1 ? k : 0;
        }
        until = wave_inclusive(n, lane);
        slots_until = wave_inclusive(slots, lane);
        if (lane == 63) {
            part[wave][0] = until;
            part[wave][1] = slots_until;
        }
        __syncthreads();
        total = 0;
        int before = 0, slots_before = 0;
        for (int w = 0; w < (int)(blockDim.x >> 6); ++w) {
            before += w < wave ? part[w][0] : 0;
            slots_before += w < wave ? part[w][1] : 0;
            total += part[w][0];
        }
        until += before;
        slots_until += slots_before;
        total = __builtin_amdgcn_readfirstlane(total);
        count = slots;
    }
    __device__ __forceinline__ Place find(int item, Place* found) const
    {
        Place at{-1, 0, 0, -1};
        if (few()) {
            // Sums over rows: the groups with the most rows first, so that the last items are short.
            int group = lane, last = until;
            if (ALL) {
                int rank = 0;
#pragma unroll 8
                for (int h = 0; h < p.groups; ++h) {
                    const int other = __builtin_amdgcn_readlane(count, h);
                    rank += other > count || (other == count && h < lane) ? 1 : 0;
                }
                if (lane >= p.groups) rank = lane;
                group = __builtin_amdgcn_ds_permute(rank * 4, lane);
                last = wave_inclusive(__builtin_amdgcn_ds_permute(rank * 4, n), lane);
            }
            const unsigned long behind = __ballot(last > item);
            const int where = __builtin_ctzl(behind), from = __builtin_amdgcn_readlane(group, where), pieces = __builtin_amdgcn_readlane(n, from);
            const int mine = item - (__builtin_amdgcn_readlane(last, where) - pieces), begin = __builtin_amdgcn_readlane(first, from);
            at.group = from;
            at.begin = begin + mine * high;
            at.end = min(begin + __builtin_amdgcn_readlane(count, from), at.begin + high);
            if (ALL && pieces > 1) at.slot = __builtin_amdgcn_readlane(slots_until, from) - pieces + mine;
            return at;
        }
        if (item < until && item >= until - n) {      // (one thread's)
            int left = item - (until - n), slots = slots_until - count;
            for (int g = threadIdx.x * per_thread();; ++g) {
                int begin;
                const int rows = rows_of(g, begin), k = items_of(rows);
                if (left < k) {
                    at.group = g;
                    at.begin = begin + left * high;
                    at.end = min(begin + rows, at.begin + high);
                    if (ALL && k > 1) at.slot = slots + left;
                    break;
                }
                left -= k;
                slots += ALL && k > 1 ? k : 0;
            }
            *found = at;
        }
        __syncthreads();
        at = *found;
        return Place{__builtin_amdgcn_readfirstlane(at.group), __builtin_amdgcn_readfirstlane(at.begin), __builtin_amdgcn_readfirstlane(at.end),
                     __builtin_amdgcn_readfirstlane(at.slot)};
    }
};

// Tiles of a grid, four row tiles high, one below the other: neighbours share operands.
__device__ __forceinline__ void tile_at(int row_tiles, int col_tiles, int at, int& rt, int& ct)
{
    const int band = at / (4 * col_tiles), high = min(4, row_tiles - 4 * band), in_band = at - band * 4 * col_tiles;
    rt = band * 4 + in_band % high;
    ct = in_band / high;
}
// A block's place and its tile; `parts`: into how many the tile is cut, of which the block has number `part`; false: there is no tile
// for it.  The blocks of a die (every eighth) take neighbouring tiles, so that they share operands in its L2.
// With CUT, of tiles that run one on a CU, those of the last round are cut where they are few: all others are done when they begin.
constexpr int kCUs = 256;
template <int MODE, bool CUT>
__device__ __forceinline__ bool find_tile(const Product& p, int high, int lane, Place& at, int& rt, int& ct, int& parts, int& part)
{
    __shared__ int sums[8][2];
    __shared__ Place found;
    parts = 1;
    part = 0;
    const Items<MODE == WEIGHTS> items(p, MODE == WEIGHTS ? p.piece : high, lane, sums);
    if constexpr (MODE == WEIGHTS) {
        // (items take different times: every die has a share of each)
        const int tiles = p.row_tiles * p.col_tiles, share = (tiles + 7) / 8;
        int item, tile;
        if (tiles >= 8) {
            item = (int)(blockIdx.x / 8) / share;
            tile = blockIdx.x % 8 * share + (int)(blockIdx.x / 8) % share;
            if (tile >= tiles) return false;
        } else {
            item = blockIdx.x / tiles;
            tile = blockIdx.x % tiles;
        }
        if (item >= items.total) return false;
        at = items.find(item, &found);
        tile_at(p.row_tiles, p.col_tiles, tile, rt, ct);
    } else {
        const int row_tiles = items.total, tiles = row_tiles * p.col_tiles;
        const int rest = CUT ? tiles % kCUs : 0, full = CUT ? tiles - rest : tiles;
        int block = blockIdx.x, count = full, first = 0;
        if (CUT && block >= full) {
            parts = rest <= kCUs / 4 ? 4 : rest <= kCUs / 2 ? 2 : 1;
            block -= full;
            first = full;
            count = rest * parts;
        }
        const int per = (count + 7) / 8, id = block % 8 * per + block / 8;
        if (id >= count || block / 8 >= per) return false;
        part = id % parts;
        tile_at(row_tiles, p.col_tiles, first + id / parts, rt, ct);
        at = items.find(rt, &found);
    }
    return true;
}

// What rows without a group have for results: eight numbers a thread, rows and columns at once.
template <typename T>
__device__ __forceinline__ void store_none(const Product& p, const Place& at, int col0, int wide)
{
    const float v = at.group == p.groups ? 0.0f : std::numeric_limits<float>::quiet_NaN();
    const float eight[8] = {v, v, v, v, v, v, v, v};
    const int pieces = wide / 8, all = (at.end - at.begin) * pieces;
#pragma unroll 4
    for (int e = threadIdx.x; e < all; e += blockDim.x) {
        const int row = p.order[at.begin + e / pieces], col = col0 + e % pieces * 8;
        if (col < p.cols) store_run<8>(static_cast<T*>(p.out) + row * p.out_stride + col, p.cols - col, eight);
    }
}

// Lane (n, g) holds of tile (i, t) row 16 i + n and columns 16 t + 4 g + 0..3.  What is stored goes by way of other lanes, so that four
// neighbouring lanes have 64 neighbouring bytes.
// row(i): where row 16 i + lane / 4 of the tile goes, or null; left: columns from the tile's first on that there are.
template <typename T, int NM, int NT, typename Row>
__device__ __forceinline__ void store_tiles(int lane, const f32x4 (&acc)[NM][NT], int left, Row&& row)
{
#pragma unroll
    for (int i = 0; i < NM; ++i) {
        T* out = row(i);
        if constexpr (std::is_same_v<T, float>) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const f32x4 v = from_operand(acc[i][t], lane);
                const int col = 16 * t + 4 * (lane & 3);
                const float u[4] = {v[0], v[1], v[2], v[3]};
                if (out) store_run<4>(out + col, left - col, u);
            }
        } else {
            typedef int i32x4 __attribute__((ext_vector_type(4)));
            const bool odd = lane >> 4 & 1;
            // (lane group g has, after it has exchanged four numbers with its neighbour, eight from 16 (g % 2) + 8 (g / 2) on)
            const int from = (16 * ((lane & 1) * 2 + (lane >> 1 & 1)) + (lane >> 2)) * 4;
#pragma unroll
            for (int t = 0; t < NT; t += 2) {
                typename Run<T, 8>::type v;
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = (T)acc[i][t + j / 4][j % 4];
                i32x4 d = __builtin_bit_cast(i32x4, v);
                const int give[2] = {odd ? d[0] : d[2], odd ? d[1] : d[3]};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int got = __shfl_xor(give[h], 16, 64);
                    d[h] = odd ? got : d[h];
                    d[2 + h] = odd ? d[2 + h] : got;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) d[j] = __builtin_amdgcn_ds_bpermute(from, d[j]);
                v = __builtin_bit_cast(typename Run<T, 8>::type, d);
                const int col = 16 * t + 8 * (lane & 3);
                if (!out) continue;
                if (left - col >= 8) *reinterpret_cast<typename Run<T, 8>::loose*>(out + col) = v;
                else {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (col + j < left) out[col + j] = v[j];
                }
            }
        }
    }
}

// Bias, and where the results go: what follows the sums of all modes.  row0, col0: the wavefront's first in the tile's place; rows: the
// tile's, in LDS.
template <typename T, int MODE, int NM, int NT>
__device__ __forceinline__ void finish(const Product& p, const Place& at, int lane, int row0, int col0, const int* rows, f32x4 (&acc)[NM][NT])
{
    if constexpr (MODE == WEIGHTS) {
        if (at.slot >= 0) {
            float* base = p.partial + (long)at.slot * p.m * p.cols + col0;
            store_tiles<float>(lane, acc, p.cols - col0, [&](int i) {
                const int m = row0 + 16 * i + lane / 4;
                return m < p.m ? base + (long)m * p.cols : nullptr;
            });
        } else {
            T* base = static_cast<T*>(p.out) + (long)at.group * p.m * p.cols + col0;
            store_tiles<T>(lane, acc, p.cols - col0, [&](int i) {
                const int m = row0 + 16 * i + lane / 4;
                return m < p.m ? base + (long)m * p.cols : nullptr;
            });
        }
    } else {
        if (MODE == FORWARD && p.bias) {
            const T* bias = static_cast<const T*>(p.bias) + (long)at.group * p.cols;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int col = col0 + 16 * t + 4 * (lane >> 4);
                float b[4];
                load_run<4>(bias + col, p.cols - col, b);
#pragma unroll
                for (int i = 0; i < NM; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][t][j] += b[j];
            }
        }
        store_tiles<T>(lane, acc, p.cols - col0, [&](int i) {
            const int r = row0 + 16 * i + lane / 4;
            return r < at.end - at.begin ? static_cast<T*>(p.out) + rows[r] * p.out_stride + col0 : nullptr;
        });
    }
}

template <typename T>
__device__ __forceinline__ void store_sum(const Product& p, const Place& at, int m, float sum)      // of db
{
    if (at.slot >= 0) p.partial_sums[(long)at.slot * p.m + m] = sum;
    else static_cast<T*>(p.sums)[(long)at.group * p.m + m] = (T)sum;
}

// ---- operands in LDS
//
// Steps of K terms (64 for 16-bit types as they are, 32 for single precision in parts); an operand has `wide` rows or columns of C.  It lies
//   along: where its terms are neighbours in memory: [wide][K], the 16-byte pieces of a row in an order that depends on the row;
//   across: where neighbours in memory are neighbours in C: [K][wide], 32-byte pieces in an order that depends on the term; lanes get it
//   turned by the instruction that reads it.
// The orders are for the banks: lanes that read together meet different ones.
template <int K>
__device__ __forceinline__ int along_piece(int row, int piece) { return K == 64 ? piece ^ (row & 7) : piece ^ (row >> 1 & 3); }
template <int WIDE>
__device__ __forceinline__ int across_turn(int k) { return WIDE >= 128 ? (k & 3) | (k >> 3 & 1) << 2 : (k >> 1 & 1) | (k >> 3 & 1) << 1; }

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
// What a wavefront reads of an operand: 16 rows or columns from 16 `tile` on, 32 terms from 32 h on.
template <typename F, int K, int WIDE, bool ACROSS>
struct Reader {
    unsigned at;      // of tile 0 and h 0
    __device__ __forceinline__ Reader(unsigned base, int tile0, int lane)
    {
        const int n = lane & 15, g = lane >> 4;
        if constexpr (ACROSS) at = base + (8 * g + n / 4) * (2 * WIDE) + ((tile0 ^ across_turn<WIDE>(8 * g + n / 4)) << 5) + 8 * (n & 3);
        else at = base + (16 * tile0 + n) * (2 * K) + 16 * along_piece<K>(n, g);
    }
    // (tile 0 and step 0 of 16-byte pieces: a tile is 16 rows further, which along_piece does not see; h turns a bit of the piece)
    __device__ __forceinline__ F get(int tile, int h, unsigned more) const
    {
        if constexpr (ACROSS) {
            const unsigned a = (at ^ (unsigned)tile << 5) + more + h * 32 * (2 * WIDE);
            const s16x4 u = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)a), v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(a + 4 * 2 * WIDE));
            return __builtin_bit_cast(F, __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            return *(const __attribute__((address_space(3))) F*)((at ^ h << 6) + more + tile * 16 * (2 * K));
        }
    }
};

// 1 KB of a wavefront from global memory into LDS as load_into_lds brings it, every lane from an address of its own.
__device__ __forceinline__ void load_into_lds_from(const void* from, unsigned to)
{
    unsigned m0;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0) : "v"(from), "s"(to) : "memory");
}
// 4 bytes of every lane, from base + offset, to `to` + 4 lane
__device__ __forceinline__ void load_words_into_lds(const void* base, unsigned offset, unsigned to)
{
    unsigned m0;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0) : "v"(offset), "s"(base), "s"(to) : "memory");
}
__device__ const uint4 kZeros = {0, 0, 0, 0};      // what is fetched for terms that do not exist

// 16-bit types whose rows begin at multiples of 16 bytes: straight from memory into LDS, STAGES steps of 64 terms under way.
// WM x WN wavefronts share the tile.  32 terms have their operands fetched during the 32 before.
template <typename T, int MODE, int BM, int BN, int WM, int WN, int STAGES>
__device__ __forceinline__ void direct_tile(const Product& p, const Place& at, int row0, int col0, unsigned char* lds)
{
    constexpr int WAVES = WM * WN, NM = BM / WM / 16, NT = BN / WN / 16, PA = BM / 8 / WAVES, PB = BN / 8 / WAVES, PER = PA + PB, STAGE = (BM + BN) * 128;
    constexpr bool A_ACROSS = MODE == WEIGHTS, B_ACROSS = MODE != FORWARD;
    static_assert(BM / 8 % WAVES == 0 && BN / 8 % WAVES == 0, "loads of a wavefront");
    typedef typename Operand<T>::type frag;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), count = at.end - at.begin;
    const int terms = MODE == WEIGHTS ? count : p.k, stages = (terms + 63) / 64;
    // What a lane asks for, in bytes from a base that moves from step to step: 16 bytes at a time, PA + PB times.
    constexpr int A_PIECES = BM / 8, B_PIECES = BN / 8;      // of a term, where it lies across
    const int* order = p.order + at.begin;
    unsigned from_a[PA], from_b[PB];
#pragma unroll
    for (int u = 0; u < PA; ++u) {
        const int slot = (wave * PA + u) * 64 + lane;      // 16 bytes of the operand in LDS
        if constexpr (A_ACROSS) {
            const int k = slot / A_PIECES, piece = slot % A_PIECES ^ across_turn<BM>(k) << 1;
            from_a[u] = 2 * min(row0 + 8 * piece, p.m - 8);
        } else {
            const int r = slot / 8;
            from_a[u] = (unsigned)(order[min(r, count - 1)] * p.a_stride * 2) + 16 * along_piece<64>(r, slot % 8);
        }
    }
    const char* b_base = static_cast<const char*>(p.b) + (MODE == WEIGHTS ? 0 : 2 * (at.group * p.b_each + (MODE == FORWARD ? col0 * p.b_stride : 0)));
#pragma unroll
    for (int u = 0; u < PB; ++u) {
        const int slot = (wave * PB + u) * 64 + lane;
        if constexpr (B_ACROSS) {
            const int k = slot / B_PIECES, piece = slot % B_PIECES ^ across_turn<BN>(k) << 1;
            from_b[u] = (MODE == ROWS ? (unsigned)(2 * k * p.b_stride) : 0) + 2 * min(col0 + 8 * piece, p.cols - 8);
        } else {
            const int r = slot / 8;
            from_b[u] = (unsigned)(2 * min(r, p.cols - 1 - col0) * p.b_stride) + 16 * along_piece<64>(r, slot % 8);
        }
    }
    const unsigned lds0 = lds_address(lds);
    int* const tile_rows = reinterpret_cast<int*>(lds + STAGES * STAGE);      // (for the results; there at the first barrier)
    if (MODE != WEIGHTS)
        for (int i = threadIdx.x; i < count; i += 64 * WAVES) tile_rows[i] = order[i];
    // Of WEIGHTS: which rows the terms of the next steps are, sixteen steps' in LDS behind the tiles.  They are asked for AHEAD steps before
    // they are needed, in front of that step's tiles: AHEAD (and no fewer) steps' tiles later, a wait for all but the youngest STAGES - 2 steps'
    // has waited for them too, and a barrier shows them to the other wavefronts.
    constexpr int AHEAD = STAGES > 3 ? STAGES - 2 : 1;
    const unsigned rows0 = lds0 + STAGES * STAGE;
    auto look_up = [&](int s) {
        if (MODE == WEIGHTS && wave == s % WAVES) load_words_into_lds(order, 4 * min(64 * s + lane, terms - 1), rows0 + s % 16 * 256);
    };
    static_assert(MODE != WEIGHTS || PA == PB, "one row for both operands");
    auto rows_of = [&](int s, unsigned (&row)[PA]) {      // of a lane's terms
        if constexpr (MODE == WEIGHTS) {
#pragma unroll
            for (int u = 0; u < PA; ++u)
                row[u] = *(const __attribute__((address_space(3))) unsigned*)(rows0 + s % 16 * 256 + ((wave * PA + u) * 64 + lane) / A_PIECES * 4);
        }
    };
    const unsigned a_row = (unsigned)p.a_stride * 2, b_row = (unsigned)p.b_stride * 2;
    auto request = [&](int s) {
        const unsigned to = lds0 + s % STAGES * STAGE;
        const char* a = static_cast<const char*>(p.a) + (A_ACROSS ? 0 : (long)s * 128);
        const char* b = b_base + (MODE == FORWARD ? (long)s * 128 : MODE == ROWS ? (long)s * 128 * p.b_stride : 0);
        unsigned row[PA];
        rows_of(s, row);
#pragma unroll
        for (int u = 0; u < PA; ++u) load_into_lds(a, from_a[u] + (A_ACROSS ? row[u] * a_row : 0), to + (wave * PA + u) * 1024);
#pragma unroll
        for (int u = 0; u < PB; ++u) load_into_lds(b, from_b[u] + (MODE == WEIGHTS ? row[u % PA] * b_row : 0), to + BM * 128 + (wave * PB + u) * 1024);
    };
    auto request_last = [&](int s) {      // of a step that need not be whole
        if (64 * s + 64 <= terms) return request(s);
        const unsigned to = lds0 + s % STAGES * STAGE;
        const char* a = static_cast<const char*>(p.a) + (A_ACROSS ? 0 : (long)s * 128);
        const char* b = b_base + (MODE == FORWARD ? (long)s * 128 : MODE == ROWS ? (long)s * 128 * p.b_stride : 0);
        unsigned row[PA];
        rows_of(s, row);
#pragma unroll
        for (int u = 0; u < PA; ++u) {
            const int slot = (wave * PA + u) * 64 + lane, k = 64 * s + (A_ACROSS ? slot / A_PIECES : 8 * along_piece<64>(slot / 8, slot % 8));
            const char* from = a + (from_a[u] + (A_ACROSS ? row[u] * a_row : 0));
            load_into_lds_from(k < terms ? from : reinterpret_cast<const char*>(&kZeros), to + (wave * PA + u) * 1024);
        }
#pragma unroll
        for (int u = 0; u < PB; ++u) {
            const int slot = (wave * PB + u) * 64 + lane, k = 64 * s + (B_ACROSS ? slot / B_PIECES : 8 * along_piece<64>(slot / 8, slot % 8));
            const char* from = b + (from_b[u] + (MODE == WEIGHTS ? row[u % PA] * b_row : 0));
            load_into_lds_from(k < terms ? from : reinterpret_cast<const char*>(&kZeros), to + BM * 128 + (wave * PB + u) * 1024);
        }
    };
    f32x4 acc[NM][NT];
#pragma unroll
    for (int i = 0; i < NM; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[i][t] = f32x4{0, 0, 0, 0};
    const int wm = wave / WN, wn = wave % WN;
    const Reader<frag, 64, BM, A_ACROSS> read_a(lds0, wm * NM, lane);
    const Reader<frag, 64, BN, B_ACROSS> read_b(lds0 + BM * 128, wn * NT, lane);
    struct Frags {
        frag x[NM], w[NT];
    };
    auto fetch = [&](int s, int h, Frags& f) {
        const unsigned more = s % STAGES * STAGE;
#pragma unroll
        for (int t = 0; t < NT; ++t) f.w[t] = read_b.get(t, h, more);
#pragma unroll
        for (int i = 0; i < NM; ++i) f.x[i] = read_a.get(i, h, more);
    };
    auto sums = [&](const Frags& now) {
#pragma unroll
        for (int i = 0; i < NM; ++i)
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[i][t] = mma(now.w[t], now.x[i], acc[i][t]);
    };
    // db: the sums of dy alone, as one column more whose numbers are ones, of the first column of tiles; the wavefronts that have the same rows
    // of A share them.  (Of small tiles: 12 731 rows, 192 -> 224, 47 groups in bfloat16: 28 us with a launch for db, 16.  Larger ones have no registers
    // for it: 16 384 rows, 4 096 -> 2 048: 305 us without, 532.)
    constexpr bool SUMS = MODE == WEIGHTS && BM == 64;
    constexpr int OWN = NM / WN;
    const bool with_sums = SUMS && p.sums && col0 == 0;
    f32x4 ones_acc[SUMS ? OWN : 1];
#pragma unroll
    for (int o = 0; o < (SUMS ? OWN : 1); ++o) ones_acc[o] = f32x4{0, 0, 0, 0};
    auto add_sums = [&](const Frags& now) {
        if constexpr (SUMS) {
            if (!with_sums) return;
            frag ones;
#pragma unroll
            for (int j = 0; j < 8; ++j) ones[j] = (T)1.0f;
#pragma unroll
            for (int w = 0; w < WN; ++w)
                if (wn == w)
#pragma unroll
                    for (int o = 0; o < OWN; ++o) ones_acc[o] = mma(ones, now.x[w * OWN + o], ones_acc[o]);
        }
    };
    auto woven = [&] {      // sums and the fetches beside them, by turns
        constexpr int READS = NM * (A_ACROSS ? 2 : 1) + NT * (B_ACROSS ? 2 : 1), EACH = NM * NT / READS;
        if constexpr (EACH >= 1) {
#pragma unroll
            for (int i = 0; i < READS; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x008, NM * NT - EACH * READS, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    // (a wavefront without rows takes part in the loads alone, and leaves the matrix cores to the others)
    const bool idle = MODE != WEIGHTS && wm * NM * 16 >= count;
    if (stages > 0) {
        if constexpr (MODE == WEIGHTS) {
            static_assert(STAGES + AHEAD < 16, "rows of sixteen steps");
            for (int i = threadIdx.x; i < (STAGES + AHEAD) * 64; i += 64 * WAVES) *(__attribute__((address_space(3))) int*)(rows0 + 4 * i) = order[min(i, terms - 1)];
            __syncthreads();
        }
#pragma unroll
        for (int s = 0; s < STAGES; ++s)
            if (s < stages) request_last(s);
        if (STAGES <= stages) wait_loads<(STAGES - 1) * PER>();
        else wait_loads<0>();
        barrier_only();
        int s = 0;
        if (idle) {
#pragma unroll 1
            for (; s + STAGES + 1 < stages; ++s) {
                wait_loads<(STAGES - 2) * PER>();
                barrier_only();
                request(s + STAGES);
            }
#pragma unroll 1
            for (; s + 1 < stages; ++s) {
                wait_loads<0>();
                barrier_only();
                if (s + STAGES < stages) request_last(s + STAGES);
            }
            return;
        }
        Frags f[2];
        fetch(0, 0, f[0]);
#pragma unroll 1
        for (; s + STAGES + 1 < stages; ++s) {
            fetch(s, 1, f[1]);
            sums(f[0]);
            woven();
            add_sums(f[0]);
            wait_loads<(STAGES - 2) * PER>();
            barrier_only();      // the next tiles are there, and everybody has read these
            look_up(s + STAGES + AHEAD);
            request(s + STAGES);
            fetch(s + 1, 0, f[0]);
            sums(f[1]);
            woven();
            add_sums(f[1]);
        }
#pragma unroll 1
        for (; s < stages; ++s) {      // the last request, and none
            fetch(s, 1, f[1]);
            sums(f[0]);
            add_sums(f[0]);
            if (s + 1 < stages) {
                wait_loads<0>();
                barrier_only();
                if (s + STAGES < stages) request_last(s + STAGES);
                fetch(s + 1, 0, f[0]);
            }
            sums(f[1]);
            add_sums(f[1]);
        }
    }
    if (SUMS && with_sums && lane < 16)
#pragma unroll
        for (int o = 0; o < OWN; ++o) {
            const int m = row0 + (wm * NM + wn * OWN + o) * 16 + lane;
            if (m < p.m) store_sum<T>(p, at, m, ones_acc[SUMS ? o : 0][0]);
        }
    finish<T, MODE, NM, NT>(p, at, lane, row0 + wm * NM * 16, col0 + wn * NT * 16, tile_rows, acc);
}

// LARGE: 256 x 256 by eight wavefronts, one block on a CU, those of the last round cut in two or four (16 381 rows as above: 345 us uncut).
// Gradient of 8 179 rows of 8 groups, 2 048 x 2 048 in float16: dx 78 us, dW 74.  (dx's takes all 256 registers and keeps one more in memory, which the last
// steps of a tile alone read; dW's tiles are not cut.)
template <typename T, int MODE, bool LARGE, int BM, int STAGES>
__global__ __launch_bounds__(LARGE ? 512 : 256, 2) void k_direct(const Product p)
{
    static_assert(!LARGE || BM == 256, "tiles");
    extern __shared__ __align__(1024) unsigned char lds[];
    const int lane = threadIdx.x & 63;
    Place at;
    int rt, ct, parts, part;
    if (!find_tile<MODE, LARGE>(p, BM, lane, at, rt, ct, parts, part)) return;
    if (MODE != WEIGHTS && at.group >= p.groups) {
        if (part == 0) store_none<T>(p, at, ct * BM, BM);
        return;
    }
    const int row0 = MODE == WEIGHTS ? rt * BM : 0;
    if constexpr (LARGE && MODE != WEIGHTS) {
        if (parts > 1) {
            const int col0 = ct * BM + part / (parts / 2) * (BM / 2);
            if (col0 >= p.cols) return;
            if (parts == 2) {
                direct_tile<T, MODE, 256, 128, 4, 2, 2>(p, at, 0, col0, lds);
            } else {
                at.begin += part % 2 * (BM / 2);
                at.end = min(at.end, at.begin + BM / 2);
                if (at.begin < at.end) direct_tile<T, MODE, 128, 128, 2, 4, 4>(p, at, 0, col0, lds);
            }
            return;
        }
    }
    if constexpr (LARGE) direct_tile<T, MODE, 256, 256, 2, 4, STAGES>(p, at, row0, ct * BM, lds);
    else direct_tile<T, MODE, BM, BM, 2, 2, STAGES>(p, at, row0, ct * BM, lds);
}

// ---- operands by way of registers: any alignment, and single precision, which is brought to bf16 parts on the way

// Both operands of single precision in three bf16 parts, exactly, of whose products the six largest are formed (what is left out is below
// 1.002 2^-24 of a product), small ones first.  Numbers are brought up by 2^24 first, so that the parts of small ones are normal numbers.  Numbers from
// 2^104 on and sums from 2^80 on do not fit then (db: from 2^104 on); what they make infinite or NaN is formed again, as sums that are not finite are, in twenty
// times the time (8 192 rows, 2 048 x 2 048: 0.33 ms, 7.4).
constexpr float kSplitScale = 16777216.0f;
__device__ __forceinline__ void parts_of(const float (&x)[8], bf16x8 (&part)[3])
{
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        f32x2 rest = {x[j] * kSplitScale, x[j + 1] * kSplitScale};
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            const bf16x2 h = __builtin_convertvector(rest, bf16x2);
            part[q][j] = h[0];
            part[q][j + 1] = h[1];
            if (q < 2) rest -= __builtin_convertvector(h, f32x2);
        }
    }
}
// eight neighbours in memory on their way
template <typename T>
struct Eight {
    typename Operand<T>::type v[8 / kRun<T>];
    // from p on, all of which exist
    __device__ __forceinline__ void load(const T* p)
    {
#pragma unroll
        for (int h = 0; h < 8 / kRun<T>; ++h) v[h] = *reinterpret_cast<const typename Run<T, kRun<T>>::loose*>(p + h * kRun<T>);
    }
    // of which `left` exist; zeros for the others
    __device__ __forceinline__ void load(const T* p, int left)
    {
#pragma unroll
        for (int h = 0; h < 8 / kRun<T>; ++h) v[h] = load_operand(p + h * kRun<T>, left - h * kRun<T>);
    }
};

// Sums of a tile of 16 x 16 in single precision, on its own instructions: row m0 + n and columns c0 + 4 g + 0..3 of lane (n, g).
template <typename T, int MODE>
__device__ __forceinline__ f32x4 plain_sums(const Product& p, const Place& at, int lane, int m0, int c0)
{
    const T *a = static_cast<const T*>(p.a), *b = static_cast<const T*>(p.b);
    const int n = lane & 15, g = lane >> 4, count = at.end - at.begin, terms = MODE == WEIGHTS ? count : p.k;
    const int m = min(m0 + n, (MODE == WEIGHTS ? p.m : count) - 1), c = min(c0 + n, p.cols - 1);
    if (MODE != WEIGHTS) {
        a += p.order[at.begin + m] * p.a_stride;
        b += at.group * p.b_each + (MODE == FORWARD ? c * p.b_stride : c);
    }
    f32x4 sum{0, 0, 0, 0};
#pragma unroll 4
    for (int k0 = 0; k0 < terms; k0 += 4) {
        const int k = k0 + g;
        float u = 0.0f, v = 0.0f;
        if (k < terms) {
            const long row = MODE == WEIGHTS ? p.order[at.begin + k] : k;
            u = (float)(MODE == WEIGHTS ? a[row * p.a_stride + m] : a[k]);
            v = (float)(MODE == FORWARD ? b[k] : MODE == ROWS ? b[row * p.b_stride] : b[row * p.b_stride + c]);
        }
        sum = __builtin_amdgcn_mfma_f32_16x16x4f32(v, u, sum, 0, 0, 0);
    }
    return sum;
}

// Steps of 32 terms, or of 64 where a step's sums are short (in 16 bits; not of WEIGHTS, whose registers they would take); those of the next AHEAD
// are on their way to registers during the sums of one.  Four wavefronts, 2 x 2.  3 000 rows of 10 groups, 256 -> 512 in single precision, in tiles of
// 64: 14 us, most of it the first loads' and the last stores' latency; odd widths in 16 bits: 16 384 rows of 16 groups, 2 049 -> 4 097, 0.5 PFLOP/s.
template <typename T, int MODE, int BM, int BN, int AHEAD>
__global__ __launch_bounds__(256, 2) void k_staged(const Product p)
{
    constexpr bool SINGLE = std::is_same_v<T, float>, A_ACROSS = MODE == WEIGHTS, B_ACROSS = MODE != FORWARD;
    constexpr int PARTS = SINGLE ? 3 : 1, STEP = SINGLE || MODE == WEIGHTS ? 32 : 64, PIECES = STEP / 8, NM = BM / 32, NT = BN / 32, PA = BM * PIECES / 256, PB = BN * PIECES / 256;
    constexpr int A_PART = BM * STEP * 2, B_PART = BN * STEP * 2;
    typedef typename std::conditional_t<SINGLE, Operand<bf16>, Operand<T>>::type frag;
    __shared__ __align__(1024) unsigned char lds[PARTS * (A_PART + B_PART)];
    // The tile's rows; or of WEIGHTS the rows of the terms of two times kLook steps, in LDS: a wait for a row's number from memory would be one for all that is on its way.
    constexpr int kLook = 16;
    __shared__ int look[MODE == WEIGHTS ? 2 * kLook * STEP : BM];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Place at;
    int rt, ct, parts, part;
    if (!find_tile<MODE, false>(p, BM, lane, at, rt, ct, parts, part)) return;
    const int col0 = ct * BN, row0 = MODE == WEIGHTS ? rt * BM : 0, count = at.end - at.begin;
    if (MODE != WEIGHTS && at.group >= p.groups) {
        store_none<T>(p, at, col0, BN);
        return;
    }
    const int terms = MODE == WEIGHTS ? count : p.k, steps = (terms + STEP - 1) / STEP;
    const int* order = p.order + at.begin;
    if (MODE != WEIGHTS)      // (for the results; there at the first barrier)
        for (int i = threadIdx.x; i < count; i += 256) look[i] = order[i];
    // where a thread's numbers begin and how many of the eight there are; along: k is added
    const T* from_a[PA];
    const T* from_b[PB];
    int a_left[PA], b_left[PB];
#pragma unroll
    for (int u = 0; u < PA; ++u) {
        const int slot = u * 256 + threadIdx.x;
        if constexpr (A_ACROSS) {
            const int m = row0 + slot % (BM / 8) * 8;
            a_left[u] = p.m - m;
            from_a[u] = static_cast<const T*>(p.a) + min(m, p.m - 1);
        } else from_a[u] = static_cast<const T*>(p.a) + order[min(slot / PIECES, count - 1)] * p.a_stride + slot % PIECES * 8;
    }
#pragma unroll
    for (int u = 0; u < PB; ++u) {
        const int slot = u * 256 + threadIdx.x;
        const T* b = static_cast<const T*>(p.b) + (MODE == WEIGHTS ? 0 : at.group * p.b_each);
        if constexpr (B_ACROSS) {
            const int c = col0 + slot % (BN / 8) * 8;
            b_left[u] = p.cols - c;
            from_b[u] = b + min(c, p.cols - 1);
        } else from_b[u] = b + min(col0 + slot / PIECES, p.cols - 1) * p.b_stride + slot % PIECES * 8;
    }
    auto look_up = [&](int block) {      // of kLook steps
        if constexpr (MODE == WEIGHTS)
            for (int i = threadIdx.x; i < kLook * STEP; i += 256) look[block % 2 * kLook * STEP + i] = order[min(block * kLook * STEP + i, terms - 1)];
    };
    Eight<T> raw[AHEAD][PA + PB];
    auto term = [&](int s, int u, int wide) { return STEP * s + (u * 256 + (int)threadIdx.x) / (wide / 8); };
    auto row_of = [&](int k) { return look[k % (2 * kLook * STEP)]; };
    // Of a step all numbers of which exist, without a branch; and of any.
    auto request_whole = [&](int s, Eight<T> (&to)[PA + PB]) {
#pragma unroll
        for (int u = 0; u < PA; ++u) to[u].load(from_a[u] + (A_ACROSS ? row_of(term(s, u, BM)) * p.a_stride : STEP * s));
#pragma unroll
        for (int u = 0; u < PB; ++u) {
            const int k = term(s, u, BN);
            to[PA + u].load(from_b[u] + (MODE == WEIGHTS ? row_of(k) * p.b_stride : B_ACROSS ? k * p.b_stride : STEP * s));
        }
        asm volatile("" ::: "memory");      // (asked for here, not where they are used)
    };
    auto request = [&](int s, Eight<T> (&to)[PA + PB]) {
#pragma unroll
        for (int u = 0; u < PA; ++u) {
            const int k = term(s, u, BM);
            if constexpr (A_ACROSS) to[u].load(from_a[u] + row_of(k) * p.a_stride, k < terms ? a_left[u] : 0);
            else to[u].load(from_a[u] + STEP * s, terms - STEP * s - (int)threadIdx.x % PIECES * 8);
        }
#pragma unroll
        for (int u = 0; u < PB; ++u) {
            const int k = term(s, u, BN);
            if constexpr (B_ACROSS) to[PA + u].load(from_b[u] + (MODE == WEIGHTS ? (long)row_of(k) : min(k, terms - 1)) * p.b_stride, k < terms ? b_left[u] : 0);
            else to[PA + u].load(from_b[u] + STEP * s, terms - STEP * s - (int)threadIdx.x % PIECES * 8);
        }
    };
    auto put = [&](const Eight<T>& x, unsigned char* to, int part_bytes) {
        if constexpr (SINGLE) {
            const float v[8] = {x.v[0][0], x.v[0][1], x.v[0][2], x.v[0][3], x.v[1][0], x.v[1][1], x.v[1][2], x.v[1][3]};
            bf16x8 part[3];
            parts_of(v, part);
#pragma unroll
            for (int q = 0; q < 3; ++q) *reinterpret_cast<bf16x8*>(to + q * part_bytes) = part[q];
        } else *reinterpret_cast<frag*>(to) = x.v[0];
    };
    auto store = [&](const Eight<T> (&raw)[PA + PB]) {
#pragma unroll
        for (int u = 0; u < PA; ++u) {
            const int slot = u * 256 + threadIdx.x, k = slot / (BM / 8);
            put(raw[u], lds + (A_ACROSS ? k * (2 * BM) + 16 * (slot % (BM / 8) ^ across_turn<BM>(k) << 1) : slot / PIECES * (2 * STEP) + 16 * along_piece<STEP>(slot / PIECES, slot % PIECES)), A_PART);
        }
#pragma unroll
        for (int u = 0; u < PB; ++u) {
            const int slot = u * 256 + threadIdx.x, k = slot / (BN / 8);
            put(raw[PA + u], lds + PARTS * A_PART + (B_ACROSS ? k * (2 * BN) + 16 * (slot % (BN / 8) ^ across_turn<BN>(k) << 1) : slot / PIECES * (2 * STEP) + 16 * along_piece<STEP>(slot / PIECES, slot % PIECES)),
                B_PART);
        }
    };
    f32x4 acc[NM][NT];
#pragma unroll
    for (int i = 0; i < NM; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[i][t] = f32x4{0, 0, 0, 0};
    const int wm = wave / 2, wn = wave % 2;
    // db: the sums of dy alone, as one column more whose numbers are ones, of the first column of tiles
    constexpr bool SUMS = MODE == WEIGHTS;
    const bool with_sums = SUMS && p.sums && ct == 0 && wn == 0;
    f32x4 ones_acc[SUMS ? NM : 1];
    frag ones;
#pragma unroll
    for (int j = 0; j < 8; ++j) ones[j] = 1.0f;
#pragma unroll
    for (int i = 0; i < (SUMS ? NM : 1); ++i) ones_acc[i] = f32x4{0, 0, 0, 0};
    const unsigned lds0 = lds_address(lds);
    const Reader<frag, STEP, BM, A_ACROSS> read_a(lds0, wm * NM, lane);
    const Reader<frag, STEP, BN, B_ACROSS> read_b(lds0 + PARTS * A_PART, wn * NT, lane);
    auto sums = [&] {
#pragma unroll
        for (int h = 0; h < STEP / 32; ++h) {
            frag x[NM][PARTS];
#pragma unroll
            for (int i = 0; i < NM; ++i)
#pragma unroll
                for (int q = 0; q < PARTS; ++q) x[i][q] = read_a.get(i, h, q * A_PART);
            if (SUMS && with_sums) {
#pragma unroll
                for (int q = PARTS - 1; q >= 0; --q)
#pragma unroll
                    for (int i = 0; i < NM; ++i) ones_acc[SUMS ? i : 0] = mma(ones, x[i][q], ones_acc[SUMS ? i : 0]);
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                frag w[PARTS];
#pragma unroll
                for (int q = 0; q < PARTS; ++q) w[q] = read_b.get(t, h, q * B_PART);
                if constexpr (SINGLE) {
                    constexpr int ix[6] = {2, 0, 1, 1, 0, 0}, iw[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
                    for (int o = 0; o < 6; ++o)
#pragma unroll
                        for (int i = 0; i < NM; ++i) acc[i][t] = mma(w[iw[o]], x[i][ix[o]], acc[i][t]);
                } else {
#pragma unroll
                    for (int i = 0; i < NM; ++i) acc[i][t] = mma(w[0], x[i][0], acc[i][t]);
                }
            }
        }
    };
    // (what was put into the LDS, and what is read from it; a barrier of the language would wait for what is on its way to registers too)
    auto all_there = [&] {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        barrier_only();
    };
    if (MODE == WEIGHTS && steps > 0) {
        look_up(0);
        look_up(1);
        __syncthreads();
    }
    static_assert(kLook % AHEAD == 0, "blocks of rows begin where a round of steps does");
    // Steps that are whole, in a loop of their own: what is on its way is waited for by count there, behind a branch altogether.
    const int whole = (!A_ACROSS || row0 + BM <= p.m) && (!B_ACROSS || col0 + BN <= p.cols) ? terms / STEP : 0;
    auto step = [&](int s, int d, auto&& next) {
        all_there();
        store(raw[d]);
        if (d == 0 && s > 0 && s % kLook == 0) look_up(s / kLook + 1);
        all_there();
        next(s + AHEAD, raw[d]);
        __builtin_amdgcn_s_setprio(1);      // (the matrix cores before another block's splits)
        sums();
        __builtin_amdgcn_s_setprio(0);
    };
    int s0 = 0;
    if (whole >= 2 * AHEAD) {
#pragma unroll
        for (int d = 0; d < AHEAD; ++d) request_whole(d, raw[d]);
#pragma unroll 1
        for (; s0 + 2 * AHEAD <= whole; s0 += AHEAD) {
#pragma unroll
            for (int d = 0; d < AHEAD; ++d) step(s0 + d, d, request_whole);
        }
    } else {
#pragma unroll
        for (int d = 0; d < AHEAD; ++d)
            if (d < steps) request(d, raw[d]);
    }
#pragma unroll 1
    for (; s0 < steps; s0 += AHEAD) {
#pragma unroll
        for (int d = 0; d < AHEAD; ++d) {
            if (s0 + d >= steps) break;
            step(s0 + d, d, [&](int s, Eight<T> (&to)[PA + PB]) {
                if (s < steps) request(s, to);
            });
        }
    }
    const int row_w = row0 + wm * NM * 16, col_w = col0 + wn * NT * 16;
    if constexpr (SINGLE) {
        // (sums that are not finite for the scale, or are not at all, are formed again)
        constexpr float kBack = 1.0f / (kSplitScale * kSplitScale);
        float none = 0.0f;
#pragma unroll
        for (int i = 0; i < NM; ++i)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    none = fmaf(acc[i][t][j], 0.0f, none);
                    acc[i][t][j] *= kBack;
                }
        if (__builtin_expect(__any(none != none), 0)) {
#pragma unroll
            for (int i = 0; i < NM; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    bool all = true;
#pragma unroll
                    for (int j = 0; j < 4; ++j) all = all && fabsf(acc[i][t][j]) <= std::numeric_limits<float>::max();
                    if (__all(all)) continue;
                    const f32x4 again = plain_sums<T, MODE>(p, at, lane, row_w + 16 * i, col_w + 16 * t);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (!(fabsf(acc[i][t][j]) <= std::numeric_limits<float>::max())) acc[i][t][j] = again[j];
                }
        }
    }
    if (SUMS && with_sums && lane < 16) {
#pragma unroll
        for (int i = 0; i < NM; ++i) {
            const int m = row_w + 16 * i + lane;
            if (m >= p.m) continue;
            float sum = ones_acc[SUMS ? i : 0][0];
            if (SINGLE) {
                if (fabsf(sum) <= std::numeric_limits<float>::max()) sum *= 1.0f / kSplitScale;
                else {
                    sum = 0.0f;
                    for (int k = at.begin; k < at.end; ++k) sum += (float)static_cast<const T*>(p.a)[p.order[k] * p.a_stride + m];
                }
            }
            store_sum<T>(p, at, m, sum);
        }
    }
    finish<T, MODE, NM, NT>(p, at, lane, row_w, col_w, look, acc);
}

// Sums of the pieces of a group's dW and db, in order.  (50 000 rows of 12 groups, 256 -> 512: 10 us.)
template <typename T>
__global__ __launch_bounds__(256) void k_join(const Product p)
{
    const int lane = threadIdx.x & 63, g = blockIdx.y;
    const int pieces = (p.offsets[g + 1] - p.offsets[g] + p.piece - 1) / p.piece;
    if (pieces < 2) return;
    // (the parts of the groups in front)
    int slots = 0;
    for (int h = lane; h < g; h += 64) {
        const int n = (p.offsets[h + 1] - p.offsets[h] + p.piece - 1) / p.piece;
        slots += n > 1 ? n : 0;
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) slots += __shfl_xor(slots, d, 64);
    const long each = (long)p.m * p.cols;
    for (long e = ((long)blockIdx.x * 256 + threadIdx.x) * 4; e < each; e += (long)gridDim.x * 1024) {
        const float* from = p.partial + slots * each + e;
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (int i = 0; i < pieces; ++i) {
            float v[4];
            load_run<4>(from + i * each, each - e, v);
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[j] += v[j];
        }
        store_run<4>(static_cast<T*>(p.out) + g * each + e, each - e, sum);
    }
    if (p.sums)
        for (int m = blockIdx.x * 256 + threadIdx.x; m < p.m; m += gridDim.x * 256) {
            float sum = 0.0f;
#pragma unroll 8
            for (int i = 0; i < pieces; ++i) sum += p.partial_sums[(long)(slots + i) * p.m + m];
            static_cast<T*>(p.sums)[(long)g * p.m + m] = (T)sum;
        }
}

// ---- few rows: bound by the weights' bytes
//
// Up to 64 rows are not sorted: a block has 16 columns of the product of a row's group, finds the rows of the same group itself, and leaves if
// its own is not the first of them.  Eight wavefronts have 128 bytes of the weights' rows by turns, three or four of them under way; 16 or
// 32 rows at a time, so that two blocks have room on a CU (with 64 at a time there was one: 64 us for the first call below).
// 48 rows of 32 groups, 2 048 x 2 048 in bfloat16: 48 us, 5.6 TB/s of the weights' bytes; 16 of 16, 4 096 x 4 096: 89 us, 6.0.
// In tiles of 64: 24 rows of 3 groups, 192 -> 128 in single precision 15 us, here 11; 32 rows of one, 4 096 x 4 096 in bfloat16 20 us, here 12; but 64 of
// 4 groups 27, here 31.
constexpr int kMostFew = 64;
template <typename T, int MT>
__device__ __forceinline__ void few_rows(const Product& p, int group, const int* rows, int count, f32x4 (*part)[2][64])
{
    constexpr int V = kRun<T>, UNIT = 8 * V;
    typedef typename Operand<T>::type frag;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col0 = blockIdx.x * 16, mine = (lane & 3) * V;
    const T* W = static_cast<const T*>(p.b) + group * p.b_each + min(col0 + lane / 4, p.cols - 1) * p.b_stride + mine;
    const T* in[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) in[i] = static_cast<const T*>(p.a) + rows[min(16 * i + lane / 4, count - 1)] * p.a_stride + mine;
    f32x4 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = f32x4{0, 0, 0, 0};
    struct Unit {
        frag w[2], x[MT][2];
    };
    const int full = p.k / UNIT;
    auto fetch = [&](int u, Unit& v) {
        const int k = min(u, full - 1) * UNIT;
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
        constexpr int UNITS = MT == 1 ? 4 : 3;
        Unit unit[UNITS];
#pragma unroll
        for (int q = 0; q < UNITS - 1; ++q) fetch(u + 8 * q, unit[q]);
#pragma unroll 1
        for (;;) {
            bool done = false;
#pragma unroll
            for (int q = 0; q < UNITS; ++q) {
                if (done) continue;
                fetch(u + 8 * (UNITS - 1), unit[(q + UNITS - 1) % UNITS]);
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
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MT; ++i) part[wave][i][lane] = acc[i];
    __syncthreads();
    for (int at = threadIdx.x; at < MT * 256; at += 512) {
        const int row = at / 16, c = at % 16, col = col0 + c;
        if (row >= count || col >= p.cols) continue;
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) sum += part[w][row / 16][c / 4 * 16 + row % 16][c % 4];
        if (p.bias) sum += (float)static_cast<const T*>(p.bias)[(long)group * p.cols + col];
        static_cast<T*>(p.out)[rows[row] * p.out_stride + col] = (T)sum;
    }
}
template <typename T>
__global__ __launch_bounds__(512, 4) void k_few(const Product p, const int* index)
{
    __shared__ f32x4 part[8][2][64];
    __shared__ int rows[kMostFew];
    const int lane = threadIdx.x & 63, all = (int)p.rows, key = row_key(index[min(lane, all - 1)], p.groups);
    const int group = __builtin_amdgcn_readlane(key, blockIdx.y);
    const unsigned long same = __ballot(lane < all && key == group);
    if (same & ((1ul << blockIdx.y) - 1)) return;      // (an earlier row's block does it)
    const int count = __popcll(same);
    if (threadIdx.x < 64 && (same >> lane & 1)) rows[__popcll(same & ((1ul << lane) - 1))] = lane;
    __syncthreads();
    if (group >= p.groups) {
        const T v = (T)(group == p.groups ? 0.0f : std::numeric_limits<float>::quiet_NaN());
        for (int at = threadIdx.x; at < 16 * count; at += 512)
            if ((int)blockIdx.x * 16 + at % 16 < p.cols) static_cast<T*>(p.out)[rows[at / 16] * p.out_stride + blockIdx.x * 16 + at % 16] = v;
        return;
    }
    if (count <= 16) few_rows<T, 1>(p, group, rows, count, part);
    else
        for (int first = 0; first < count; first += 32) few_rows<T, 2>(p, group, rows + first, min(32, count - first), part);
}

// ---- host side

void check(const smx_grouped_linear* p)
{
    refuse_unless(p, "the description must not be null");
    (void)type_bytes(p->type);
    refuse_unless(p->rows >= 0 && p->rows <= 1L << 28, "rows: 0 to 2^28");
    refuse_unless(p->d_in >= 1 && p->d_out >= 1 && p->d_in <= (1 << 20) && p->d_out <= (1 << 20), "d_in and d_out: 1 to 2^20");
    refuse_unless(p->num_groups >= 0 && p->num_groups <= SMX_MOST_GROUPS, "num_groups: 0 to 4096");
    refuse_unless(p->x_stride >= p->d_in && p->weight_stride >= p->d_in, "strides of x and weight: at least d_in");
    refuse_unless(p->weight_each >= 0, "the stride between matrices: from 0 on");
    refuse_unless(p->weight || p->num_groups == 0, "weight must not be null");
    refuse_unless(p->rows == 0 || (p->x && p->index), "x and index must not be null");
    refuse_unless((p->order == nullptr) == (p->offsets == nullptr) || p->rows == 0, "order and offsets: both or neither");
}

// What k_direct takes: rows at multiples of 16 bytes, whole pieces of 16 bytes; the offsets inside a tile have 32 bits,
// and so have those of rows that lie anywhere.
bool in_pieces(const void* p, long stride, long numbers) { return (reinterpret_cast<size_t>(p) & 15) == 0 && stride % 8 == 0 && numbers % 8 == 0 && stride <= 1 << 22; }
bool within_reach(long rows, long stride) { return rows * stride * 2 < 1L << 32; }

struct Call : Launches {
    const smx_grouped_linear& p;
    Arena arena;
    RowOrder groups{};
    void sort()
    {
        groups = RowOrder{const_cast<int*>(p.order), const_cast<int*>(p.offsets), nullptr};
        if (p.offsets && p.rows) return;
        groups.order = arena.take<int>(p.rows);
        groups.offsets = arena.take<int>(p.num_groups + 2L);
        sort_rows(*this, arena, p.index, p.rows, p.num_groups, groups);
    }
    template <typename T, int MODE, bool LARGE, int BM, int STAGES>
    void direct(const Product& q, long blocks)
    {
        constexpr int bytes = STAGES * 2 * BM * 128 + (MODE == WEIGHTS ? 4096 : 1024);
        auto kernel = k_direct<T, MODE, LARGE, BM, STAGES>;
        if (bytes > 64 * 1024 && !dry) hip_ok(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes), "LDS");
        // (a last round of tiles cut in four has three more blocks for each)
        start(kernel, up(blocks, 8) + (LARGE && MODE != WEIGHTS ? 3 * kCUs / 4 : 0), 1, 1, LARGE ? 512 : 256, bytes, q);
    }
    // Tiles for all rows in the worst case: every group has one that is not full.
    long row_tiles(int high) const { return p.rows / high + std::min(p.rows, p.num_groups + 2L); }

    // y or dx
    template <typename T, int MODE>
    void rows(Product q, bool direct_ok)
    {
        auto tiles = [&](int high, int wide) {
            q.col_tiles = (q.cols + wide - 1) / wide;
            return row_tiles(high) * q.col_tiles;
        };
        // The largest tiles that are enough for three quarters of the CUs (of the usual group the last tile is half full), that columns fill by three
        // quarters, and that groups of the usual size fill; those of 128 also by half, since they read the weights once for two of 64.
        // In bfloat16, 16 384 rows of 4 groups, 1 024 columns: 128 terms 14.9 us and 15.6 in tiles of 128, 1 024 terms 34 and 44.  63 855 rows of
        // 15 groups, 96 -> 32: tiles of 256 20 us.  1 000 rows of 8 groups, 4 096 x 4 096, y and dx: 66 and 61 us in tiles of 128, 92 and 86 of 64;
        // 4 000 rows of 48 groups, 2 048 x 2 048: 116 and 96, and 110 and 114 (one rule for both: dx gains more than y loses, where y loses at all);
        // 5 000 rows of 60, 512 -> 1 024 in single precision: 51 and 68, and 66 and 75.  (Groups of even size.)
        const long used = std::min(p.rows, std::max(1L, (long)p.num_groups));
        auto fits = [&](int tile) {
            const long across = (q.cols + tile - 1) / tile;
            return (p.rows / tile + used / 2) * across >= 192 && 4L * q.cols >= 3 * across * tile && (tile == 128 ? 2 : 1) * p.rows >= used * tile;
        };
        if constexpr (!std::is_same_v<T, float>) {
            if (direct_ok) {
                if (fits(256)) direct<T, MODE, true, 256, 2>(q, tiles(256, 256));
                else if (fits(128)) direct<T, MODE, false, 128, 2>(q, tiles(128, 128));
                else if (tiles(64, 64) > kCUs) direct<T, MODE, false, 64, 3>(q, tiles(64, 64));
                else direct<T, MODE, false, 64, 8>(q, tiles(64, 64));
                return;
            }
        }
        if (fits(128)) start(k_staged<T, MODE, 128, 128, (std::is_same_v<T, float> ? 2 : 1)>, up(tiles(128, 128), 8), 1, 1, 256, 0, q);
        else start(k_staged<T, MODE, 64, 64, (std::is_same_v<T, float> ? 4 : 2)>, up(tiles(64, 64), 8), 1, 1, 256, 0, q);
    }
    template <typename T>
    void forward(T* y, long y_stride)
    {
        const T *x = static_cast<const T*>(p.x), *W = static_cast<const T*>(p.weight);
        Product q{};
        q.a = x; q.a_stride = p.x_stride; q.b = W; q.b_each = p.weight_each; q.b_stride = p.weight_stride; q.bias = p.bias; q.groups = p.num_groups; q.k = p.d_in; q.cols = p.d_out;
        q.rows = p.rows; q.out = y; q.out_stride = y_stride;
        if (p.rows <= kMostFew) {
            start(k_few<T>, (p.d_out + 15) / 16, p.rows, 1, 512, 0, q, p.index);
            return;
        }
        sort();
        q.order = groups.order; q.offsets = groups.offsets;
        rows<T, FORWARD>(q, in_pieces(x, p.x_stride, p.d_in) && in_pieces(W, p.weight_stride, p.d_in) && p.weight_each % 8 == 0 && within_reach(p.rows, p.x_stride));
    }
    template <typename T>
    void backward(const T* dy, long dy_stride, T* dx, long dx_stride, T* dW, T* db)
    {
        const T *x = static_cast<const T*>(p.x), *W = static_cast<const T*>(p.weight);
        sort();
        Product q{};
        q.a = dy; q.a_stride = dy_stride; q.groups = p.num_groups; q.rows = p.rows; q.order = groups.order; q.offsets = groups.offsets;
        const bool dy_ok = in_pieces(dy, dy_stride, p.d_out) && within_reach(p.rows, dy_stride);
        if (dx && p.rows) {
            q.b = W; q.b_each = p.weight_each; q.b_stride = p.weight_stride; q.k = p.d_out; q.cols = p.d_in; q.out = dx; q.out_stride = dx_stride;
            rows<T, ROWS>(q, dy_ok && in_pieces(W, p.weight_stride, p.d_in) && p.weight_each % 8 == 0);
        }
        bool summed = false;      // (db)
        if (dW && p.num_groups) {
            q.b = x; q.b_each = 0; q.b_stride = p.x_stride; q.m = p.d_out; q.cols = p.d_in; q.out = dW;
            summed = weights<T>(q, db, dy_ok && in_pieces(x, p.x_stride, p.d_in) && within_reach(p.rows, p.x_stride));
        }
        if (db && p.num_groups && (dry || !summed)) add_rows(*this, arena, p.type, dy, dy_stride, p.index, p.rows, p.num_groups, p.d_out, groups, 1.0f, db);
    }
    // dW: which tiles, and how long the pieces of a group's rows are.  Small tiles and short pieces keep more CUs busy; large tiles
    // take fewer bytes for a product, and pieces have to be written and read again to be joined.  What each way takes is estimated from
    // the stages of 64 rows that a CU goes through (`stage`: us, of as many tiles as run on it at once), and the least is taken:
    //   16 384 rows of 4 groups, 1 024 x 1 024 in bfloat16: tiles of 128 in whole groups 119 us, in two pieces 82;
    //   50 000 rows of 12 groups, 256 x 512 in single precision: pieces of 832 rows (more blocks than run at once) 149 us, of 896 100.
    struct Way {
        int tile, piece;
    };
    Way way(int m, int cols, bool direct_ok, bool single) const
    {
        const double used = (double)std::max(1L, std::min(p.rows, (long)p.num_groups)), rows = (double)p.rows;
        Way best{64, 1 << 28};
        double least = std::numeric_limits<double>::max();
        for (int tile = direct_ok && !single ? 256 : 128; tile >= 64; tile /= 2) {
            const double each = (double)((m + tile - 1) / tile) * ((cols + tile - 1) / tile);
            const double on_cu = tile == 256 ? 1 : tile == 128 ? 2 : 4, at_once = kCUs * on_cu;
            const double stage = (tile == 256 ? 1.7 : tile == 128 ? 1.1 : 0.8) * (single ? 8 : direct_ok ? 1 : 2);
            for (int parts : {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32, 48, 64}) {
                // (a group's last piece is half as long as the others; groups of more than twice the usual rows are cut whatever the rest are)
                const double piece = std::max(256.0, 64 * std::ceil((parts == 1 ? std::max(2 * rows / used, 1.5 * rows * each / at_once) : rows / used / parts) / 64));
                const double items = rows / piece + used * (parts == 1 ? 1.0 : 0.5), blocks = items * each, rounds = blocks / at_once;
                const double usual = parts == 1 ? rows / used : piece;
                // (fewer blocks on a CU than could be there are faster, though not in proportion)
                const double shared = std::min(1.0, std::max(0.6, std::ceil(blocks / kCUs) / on_cu));
                const double time = std::max(rounds < 8 ? std::ceil(rounds) : rounds, 1.0) * (usual / 64 + 3) * stage * shared + (parts == 1 ? 0.0 : 5 + rows / piece * m * (double)cols * 8 / 4e6);
                if (time < least) least = time, best = Way{tile, (int)std::min(piece, (double)(1 << 28))};
                if (piece <= 256.0) break;
            }
        }
        return best;
    }
    // The answer is whether db is there too, if it is asked for.
    template <typename T>
    bool weights(Product q, T* db, bool direct_ok)
    {
        constexpr bool SINGLE = std::is_same_v<T, float>;
        const Way w = way(q.m, q.cols, direct_ok, SINGLE);
        q.row_tiles = (q.m + w.tile - 1) / w.tile;
        q.col_tiles = (q.cols + w.tile - 1) / w.tile;
        q.piece = w.piece;
        const long each = (long)q.row_tiles * q.col_tiles, items = p.rows / q.piece + p.num_groups, slots = 2 * (p.rows / q.piece);
        q.partial = arena.take<float>(slots * q.m * q.cols);
        const bool summed = SINGLE || !direct_ok || w.tile == 64;
        if (summed) {
            q.sums = db;
            q.partial_sums = arena.take<float>(slots * q.m);
        }
        const long blocks = items * (each >= 8 ? up(each, 8) : each);
        if constexpr (!SINGLE) {
            if (direct_ok) {
                if (w.tile == 256) direct<T, WEIGHTS, true, 256, 2>(q, blocks);
                else if (w.tile == 128) direct<T, WEIGHTS, false, 128, 2>(q, blocks);
                else if (blocks > kCUs) direct<T, WEIGHTS, false, 64, 3>(q, blocks);
                else direct<T, WEIGHTS, false, 64, 8>(q, blocks);
            }
        }
        if (SINGLE || !direct_ok) {
            if (w.tile == 128) start(k_staged<T, WEIGHTS, 128, 128, (std::is_same_v<T, float> ? 2 : 1)>, blocks, 1, 1, 256, 0, q);
            else start(k_staged<T, WEIGHTS, 64, 64, (std::is_same_v<T, float> ? 4 : 2)>, blocks, 1, 1, 256, 0, q);
        }
        // (few blocks: most groups have nothing to join)
        if (slots) start(k_join<T>, std::min(((long)q.m * q.cols + 1023) / 1024, std::max(1L, 2048L / p.num_groups)), p.num_groups, 1, 256, 0, q);
        return summed;
    }
};

// (whatever the pointers' alignment is: the size does not depend on it but for dW's pieces, which are longest for the largest tiles)
long workspace(const smx_grouped_linear* p, bool backward)
{
    long most = 0;
    for (int some = 256; some >= 2; some -= 254) {
        smx_grouped_linear q = *p;
        if (q.rows) q.x = reinterpret_cast<const void*>((size_t)some);
        Call c{{nullptr, true}, q, {reinterpret_cast<char*>(256)}};
        with_type(q.type, [&](auto t) {
            using T = decltype(t);
            T* at = reinterpret_cast<T*>((size_t)256);
            if (backward) c.backward<T>(at, q.d_out, at, q.d_in, at, at);
            else if (q.rows > 0) c.forward<T>(at, q.d_out);
        });
        most = std::max(most, c.arena.used);
    }
    return most;
}

}  // namespace

}  // namespace smx

using namespace smx;

extern "C" int smx_grouped_linear_workspace(const smx_grouped_linear* p, int backward, long* bytes)
{
    return finetune_entry("smx_grouped_linear_workspace", [&] {
        check(p);
        refuse_unless(bytes, "bytes must not be null");
        *bytes = workspace(p, backward != 0);
    });
}

extern "C" int smx_grouped_linear_forward(const smx_grouped_linear* p, void* d_y, long y_stride, void* d_workspace, long workspace_bytes, void* stream)
{
    return finetune_entry("smx_grouped_linear_forward", [&] {
        check(p);
        if (p->rows == 0) return;
        refuse_unless(d_y && y_stride >= p->d_out, "y must not be null, its stride at least d_out");
        check_workspace(d_workspace, workspace_bytes, workspace(p, false), "smx_grouped_linear_workspace");
        require_gfx950();
        Call c{{static_cast<hipStream_t>(stream), false}, *p, {static_cast<char*>(d_workspace)}};
        with_type(p->type, [&](auto t) { c.forward<decltype(t)>(static_cast<decltype(t)*>(d_y), y_stride); });
        hip_ok(hipGetLastError(), "launch");
    });
}

extern "C" int smx_grouped_linear_backward(const smx_grouped_linear* p, const void* d_dy, long dy_stride, void* d_dx, long dx_stride, void* d_dweight, void* d_dbias,
                                           void* d_workspace, long workspace_bytes, void* stream)
{
    return finetune_entry("smx_grouped_linear_backward", [&] {
        check(p);
        refuse_unless(p->rows == 0 || (d_dy && dy_stride >= p->d_out), "dy must not be null, its stride at least d_out");
        refuse_unless(!d_dx || dx_stride >= p->d_in, "the stride of dx: at least d_in");
        if (!d_dx && !d_dweight && !d_dbias) return;
        check_workspace(d_workspace, workspace_bytes, workspace(p, true), "smx_grouped_linear_workspace");
        require_gfx950();
        Call c{{static_cast<hipStream_t>(stream), false}, *p, {static_cast<char*>(d_workspace)}};
        with_type(p->type, [&](auto t) {
            using T = decltype(t);
            c.backward<T>(static_cast<const T*>(d_dy), dy_stride, static_cast<T*>(d_dx), dx_stride, static_cast<T*>(d_dweight), static_cast<T*>(d_dbias));
        });
        hip_ok(hipGetLastError(), "launch");
    });
}
