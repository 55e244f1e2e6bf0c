// A shared projection with a low-rank adapter per row beside it, and its gradient.
//
//   y = W x + B_a h,  h = c_a A_a x
//   g = c_a B_a^T dy:   dx = W^T dy + A_a^T g,   dA_a = sum over the adapter's rows of g x^T,   dB_a = sum of dy h^T
//
// Forward: h of all rows (k_down), then one product that adds the adapters' part to its sums before they are rounded and stored
// (k_product16, k_product32; few rows: k_down_few, k_product_few).  Gradient: h and g, the product with W^T, and for dA and dB the rows
// sorted by adapter (k_group_*), sums over pieces of an adapter's rows (k_outer), and the sums of those (k_join).
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

__device__ __forceinline__ bool has_adapter(int a, int n) { return a >= 0 && a < n; }
__device__ __forceinline__ bool is_bad(int a, int n) { return a < -1 || a >= n; }

constexpr int kPiece = 32;           // terms of a sum that a step of a product takes
constexpr int kMostFew = 64;         // rows of the kernels for few rows

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
    long dst_each, part;                // strides of a matrix and a part
    int rows, k, k_padded;
};
// a block takes 64 rows and 64 numbers of them
template <typename T, bool SPLIT>
__global__ __launch_bounds__(256) void k_lay_out(const Layout p)
{
    __shared__ T tile[64][65];
    const int row0 = blockIdx.y * 64, k0 = blockIdx.x * 64;
    const T* src = static_cast<const T*>(p.src) + blockIdx.z * p.src_each;
    const bool along = p.src_k == 1;
    for (int i = threadIdx.x; i < 64 * 64; i += 256) {
        const int r = along ? i / 64 : i % 64, k = along ? i % 64 : i / 64;
        tile[r][k] = row0 + r < p.rows && k0 + k < p.k ? src[(row0 + r) * p.src_row + (k0 + k) * p.src_k] : (T)0.0f;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * 32; i += 256) {
        const int r = i / 32, k = i % 32 * 2;
        if (row0 + r >= p.rows || k0 + k >= p.k_padded) continue;
        const long at = blockIdx.z * p.dst_each + (long)(row0 + r) * p.k_padded + k0 + k;
        if constexpr (SPLIT) {
            const float x[2] = {(float)tile[r][k] * kSplitScale, (float)tile[r][k + 1] * kSplitScale};
            bf16 part[3][2];
            split(x, part);
#pragma unroll
            for (int s = 0; s < 3; ++s) {
                const bf16x2 v = {part[s][0], part[s][1]};
                *reinterpret_cast<bf16x2*>(static_cast<bf16*>(p.dst) + s * p.part + at) = v;
            }
        } else {
            T* dst = static_cast<T*>(p.dst) + at;
            dst[0] = tile[r][k]; dst[1] = tile[r][k + 1];
        }
    }
}
template <typename T, bool SPLIT>
void lay_out(const Layout& p, int matrices, hipStream_t s)
{
    hipLaunchKernelGGL((k_lay_out<T, SPLIT>), dim3((p.k_padded + 63) / 64, (p.rows + 63) / 64, matrices), dim3(256), 0, s, p);
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

// A block takes 16 rows; its wavefronts have 128 bytes of a row by turns, and their sums are added in order.
template <typename T, int RT>
__global__ __launch_bounds__(256) void k_down(const Down p)
{
    constexpr int V = kRun<T>, UNIT = 8 * V;
    __shared__ f32x4 part[4][RT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    const long row = min((long)blockIdx.x * 16 + n, p.rows - 1);
    const bool live = (long)blockIdx.x * 16 + n < p.rows;
    const int a = p.index[row];
    const bool good = live && has_adapter(a, p.adapters);
    const T* in = static_cast<const T*>(p.in) + row * p.in_stride;
    if (live && !good && wave == 0)
#pragma unroll
        for (int q = 0; q < RT; ++q)
            if (16 * q < p.padded) *reinterpret_cast<f32x4*>(p.h + row * p.padded + 16 * q + 4 * g) = f32x4{0, 0, 0, 0};
    unsigned left = (unsigned)__ballot(good) & 0xffffu;
    while (left) {
        const int cur = __builtin_amdgcn_readlane(a, __builtin_ctz(left));
        const bool mine = good && a == cur;
        left &= ~(unsigned)__ballot(mine);
        f32x4 acc[RT];
#pragma unroll
        for (int q = 0; q < RT; ++q) acc[q] = f32x4{0, 0, 0, 0};
        const T* F = static_cast<const T*>(p.F) + cur * p.f_each;
        for (int k0 = wave * UNIT; k0 < p.k; k0 += 4 * UNIT)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int k = k0 + u * (UNIT / 2) + g * V;
                const auto x = load_operand(in + k, p.k - k);
#pragma unroll
                for (int q = 0; q < RT; ++q) {
                    const int r = 16 * q + n;
                    const auto f = load_operand(F + (long)min(r, p.rank - 1) * p.f_row + k, r < p.rank ? p.k - k : 0);
                    acc[q] = mma(f, x, acc[q]);
                }
            }
#pragma unroll
        for (int q = 0; q < RT; ++q) part[wave][q][lane] = acc[q];
        __syncthreads();
        const float c = p.scale ? p.scale[cur] : 1.0f;
        for (int q = wave; q < RT; q += 4) {
            f32x4 sum = part[0][q][lane];
#pragma unroll
            for (int w = 1; w < 4; ++w) sum += part[w][q][lane];
            if (mine && 16 * q < p.padded) *reinterpret_cast<f32x4*>(p.h + row * p.padded + 16 * q + 4 * g) = sum * c;
        }
        __syncthreads();
    }
}

// Few rows: a wavefront per number of h.
template <typename T>
__global__ __launch_bounds__(256) void k_down_few(const Down p)
{
    constexpr int V = kRun<T>;
    const long row = blockIdx.x;
    const int lane = threadIdx.x & 63, r = blockIdx.y * 4 + (threadIdx.x >> 6), a = p.index[row];
    float sum = 0.0f;
    if (has_adapter(a, p.adapters) && r < p.rank) {
        const T* in = static_cast<const T*>(p.in) + row * p.in_stride;
        const T* F = static_cast<const T*>(p.F) + a * p.f_each + (long)r * p.f_row;
#pragma unroll 4
        for (int k = lane * V; k < p.k; k += 64 * V) {
            float x[V], f[V];
            load_run<V>(in + k, p.k - k, x);
            load_run<V>(F + k, p.k - k, f);
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
    const void* W;               // laid out: rows (columns of the result) w_stride apart, of a multiple of 32 numbers
    long w_stride, w_part;
    const void* W0;              // as the caller has it
    long w0_col, w0_k;
    const void* F;
    long f_each, f_col, f_r;
    const float* h;
    const int* index;
    int adapters, rank, padded, k, k_padded, cols;
    long rows;
    void* out;
    long out_stride;
    int row_tiles, col_tiles;
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

// Adds the adapters' part to sums of NM tiles of 16 rows and NT of 16 columns.  Lane (n, g) holds of tile (i, t) row i * 16 + n and
// columns 4 NT g + 4 t + 0..3.
template <typename T, int NM, int NT>
__device__ __forceinline__ void add_adapters(const Product& p, int lane, long row0, int col0, f32x4 (&acc)[NM][NT])
{
    const int n = lane & 15, g = lane >> 4;
    const T* F[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) F[t] = static_cast<const T*>(p.F) + min(col0 + 4 * NT * (n >> 2) + 4 * t + (n & 3), p.cols - 1) * p.f_col;
#pragma unroll
    for (int i = 0; i < NM; ++i) {
        const long row = min(row0 + 16 * i + n, p.rows - 1);
        const int a = p.index[row];
        const bool good = row0 + 16 * i + n < p.rows && has_adapter(a, p.adapters);
        unsigned left = (unsigned)__ballot(good) & 0xffffu;
        while (left) {
            const int cur = __builtin_amdgcn_readlane(a, __builtin_ctz(left));
            const bool mine = good && a == cur;
            left &= ~(unsigned)__ballot(mine);
            f32x4 sum[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) sum[t] = f32x4{0, 0, 0, 0};
            for (int r = 4 * g; r < p.padded; r += 16) {
                const f32x4 h = *reinterpret_cast<const f32x4*>(p.h + row * p.padded + r);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const T* from = F[t] + cur * p.f_each + r * p.f_r;
                    float f[4];
                    if (p.f_r == 1) load_run<4>(from, p.rank - r, f);
                    else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) f[j] = r + j < p.rank ? (float)from[j * p.f_r] : 0.0f;
                    }
                    sum[t] = mma(f32x4{f[0], f[1], f[2], f[3]}, h, sum[t]);
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][t][j] += mine ? sum[t][j] : 0.0f;
        }
    }
}
template <typename T, int NM, int NT>
__device__ __forceinline__ void store_tiles(const Product& p, int lane, long row0, int col0, const f32x4 (&acc)[NM][NT])
{
    constexpr int V = kRun<T>, N = 4 * NT < V ? 4 * NT : V;
    const int n = lane & 15, g = lane >> 4, col = col0 + 4 * NT * g;
#pragma unroll
    for (int i = 0; i < NM; ++i) {
        const long row = row0 + 16 * i + n;
        if (row >= p.rows) continue;
        const bool bad = is_bad(p.index[row], p.adapters);
        T* out = static_cast<T*>(p.out) + row * p.out_stride + col;
#pragma unroll
        for (int u = 0; u < 4 * NT; u += N) {
            float v[N];
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = bad ? std::numeric_limits<float>::quiet_NaN() : acc[i][(u + j) / 4][(u + j) % 4];
            store_run<N>(out + u, p.cols - col - u, v);
        }
    }
}

// 16-bit types.  Tiles of 32 terms come straight from memory into LDS, three steps ahead, four places; WM x WN wavefronts share the
// tile.  16 bytes of a row lie at a place that depends on the row, so that lanes that read together meet different banks.
template <typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 2) void k_product16(const Product p)
{
    constexpr int WAVES = WM * WN, NM = BM / WM / 16, NT = BN / WN / 16, PER = (BM + BN) / 16 / WAVES, STAGES = 4, AHEAD = 3, STAGE = (BM + BN) * 64;
    static_assert((BM + BN) / 16 % WAVES == 0, "loads of a wavefront");
    typedef typename Operand<T>::type frag;
    extern __shared__ __align__(16) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    int rt, ct;
    if (!tile_of(p, rt, ct)) return;
    const long row0 = (long)rt * BM;
    const int col0 = ct * BN;
    const char* from[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        const int chunk = wave + u * WAVES;
        if (chunk < BM / 16) {
            const int r = chunk * 16 + lane / 4;
            from[u] = static_cast<const char*>(p.in) + 2 * min(row0 + r, p.rows - 1) * p.in_stride + 16 * ((lane & 3) ^ (r >> 1 & 3));
        } else {
            const int r = (chunk - BM / 16) * 16 + lane / 4;
            from[u] = static_cast<const char*>(p.W) + 2 * (long)min(col0 + r, p.cols - 1) * p.w_stride + 16 * ((lane & 3) ^ ((r >> 1 & 1) | (r / (4 * NT) & 1) << 1));
        }
    }
    const unsigned lds0 = lds_address(lds);
    const int steps = p.k_padded / kPiece;
    auto request = [&](int s) {
#pragma unroll
        for (int u = 0; u < PER; ++u) load_into_lds(from[u] + (long)s * 64, lds0 + s % STAGES * STAGE + (wave + u * WAVES) * 1024);
    };
    f32x4 acc[NM][NT];
#pragma unroll
    for (int i = 0; i < NM; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[i][t] = f32x4{0, 0, 0, 0};
    const int wm = wave / WN, wn = wave % WN;
    const unsigned char* xs = lds + (wm * NM * 16 + n) * 64 + 16 * (g ^ (n >> 1 & 3));
    const unsigned char* ws = lds + (BM + wn * NT * 16 + 4 * NT * (n >> 2) + (n & 3)) * 64 + 16 * (g ^ ((n >> 1 & 1) | (n >> 2 & 1) << 1));
#pragma unroll
    for (int s = 0; s < AHEAD; ++s)
        if (s < steps) request(s);
    for (int s = 0; s < steps; ++s) {
        if (s + AHEAD <= steps) wait_loads<(AHEAD - 1) * PER>();
        else wait_loads<0>();
        barrier_only();      // this step's tiles are there, and everybody has read those of the step before
        if (s + AHEAD < steps) request(s + AHEAD);
        const int at = s % STAGES * STAGE;
        frag x[NM], w[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) w[t] = *reinterpret_cast<const frag*>(ws + at + t * 256);
#pragma unroll
        for (int i = 0; i < NM; ++i) x[i] = *reinterpret_cast<const frag*>(xs + at + i * 1024);
#pragma unroll
        for (int i = 0; i < NM; ++i)
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[i][t] = mma(w[t], x[i], acc[i][t]);
    }
    const long row_w = row0 + wm * NM * 16;
    const int col_w = col0 + wn * NT * 16;
    add_adapters<T, NM, NT>(p, lane, row_w, col_w, acc);
    store_tiles<T, NM, NT>(p, lane, row_w, col_w, acc);
}

// Single precision on the bf16 matrix instructions: both operands in three parts, exactly, of whose products the six largest are formed
// (what is left out is below 1.002 2^-24 of a product), small ones first.  The rows' numbers are split here, W's beforehand.  Numbers are
// brought up by 2^24 first, so that the parts of small ones are normal numbers; sums that are not finite for it, or are not at all, are
// formed again in single precision.
template <int NM, int NT>
__global__ __launch_bounds__(256, 2) void k_product32(const Product p)
{
    constexpr int BM = 32 * NM, BN = 32 * NT, XR = BM * 4 / 256, WR = 3 * BN * 4 / 256;
    __shared__ __align__(16) unsigned char lds[3 * (BM + BN) * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    int rt, ct;
    if (!tile_of(p, rt, ct)) return;
    const long row0 = (long)rt * BM;
    const int col0 = ct * BN;
    const float* from[XR];
    const bf16* wfrom[WR];
    int to[XR], wto[WR];
#pragma unroll
    for (int u = 0; u < XR; ++u) {
        const int i = threadIdx.x + 256 * u, r = i / 4;
        from[u] = static_cast<const float*>(p.in) + min(row0 + r, p.rows - 1) * p.in_stride + 8 * (i & 3);
        to[u] = r * 64 + 16 * ((i & 3) ^ (r >> 1 & 3));
    }
#pragma unroll
    for (int u = 0; u < WR; ++u) {
        const int i = threadIdx.x + 256 * u, part = i / (BN * 4), r = i / 4 % BN;
        wfrom[u] = static_cast<const bf16*>(p.W) + part * p.w_part + (long)min(col0 + r, p.cols - 1) * p.w_stride + 8 * (i & 3);
        wto[u] = 3 * BM * 64 + part * BN * 64 + r * 64 + 16 * ((i & 3) ^ ((r >> 1 & 1) | (r / (4 * NT) & 1) << 1));
    }
    float x[XR][8];
    bf16x8 w[WR];
    auto request = [&](int s) {
        const int k = s * kPiece;
#pragma unroll
        for (int u = 0; u < XR; ++u) load_run<8>(from[u] + k, p.k - k - 8 * (int)(threadIdx.x & 3), x[u]);
#pragma unroll
        for (int u = 0; u < WR; ++u) w[u] = *reinterpret_cast<const bf16x8*>(wfrom[u] + k);
    };
    f32x4 acc[NM][NT];
#pragma unroll
    for (int i = 0; i < NM; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[i][t] = f32x4{0, 0, 0, 0};
    const int wm = wave >> 1, wn = wave & 1;
    const unsigned char* xs = lds + (wm * NM * 16 + n) * 64 + 16 * (g ^ (n >> 1 & 3));
    const unsigned char* ws = lds + 3 * BM * 64 + (wn * NT * 16 + 4 * NT * (n >> 2) + (n & 3)) * 64 + 16 * (g ^ ((n >> 1 & 1) | (n >> 2 & 1) << 1));
    const int steps = p.k_padded / kPiece;
    request(0);
    for (int s = 0; s < steps; ++s) {
        __syncthreads();      // everybody has read the step before
#pragma unroll
        for (int u = 0; u < XR; ++u) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[u][j] *= kSplitScale;
            bf16 part[3][8];
            split(x[u], part);
#pragma unroll
            for (int q = 0; q < 3; ++q) {
                bf16x8 v;
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = part[q][j];
                *reinterpret_cast<bf16x8*>(lds + q * BM * 64 + to[u]) = v;
            }
        }
#pragma unroll
        for (int u = 0; u < WR; ++u) *reinterpret_cast<bf16x8*>(lds + wto[u]) = w[u];
        __syncthreads();
        if (s + 1 < steps) request(s + 1);
        bf16x8 wf[NT][3];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int q = 0; q < 3; ++q) wf[t][q] = *reinterpret_cast<const bf16x8*>(ws + q * BN * 64 + t * 256);
#pragma unroll
        for (int i = 0; i < NM; ++i) {
            bf16x8 xf[3];
#pragma unroll
            for (int q = 0; q < 3; ++q) xf[q] = *reinterpret_cast<const bf16x8*>(xs + q * BM * 64 + i * 1024);
            constexpr int ix[6] = {2, 0, 1, 1, 0, 0}, iw[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
            for (int o = 0; o < 6; ++o)
#pragma unroll
                for (int t = 0; t < NT; ++t) acc[i][t] = mma(wf[t][iw[o]], xf[ix[o]], acc[i][t]);
        }
    }
    constexpr float kBack = 1.0f / (kSplitScale * kSplitScale);
    const long row_w = row0 + wm * NM * 16;
    const int col_w = col0 + wn * NT * 16;
#pragma unroll
    for (int i = 0; i < NM; ++i) {
        bool fine = true;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                acc[i][t][j] *= kBack;
                fine = fine && fabsf(acc[i][t][j]) <= std::numeric_limits<float>::max();
            }
        if (__builtin_expect(!fine, 0)) {
            const float* row = static_cast<const float*>(p.in) + min(row_w + 16 * i + n, p.rows - 1) * p.in_stride;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (!(fabsf(acc[i][t][j]) <= std::numeric_limits<float>::max())) {
                        const float* wc = static_cast<const float*>(p.W0) + min(col_w + 4 * NT * g + 4 * t + j, p.cols - 1) * p.w0_col;
                        float sum = 0.0f;
                        for (int k = 0; k < p.k; ++k) sum = fmaf(row[k], wc[k * p.w0_k], sum);
                        acc[i][t][j] = sum;
                    }
        }
    }
    add_adapters<float, NM, NT>(p, lane, row_w, col_w, acc);
    store_tiles<float, NM, NT>(p, lane, row_w, col_w, acc);
}

// Few rows: a block takes 16 columns and all rows; eight wavefronts have 128 bytes of W's rows by turns.
template <typename T, int MT>
__global__ __launch_bounds__(512) void k_product_few(const Product p)
{
    constexpr int V = kRun<T>, UNIT = 8 * V;
    __shared__ f32x4 part[8][MT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4, col0 = blockIdx.x * 16;
    const T* W = static_cast<const T*>(p.W0) + (long)min(col0 + n, p.cols - 1) * p.w0_col;
    const T* in[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) in[i] = static_cast<const T*>(p.in) + min(16L * i + n, p.rows - 1) * p.in_stride;
    f32x4 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = f32x4{0, 0, 0, 0};
    for (int k0 = wave * UNIT; k0 < p.k; k0 += 8 * UNIT)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int k = k0 + u * (UNIT / 2) + g * V;
            const auto w = load_operand(W + k, p.k - k);
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[i] = mma(w, load_operand(in[i] + k, p.k - k), acc[i]);
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

// ---- rows sorted by adapter, in their order: places [start[a], start[a + 1]) of perm hold adapter a's; rows with no adapter, and with an
// index out of range, come last.  Pieces of kPieceRows rows of one adapter: [first[a], first[a + 1]).

__device__ __forceinline__ int key_of(int a, int n) { return has_adapter(a, n) ? a : (a == -1 ? n : n + 1); }

struct Groups {
    const int* index;
    int adapters, blocks, rows_per_block, piece;
    long rows;
    int *count;      // [key][block], later its exclusive sums over blocks
    int *total;      // [key]
    int *start, *first;      // [adapters + 1]
    int *perm;
};
__global__ __launch_bounds__(64) void k_group_count(const Groups p)
{
    extern __shared__ int hist[];
    for (int k = threadIdx.x; k < p.adapters + 2; k += 64) hist[k] = 0;
    __syncthreads();
    const long begin = (long)blockIdx.x * p.rows_per_block, end = min(begin + p.rows_per_block, p.rows);
    for (long i = begin + threadIdx.x; i < end; i += 64) atomicAdd(&hist[key_of(p.index[i], p.adapters)], 1);
    __syncthreads();
    for (int k = threadIdx.x; k < p.adapters + 2; k += 64) p.count[(long)k * p.blocks + blockIdx.x] = hist[k];
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
__global__ __launch_bounds__(256) void k_group_scan(const Groups p)
{
    const int key = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (key >= p.adapters + 2) return;
    int run = 0;
    int* count = p.count + (long)key * p.blocks;
    for (int b = 0; b < p.blocks; b += 64) {
        int total;
        const int x = b + lane < p.blocks ? count[b + lane] : 0, before = wave_exclusive(x, lane, total);
        if (b + lane < p.blocks) count[b + lane] = run + before;
        run += total;
    }
    if (lane == 0) p.total[key] = run;
}
__global__ __launch_bounds__(64) void k_group_place(const Groups p)
{
    extern __shared__ int base[];
    const int lane = threadIdx.x, keys = p.adapters + 2;
    int rows = 0, pieces = 0;
    for (int k = 0; k < keys; k += 64) {
        int row_total, piece_total;
        const int x = k + lane < keys ? p.total[k + lane] : 0;
        const int row_before = rows + wave_exclusive(x, lane, row_total);
        const int piece_before = pieces + wave_exclusive(k + lane < p.adapters ? (x + p.piece - 1) / p.piece : 0, lane, piece_total);
        if (k + lane < keys) base[k + lane] = row_before + p.count[(long)(k + lane) * p.blocks + blockIdx.x];
        if (blockIdx.x == 0 && k + lane <= p.adapters) {
            p.start[k + lane] = row_before;
            p.first[k + lane] = piece_before;
        }
        rows += row_total;
        pieces += piece_total;
    }
    __syncthreads();
    const long begin = (long)blockIdx.x * p.rows_per_block, end = min(begin + p.rows_per_block, p.rows);
    for (long i = begin; i < end; i += 64) {
        const bool live = i + lane < end;
        const int key = live ? key_of(p.index[i + lane], p.adapters) : keys;
        unsigned long same = __ballot(live);
        for (int bit = 0; (1 << bit) <= keys; ++bit) {
            const unsigned long set = __ballot(key >> bit & 1);
            same &= key >> bit & 1 ? set : ~set;
        }
        const int before = __popcll(same & ((1ul << lane) - 1));
        int at = 0;
        if (live) at = base[key] + before;
        __syncthreads();
        if (live) {
            p.perm[at] = (int)(i + lane);
            if (before == 0) base[key] = at + __popcll(same);
        }
        __syncthreads();
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
// A block takes a piece, 64 r at most, and 64 V columns; a wavefront 16 V of them, four rows at a time.
template <typename T, int RT>
__global__ __launch_bounds__(256) void k_outer(const Outer p)
{
    constexpr int V = kRun<T>, U = 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4, item = blockIdx.x;
    if (item >= p.first[p.adapters]) return;
    int low = 0, high = p.adapters;
    while (high - low > 1) {
        const int mid = (low + high) / 2;
        if (p.first[mid] <= item) low = mid;
        else high = mid;
    }
    const int begin = p.start[low] + (item - p.first[low]) * p.piece, end = min(begin + p.piece, p.start[low + 1]);
    const int col = (blockIdx.y * 4 + wave) * 16 * V + V * n, r0 = blockIdx.z * 64;
    if ((blockIdx.y * 4 + wave) * 16 * V >= p.cols) return;
    const T* in = static_cast<const T*>(p.in) + col;
    const float* h = p.h + r0 + n;
    f32x4 acc[RT][V];
#pragma unroll
    for (int q = 0; q < RT; ++q)
#pragma unroll
        for (int t = 0; t < V; ++t) acc[q][t] = f32x4{0, 0, 0, 0};
    for (int at = begin; at < end; at += 4 * U) {
        float x[U][V], hv[U][RT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = at + 4 * u + g;
            const bool live = i < end;
            const long row = p.perm[min(i, end - 1)];
            load_run<V>(in + row * p.in_stride, live ? p.cols - col : 0, x[u]);
#pragma unroll
            for (int q = 0; q < RT; ++q) hv[u][q] = live && r0 + 16 * q + n < p.rank ? h[row * p.padded + 16 * q] : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int q = 0; q < RT; ++q)
#pragma unroll
                for (int t = 0; t < V; ++t) acc[q][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(hv[u][q], x[u][t], acc[q][t], 0, 0, 0);
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
template <typename T>
__global__ __launch_bounds__(256) void k_join(const Outer p)
{
    const int a = blockIdx.y, each = p.rank * p.cols, e = blockIdx.x * 256 + threadIdx.x;
    if (e >= each) return;
    float sum = 0.0f;
    for (int i = p.first[a]; i < p.first[a + 1]; ++i) sum += p.partial[(long)i * each + e];
    const int r = e / p.cols, col = e % p.cols;
    static_cast<T*>(p.out)[a * p.out_each + r * p.out_r + col * p.out_col] = (T)sum;
}

// ---- host side

void check(const smx_adapted_linear* p)
{
    refuse_unless(p, "the description must not be null");
    (void)type_bytes(p->type);
    refuse_unless(p->rows >= 0 && p->rows <= 0x7fffffffL - 4096, "rows: 0 to 2^31 - 4097");
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
bool as_it_is(const void* p, long stride, long k) { return (reinterpret_cast<size_t>(p) & 15) == 0 && stride % 8 == 0 && k % kPiece == 0; }

struct Call {
    const smx_adapted_linear& p;
    hipStream_t s;
    Arena arena;
    const bool dry;      // nothing is launched, the workspace is counted
    const int padded;
    Call(const smx_adapted_linear& p_, void* base, hipStream_t s_, bool dry_)
        : p(p_), s(s_), arena{static_cast<char*>(base)}, dry(dry_), padded((int)up(p_.rank, 16)) {}

    template <typename T>
    void down(const T* in, long in_stride, const T* F, long f_each, long f_row, int k, float* h, bool few)
    {
        if (dry) return;
        const Down d{in, in_stride, F, f_each, f_row, p.scale, p.index, p.num_adapters, p.rank, padded, k, p.rows, h};
        if (few) {
            hipLaunchKernelGGL((k_down_few<T>), dim3((unsigned)p.rows, padded / 4), dim3(256), 0, s, d);
            return;
        }
        const dim3 grid((unsigned)((p.rows + 15) / 16));
        auto go = [&](auto rt) { hipLaunchKernelGGL((k_down<T, decltype(rt)::value>), grid, dim3(256), 0, s, d); };
        if (padded == 16) go(std::integral_constant<int, 1>{});
        else if (padded == 32) go(std::integral_constant<int, 2>{});
        else if (padded <= 64) go(std::integral_constant<int, 4>{});
        else go(std::integral_constant<int, 8>{});
    }

    // out[rows][cols] = in W^T + adapters' part; W(col, k) = W[col * w_col + k * w_k], F(col, r) = F[a][col * f_col + r * f_r]
    template <typename T>
    void product(const T* in, long in_stride, const T* W, long w_col, long w_k, const T* F, long f_each, long f_col, long f_r, const float* h, int k, int cols,
                 T* out, long out_stride, bool few)
    {
        Product q{};
        q.in = in; q.in_stride = in_stride; q.W0 = W; q.w0_col = w_col; q.w0_k = w_k; q.F = F; q.f_each = f_each; q.f_col = f_col; q.f_r = f_r; q.h = h;
        q.index = p.index; q.adapters = p.num_adapters; q.rank = p.rank; q.padded = padded; q.k = k; q.k_padded = (int)up(k, kPiece); q.cols = cols;
        q.rows = p.rows; q.out = out; q.out_stride = out_stride;
        if (few) {
            if (dry) return;
            auto go = [&](auto mt) { hipLaunchKernelGGL((k_product_few<T, decltype(mt)::value>), dim3((cols + 15) / 16), dim3(512), 0, s, q); };
            if (p.rows <= 16) go(std::integral_constant<int, 1>{});
            else if (p.rows <= 32) go(std::integral_constant<int, 2>{});
            else go(std::integral_constant<int, 4>{});
            return;
        }
        auto tiles = [&](int bm, int bn) {
            q.row_tiles = (int)((p.rows + bm - 1) / bm);
            q.col_tiles = (cols + bn - 1) / bn;
            return (long)q.row_tiles * q.col_tiles;
        };
        auto blocks = [&] {
            const long t = (long)q.row_tiles * q.col_tiles;
            refuse_unless(t < 0x7ffffff0L / 8, "more tiles than a launch takes");
            return dim3((unsigned)((t + 7) / 8 * 8));
        };
        if constexpr (std::is_same_v<T, float>) {
            bf16* parts = arena.take<bf16>(3L * cols * q.k_padded);
            if (dry) return;
            lay_out<float, true>(Layout{W, 0, w_col, w_k, parts, 0, (long)cols * q.k_padded, cols, k, q.k_padded}, 1, s);
            q.W = parts; q.w_stride = q.k_padded; q.w_part = (long)cols * q.k_padded;
            if (tiles(128, 128) >= 256) hipLaunchKernelGGL((k_product32<4, 4>), blocks(), dim3(256), 0, s, q);
            else {
                tiles(64, 64);
                hipLaunchKernelGGL((k_product32<2, 2>), blocks(), dim3(256), 0, s, q);
            }
        } else {
            if (!(w_k == 1 && as_it_is(W, w_col, k))) {
                T* laid = arena.take<T>((long)cols * q.k_padded);
                if (!dry) lay_out<T, false>(Layout{W, 0, w_col, w_k, laid, 0, 0, cols, k, q.k_padded}, 1, s);
                q.W = laid; q.w_stride = q.k_padded;
            } else {
                q.W = W; q.w_stride = w_col;
            }
            if (!as_it_is(in, in_stride, k)) {
                T* laid = arena.take<T>(p.rows * q.k_padded);
                for (long r = 0; !dry && r < p.rows; r += 4000000)      // (the rows of a grid)
                    lay_out<T, false>(Layout{in + r * in_stride, 0, in_stride, 1, laid + r * q.k_padded, 0, 0, (int)std::min(4000000L, p.rows - r), k, q.k_padded}, 1, s);
                q.in = laid; q.in_stride = q.k_padded;
            }
            if (dry) return;
            auto go = [&](auto bm, auto bn, auto wm, auto wn) {
                constexpr int BM = decltype(bm)::value, BN = decltype(bn)::value, WM = decltype(wm)::value, WN = decltype(wn)::value;
                constexpr int bytes = 4 * (BM + BN) * 64;
                if constexpr (bytes > 64 * 1024)
                    hip_ok(hipFuncSetAttribute(reinterpret_cast<const void*>(&k_product16<T, BM, BN, WM, WN>), hipFuncAttributeMaxDynamicSharedMemorySize, bytes), "LDS");
                hipLaunchKernelGGL((k_product16<T, BM, BN, WM, WN>), blocks(), dim3(64 * WM * WN), bytes, s, q);
            };
            if (tiles(256, 256) >= 192) go(std::integral_constant<int, 256>{}, std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{}, std::integral_constant<int, 4>{});
            else if (tiles(128, 128) >= 192) go(std::integral_constant<int, 128>{}, std::integral_constant<int, 128>{}, std::integral_constant<int, 2>{}, std::integral_constant<int, 2>{});
            else {
                tiles(64, 64);
                go(std::integral_constant<int, 64>{}, std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{}, std::integral_constant<int, 2>{});
            }
        }
    }

    template <typename T>
    void forward(T* y, long y_stride)
    {
        const bool few = p.rows <= kMostFew;
        const T *x = static_cast<const T*>(p.x), *W = static_cast<const T*>(p.weight), *A = static_cast<const T*>(p.A), *B = static_cast<const T*>(p.B);
        float* h = arena.take<float>(p.rows * padded);
        down(x, p.x_stride, A, (long)p.rank * p.d_in, p.d_in, p.d_in, h, few);
        product(x, p.x_stride, W, p.weight_stride, 1, B, (long)p.rank * p.d_out, p.rank, 1, h, p.d_in, p.d_out, y, y_stride, few);
    }

    template <typename T>
    void outer(Outer q, long most, const T* in, long in_stride, const float* h, int cols, void* out, long out_each, long out_r, long out_col)
    {
        q.in = in; q.in_stride = in_stride; q.h = h; q.cols = cols; q.out = out; q.out_each = out_each; q.out_r = out_r; q.out_col = out_col;
        const int slab = 64 * kRun<T>;
        if (p.rows > 0) {
            const dim3 grid((unsigned)most, (cols + slab - 1) / slab, (p.rank + 63) / 64);
            if (padded == 16) hipLaunchKernelGGL((k_outer<T, 1>), grid, dim3(256), 0, s, q);
            else if (padded == 32) hipLaunchKernelGGL((k_outer<T, 2>), grid, dim3(256), 0, s, q);
            else hipLaunchKernelGGL((k_outer<T, 4>), grid, dim3(256), 0, s, q);
        }
        hipLaunchKernelGGL((k_join<T>), dim3((p.rank * cols + 255) / 256, p.num_adapters), dim3(256), 0, s, q);
    }

    template <typename T>
    void backward(const T* dy, long dy_stride, T* dx, long dx_stride, T* dA, T* dB)
    {
        const T *x = static_cast<const T*>(p.x), *W = static_cast<const T*>(p.weight), *A = static_cast<const T*>(p.A), *B = static_cast<const T*>(p.B);
        const long each_a = (long)p.rank * p.d_in, each_b = (long)p.rank * p.d_out;
        const int n = p.num_adapters;
        const bool sums = (dA || dB || dry) && n > 0;
        float *h = arena.take<float>(p.rows * padded), *g = arena.take<float>(p.rows * padded);
        if (p.rows > 0) {
            // B_a^T, so that sums over d_out run along rows
            const int k_padded = (int)up(p.d_out, kPiece);
            T* Bt = arena.take<T>((long)n * p.rank * k_padded);
            if (!dry && (dx || dA)) {
                if (n) lay_out<T, false>(Layout{B, each_b, 1, p.rank, Bt, (long)p.rank * k_padded, 0, p.rank, p.d_out, k_padded}, n, s);
                down(dy, dy_stride, Bt, (long)p.rank * k_padded, k_padded, p.d_out, g, false);
            }
            if (!dry && dB) down(x, p.x_stride, A, each_a, p.d_in, p.d_in, h, false);
            if (dx || dry) product(dy, dy_stride, W, 1, p.weight_stride, A, each_a, 1, p.d_in, g, p.d_out, p.d_in, dx, dx_stride, false);
        }
        if (!sums) return;
        Groups q{};
        q.index = p.index; q.adapters = n; q.rows = p.rows;
        q.rows_per_block = (int)std::max(256L, up((p.rows + 1023) / 1024, 64));
        q.blocks = (int)std::max(1L, (p.rows + q.rows_per_block - 1) / q.rows_per_block);
        q.piece = (int)std::max(64L, up((p.rows + 511) / 512, 16));
        q.count = arena.take<int>((long)(n + 2) * q.blocks);
        q.total = arena.take<int>(n + 2);
        q.start = arena.take<int>(n + 1);
        q.first = arena.take<int>(n + 1);
        q.perm = arena.take<int>(p.rows);
        const long most = std::min<long>(p.rows, p.rows / q.piece + n);      // pieces: of an adapter's rows, one that is not full
        float* partial = arena.take<float>(most * p.rank * std::max(p.d_in, p.d_out));
        if (dry) return;
        const unsigned lds = (n + 2) * sizeof(int);
        hipLaunchKernelGGL(k_group_count, dim3(q.blocks), dim3(64), lds, s, q);
        hipLaunchKernelGGL(k_group_scan, dim3((n + 2 + 3) / 4), dim3(256), 0, s, q);
        hipLaunchKernelGGL(k_group_place, dim3(q.blocks), dim3(64), lds, s, q);
        Outer o{};
        o.start = q.start; o.first = q.first; o.perm = q.perm; o.adapters = n; o.rank = p.rank; o.padded = padded; o.piece = q.piece; o.partial = partial;
        if (dA) outer(o, most, x, p.x_stride, g, p.d_in, dA, each_a, p.d_in, 1);
        if (dB) outer(o, most, dy, dy_stride, h, p.d_out, dB, each_b, 1, p.rank);
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
