// Layer norm over the features of a row and its gradient.
//
//   mean = sum x / D,  var = sum (x - mean)^2 / D,  rstd = 1 / sqrt(var + eps),  y = (x - mean) rstd w + b
//   xh = (x - mean) rstd,  g = dy w:   dx = rstd (g - mean(g) - xh mean(g xh)),   dw = sum over rows of dy xh,   db = sum over rows of dy
//
// A row lies in the registers of a group of lanes, or of a block, between its sums and its output, so that memory is read once;
// the variance is summed from centered values.  All sums are in single precision.
//
// What bounds it is memory: forward 55 us for 16 381 rows of 4 096 numbers in bfloat16 (268 MB, 4.9 TB/s), gradient 33 us a call for
// 50 000 rows of 256 in single precision (154 MB, 4.7 TB/s with the joining of the parts); a few rows cost a launch, 10 us a call.
#include "smx_finetune.hpp"

#include <algorithm>

namespace smx {

namespace {

struct NormForward {
    long rows, x_stride, y_stride;
    int dim;
    float eps;
    const void *x, *weight, *bias;
    void* y;
    float *mean, *rstd;
};
struct NormBackward {
    long rows, dy_stride, x_stride, dx_stride;
    int dim;
    const void *dy, *x, *weight;
    const float *mean, *rstd;
    void *dx;
    float* partial;      // [blocks][2][dim]: sums over a block's rows of dy xh and dy (null: not wanted)
};

// sum over the threads that share a row: G lanes, or WAVES wavefronts
template <int G, int WAVES>
__device__ __forceinline__ float row_sum(float x, float* place)
{
    x = group_sum<(WAVES > 1 ? 64 : G)>(x);
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & 63) == 0) place[threadIdx.x >> 6] = x;
        __syncthreads();
        x = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) x += place[w];
    }
    return x;
}

// G lanes (WAVES == 1) or WAVES wavefronts share a row; a thread has NV runs of V numbers of it, run u the one at (u * threads + thread) * V.
template <typename T, typename TW, int V, int NV, int G, int WAVES>
__global__ __launch_bounds__(256) void k_norm_fwd(const NormForward p)
{
    constexpr int SHARE = WAVES > 1 ? 64 * WAVES : G, PER = 256 / SHARE;
    __shared__ float place[2][4];
    const int t = threadIdx.x % SHARE;
    const long row = (long)blockIdx.x * PER + threadIdx.x / SHARE;
    if (row >= p.rows) return;      // (whole blocks where a block shares a row)
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    float v[NV][V];
    float sum = 0.0f;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        const int at = (u * SHARE + t) * V;
        load_run<V>(x + at, p.dim - at, v[u]);
    }
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
        for (int j = 0; j < V; ++j) sum += v[u][j];
    const float dim = (float)p.dim;
    const float mean = row_sum<G, WAVES>(sum, place[0]) / dim;
    float square = 0.0f;
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
        for (int j = 0; j < V; ++j) {
            v[u][j] -= mean;
            if ((u * SHARE + t) * V + j < p.dim) square = fmaf(v[u][j], v[u][j], square);
        }
    const float var = row_sum<G, WAVES>(square, place[1]) / dim;
    const float rstd = 1.0f / sqrtf(var + p.eps);
    T* y = static_cast<T*>(p.y) + row * p.y_stride;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        const int at = (u * SHARE + t) * V;
        float w[V], b[V];
        if (p.weight) load_run<V>(static_cast<const TW*>(p.weight) + at, p.dim - at, w);
        if (p.bias) load_run<V>(static_cast<const TW*>(p.bias) + at, p.dim - at, b);
#pragma unroll
        for (int j = 0; j < V; ++j) v[u][j] = fmaf(v[u][j] * rstd, p.weight ? w[j] : 1.0f, p.bias ? b[j] : 0.0f);
        store_run<V>(y + at, p.dim - at, v[u]);
    }
    if (t == 0) {
        if (p.mean) p.mean[row] = mean;
        if (p.rstd) p.rstd[row] = rstd;
    }
}

// Rows longer than the registers of a block: the row is read three times, from the caches after the first.
template <typename T, typename TW>
__global__ __launch_bounds__(256) void k_norm_fwd_long(const NormForward p)
{
    constexpr int V = kRun<T>;
    __shared__ float place[2][4];
    const long row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    float sum = 0.0f, square = 0.0f, v[V];
    for (int at = threadIdx.x * V; at < p.dim; at += 256 * V) {
        load_run<V>(x + at, p.dim - at, v);
#pragma unroll
        for (int j = 0; j < V; ++j) sum += v[j];
    }
    const float dim = (float)p.dim;
    const float mean = row_sum<64, 4>(sum, place[0]) / dim;
    for (int at = threadIdx.x * V; at < p.dim; at += 256 * V) {
        load_run<V>(x + at, p.dim - at, v);
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (at + j < p.dim) square = fmaf(v[j] - mean, v[j] - mean, square);
    }
    const float var = row_sum<64, 4>(square, place[1]) / dim;
    const float rstd = 1.0f / sqrtf(var + p.eps);
    T* y = static_cast<T*>(p.y) + row * p.y_stride;
    for (int at = threadIdx.x * V; at < p.dim; at += 256 * V) {
        float w[V], b[V];
        load_run<V>(x + at, p.dim - at, v);
        if (p.weight) load_run<V>(static_cast<const TW*>(p.weight) + at, p.dim - at, w);
        if (p.bias) load_run<V>(static_cast<const TW*>(p.bias) + at, p.dim - at, b);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = fmaf((v[j] - mean) * rstd, p.weight ? w[j] : 1.0f, p.bias ? b[j] : 0.0f);
        store_run<V>(y + at, p.dim - at, v);
    }
    if (threadIdx.x == 0) {
        if (p.mean) p.mean[row] = mean;
        if (p.rstd) p.rstd[row] = rstd;
    }
}

// A block takes rows blockIdx.x * PER, + gridDim.x * PER, ...; a thread has the same columns of all of them, and adds up what they give
// to the gradients of weight and bias.
template <typename T, typename TW, int V, int NV, int G, int WAVES>
__global__ __launch_bounds__(256) void k_norm_bwd(const NormBackward p)
{
    constexpr int SHARE = WAVES > 1 ? 64 * WAVES : G, PER = 256 / SHARE;
    __shared__ float place[4][4];
    const int t = threadIdx.x % SHARE;
    float w[NV][V], dw[NV][V], db[NV][V];
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        const int at = (u * SHARE + t) * V;
        if (p.weight) load_run<V>(static_cast<const TW*>(p.weight) + at, p.dim - at, w[u]);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (!p.weight) w[u][j] = 1.0f;
            dw[u][j] = 0.0f; db[u][j] = 0.0f;
        }
    }
    const float dim = (float)p.dim;
    int turn = 0;
    for (long row = (long)blockIdx.x * PER + threadIdx.x / SHARE; row < p.rows; row += (long)gridDim.x * PER) {
        const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
        const T* dy = static_cast<const T*>(p.dy) + row * p.dy_stride;
        float xh[NV][V], g[NV][V];
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const int at = (u * SHARE + t) * V;
            load_run<V>(x + at, p.dim - at, xh[u]);
            load_run<V>(dy + at, p.dim - at, g[u]);
        }
        const float mean = p.mean[row], rstd = p.rstd[row];
        float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
        for (int u = 0; u < NV; ++u)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                // (behind the row's end g is zero, and an infinite or NaN statistic has no say there: nothing of it is stored)
                xh[u][j] = (xh[u][j] - mean) * rstd;
                db[u][j] += g[u][j];
                dw[u][j] = fmaf(g[u][j], xh[u][j], dw[u][j]);
                g[u][j] *= w[u][j];
                if ((u * SHARE + t) * V + j < p.dim) {
                    s0 += g[u][j];
                    s1 = fmaf(g[u][j], xh[u][j], s1);
                }
            }
        // (two places by turns: a wavefront may be one row ahead of those that still read)
        s0 = row_sum<G, WAVES>(s0, place[turn]) / dim;
        s1 = row_sum<G, WAVES>(s1, place[turn + 1]) / dim;
        turn ^= 2;
        if (p.dx) {
            T* dx = static_cast<T*>(p.dx) + row * p.dx_stride;
#pragma unroll
            for (int u = 0; u < NV; ++u) {
                const int at = (u * SHARE + t) * V;
#pragma unroll
                for (int j = 0; j < V; ++j) g[u][j] = rstd * (g[u][j] - fmaf(xh[u][j], s1, s0));
                store_run<V>(dx + at, p.dim - at, g[u]);
            }
        }
    }
    if (!p.partial) return;
    float* out = p.partial + (size_t)blockIdx.x * 2 * p.dim;
    if constexpr (PER == 1) {
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const int at = (u * SHARE + t) * V;
            store_run<V>(out + at, p.dim - at, dw[u]);
            store_run<V>(out + p.dim + at, p.dim - at, db[u]);
        }
    } else {
        // the groups of a block, in order
        __shared__ float part[PER][2][SHARE][V];
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < V; ++j) {
                part[threadIdx.x / SHARE][0][t][j] = dw[u][j];
                part[threadIdx.x / SHARE][1][t][j] = db[u][j];
            }
            __syncthreads();
            for (int i = threadIdx.x; i < 2 * SHARE * V; i += 256) {
                const int which = i / (SHARE * V), c = i % (SHARE * V), at = u * SHARE * V + c;
                float sum = 0.0f;
#pragma unroll
                for (int q = 0; q < PER; ++q) sum += part[q][which][c / V][c % V];
                if (at < p.dim) out[which * p.dim + at] = sum;
            }
        }
    }
}

// Rows longer than the registers of a block: dx, a block per row.
template <typename T, typename TW>
__global__ __launch_bounds__(256) void k_norm_bwd_long(const NormBackward p)
{
    constexpr int V = kRun<T>;
    __shared__ float place[2][4];
    const long row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    const T* dy = static_cast<const T*>(p.dy) + row * p.dy_stride;
    const float mean = p.mean[row], rstd = p.rstd[row], dim = (float)p.dim;
    float s0 = 0.0f, s1 = 0.0f, xv[V], g[V], w[V];
#pragma unroll
    for (int j = 0; j < V; ++j) w[j] = 1.0f;
    for (int at = threadIdx.x * V; at < p.dim; at += 256 * V) {
        load_run<V>(x + at, p.dim - at, xv);
        load_run<V>(dy + at, p.dim - at, g);
        if (p.weight) load_run<V>(static_cast<const TW*>(p.weight) + at, p.dim - at, w);
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (at + j < p.dim) {
                s0 = fmaf(g[j], w[j], s0);
                s1 = fmaf(g[j] * w[j], (xv[j] - mean) * rstd, s1);
            }
    }
    s0 = row_sum<64, 4>(s0, place[0]) / dim;
    s1 = row_sum<64, 4>(s1, place[1]) / dim;
    T* dx = static_cast<T*>(p.dx) + row * p.dx_stride;
    for (int at = threadIdx.x * V; at < p.dim; at += 256 * V) {
        load_run<V>(x + at, p.dim - at, xv);
        load_run<V>(dy + at, p.dim - at, g);
        if (p.weight) load_run<V>(static_cast<const TW*>(p.weight) + at, p.dim - at, w);
#pragma unroll
        for (int j = 0; j < V; ++j) g[j] = rstd * (g[j] * w[j] - fmaf((xv[j] - mean) * rstd, s1, s0));
        store_run<V>(dx + at, p.dim - at, g);
    }
}
// ... and what they give to the gradients of weight and bias: a block takes 256 columns and every gridDim.y-th row.
template <typename T>
__global__ __launch_bounds__(256) void k_norm_bwd_columns(const NormBackward p)
{
    const int col = blockIdx.x * 256 + threadIdx.x;
    if (col >= p.dim) return;
    float dw = 0.0f, db = 0.0f;
    for (long row = blockIdx.y; row < p.rows; row += gridDim.y) {
        const float g = (float)static_cast<const T*>(p.dy)[row * p.dy_stride + col];
        const float xh = ((float)static_cast<const T*>(p.x)[row * p.x_stride + col] - p.mean[row]) * p.rstd[row];
        dw = fmaf(g, xh, dw);
        db += g;
    }
    float* out = p.partial + (size_t)blockIdx.y * 2 * p.dim;
    out[col] = dw;
    out[p.dim + col] = db;
}

// Sums of the blocks' parts, in order: a block takes 16 columns, 64 threads a column.  (16 threads with a load at a time: 21 us for 1 024
// parts of 512 columns, as long as the kernel that makes them.)
template <typename TW>
__global__ __launch_bounds__(1024) void k_norm_join(const float* partial, int parts, int dim, TW* dweight, TW* dbias)
{
    constexpr int Q = 64;
    __shared__ float sums[Q][17];
    const int c = threadIdx.x % 16, q = threadIdx.x / 16, col = blockIdx.x * 16 + c;
    float sum = 0.0f;
    if (col < 2 * dim)
#pragma unroll 8
        for (int i = q; i < parts; i += Q) sum += partial[(size_t)i * 2 * dim + col];
    sums[q][c] = sum;
    __syncthreads();
    if (q == 0 && col < 2 * dim) {
        sum = 0.0f;
#pragma unroll
        for (int i = 0; i < Q; ++i) sum += sums[i][c];
        TW* out = col < dim ? dweight : dbias;
        if (out) out[col < dim ? col : col - dim] = (TW)sum;
    }
}

constexpr long kMostDim = 1L << 24;      // of a row
constexpr long kMostRows = 0x7fffffffL;
constexpr long kMostBlocks = 1L << 22;      // of a launch, which takes fewer than 2^32 threads

constexpr long kMostHeld = 256 * 32;       // numbers of a row that a block holds in registers

// how many blocks add up parts of the gradients of weight and bias
long parts_of(long rows, long dim)
{
    if (rows == 0) return 0;
    if (dim > kMostHeld) return std::min<long>(rows, 64);
    const long per = dim <= 64 * 16 ? 4 : 1;
    return std::min<long>((rows + per - 1) / per, 1024);
}

// fn(V, NV, G, WAVES) as integral constants: how a row of dim numbers is shared.  The fewest lanes that hold it with 16 bytes each, then more
// bytes a lane and last four wavefronts: sums inside a wavefront need no barrier, and no lane is without work while others have two runs.
template <typename T, typename Fn>
void shared_rows(int dim, Fn&& fn)
{
    constexpr int V = kRun<T>;
#define SMX_SHARE(NV, G, WAVES) fn(std::integral_constant<int, V>{}, std::integral_constant<int, NV>{}, std::integral_constant<int, G>{}, std::integral_constant<int, WAVES>{})
    const int runs = (dim + V - 1) / V;
    if (runs <= 8) SMX_SHARE(1, 8, 1);
    else if (runs <= 16) SMX_SHARE(1, 16, 1);
    else if (runs <= 32) SMX_SHARE(1, 32, 1);
    else if (runs <= 64) SMX_SHARE(1, 64, 1);
    else if (runs <= 128) SMX_SHARE(2, 64, 1);
    else if (V == 4 && runs <= 256) SMX_SHARE(4, 64, 1);
    else if (runs <= 256) SMX_SHARE(1, 64, 4);
    else if (runs <= 512) SMX_SHARE(2, 64, 4);
    else if (runs <= 1024) SMX_SHARE(4, 64, 4);
    else if constexpr (V == 4) SMX_SHARE(8, 64, 4);
#undef SMX_SHARE
}

void check_common(long rows, long dim, int type, int weight_type)
{
    refuse_unless(rows >= 0 && rows <= kMostRows, "rows: 0 to 2^31 - 1");
    refuse_unless(dim >= 1 && dim <= kMostDim, "dim: 1 to 2^24");
    (void)type_bytes(type);
    refuse_unless(weight_type == type || weight_type == SMX_TYPE_F32, "weight and bias: the features' type or single precision");
}

}  // namespace

}  // namespace smx

using namespace smx;

extern "C" int smx_layer_norm_forward(int type, int weight_type, long rows, long dim, const void* d_x, long x_stride, const void* d_weight,
                                      const void* d_bias, double eps, void* d_y, long y_stride, float* d_mean, float* d_rstd, void* stream)
{
    return finetune_entry("smx_layer_norm_forward", [&] {
        check_common(rows, dim, type, weight_type);
        refuse_unless(eps >= 0 && eps < 1e30, "eps: a number from 0 on");
        refuse_unless(x_stride >= dim && y_stride >= dim, "strides: at least dim");
        if (rows == 0) return;
        refuse_unless(d_x && d_y, "x and y must not be null");
        require_gfx950();
        const hipStream_t s = static_cast<hipStream_t>(stream);
        NormForward p{rows, x_stride, y_stride, (int)dim, (float)eps, d_x, d_weight, d_bias, d_y, d_mean, d_rstd};
        with_type(type, [&](auto t) {
            using T = decltype(t);
            // fn(blocks) for as many rows at a time as kMostBlocks blocks take, of `per` rows each
            auto in_slabs = [&](long per, auto&& fn) {
                for (long left = rows; left > 0; left -= p.rows) {
                    p.rows = std::min(left, per * kMostBlocks);
                    fn(dim3((unsigned)((p.rows + per - 1) / per)));
                    p.x = static_cast<const T*>(p.x) + p.rows * x_stride;
                    p.y = static_cast<T*>(p.y) + p.rows * y_stride;
                    if (p.mean) p.mean += p.rows;
                    if (p.rstd) p.rstd += p.rows;
                }
            };
            auto go = [&](auto tw) {
                using TW = decltype(tw);
                if (dim > kMostHeld) {
                    in_slabs(1, [&](dim3 blocks) { hipLaunchKernelGGL((k_norm_fwd_long<T, TW>), blocks, dim3(256), 0, s, p); });
                    return;
                }
                shared_rows<T>((int)dim, [&](auto v, auto nv, auto g, auto waves) {
                    constexpr int V = decltype(v)::value, NV = decltype(nv)::value, G = decltype(g)::value, WAVES = decltype(waves)::value;
                    in_slabs(WAVES > 1 ? 1 : 256 / G, [&](dim3 blocks) { hipLaunchKernelGGL((k_norm_fwd<T, TW, V, NV, G, WAVES>), blocks, dim3(256), 0, s, p); });
                });
            };
            if (weight_type == type) go(T{});
            else go(float{});
        });
        hip_ok(hipGetLastError(), "launch");
    });
}

extern "C" int smx_layer_norm_backward_workspace(long rows, long dim, long* bytes)
{
    return finetune_entry("smx_layer_norm_backward_workspace", [&] {
        check_common(rows, dim, SMX_TYPE_F32, SMX_TYPE_F32);
        refuse_unless(bytes, "bytes must not be null");
        *bytes = parts_of(rows, dim) * 2 * dim * (long)sizeof(float);
    });
}

extern "C" int smx_layer_norm_backward(int type, int weight_type, long rows, long dim, const void* d_dy, long dy_stride, const void* d_x,
                                       long x_stride, const float* d_mean, const float* d_rstd, const void* d_weight, void* d_dx,
                                       long dx_stride, void* d_dweight, void* d_dbias, void* d_workspace, long workspace_bytes, void* stream)
{
    return finetune_entry("smx_layer_norm_backward", [&] {
        check_common(rows, dim, type, weight_type);
        refuse_unless(dy_stride >= dim && x_stride >= dim && (dx_stride >= dim || !d_dx), "strides: at least dim");
        const bool sums = d_dweight || d_dbias;
        refuse_unless(rows == 0 || (d_dy && d_x && d_mean && d_rstd), "dy, x, mean and rstd must not be null");
        const long parts = sums ? parts_of(rows, dim) : 0;
        refuse_unless(parts == 0 || (d_workspace && workspace_bytes >= parts * 2 * dim * (long)sizeof(float)),
                      "the workspace is smaller than smx_layer_norm_backward_workspace says");
        if (!sums && (rows == 0 || !d_dx)) return;
        require_gfx950();
        const hipStream_t s = static_cast<hipStream_t>(stream);
        const NormBackward p{rows, dy_stride, x_stride, dx_stride, (int)dim, d_dy, d_x, d_weight, d_mean, d_rstd, d_dx,
                             sums ? static_cast<float*>(d_workspace) : nullptr};
        with_type(type, [&](auto t) {
            using T = decltype(t);
            auto go = [&](auto tw) {
                using TW = decltype(tw);
                if (rows > 0 && dim > kMostHeld) {
                    refuse_unless(rows < 1L << 24, "more rows than a launch takes");      // (of more than 8 192 numbers)
                    if (d_dx) hipLaunchKernelGGL((k_norm_bwd_long<T, TW>), dim3((unsigned)rows), dim3(256), 0, s, p);
                    if (sums) hipLaunchKernelGGL((k_norm_bwd_columns<T>), dim3((unsigned)((dim + 255) / 256), (unsigned)parts), dim3(256), 0, s, p);
                } else if (rows > 0) {
                    shared_rows<T>((int)dim, [&](auto v, auto nv, auto g, auto waves) {
                        constexpr int PER = decltype(waves)::value > 1 ? 1 : 256 / decltype(g)::value;
                        const long blocks = sums ? parts : std::min<long>((rows + PER - 1) / PER, 4096);
                        hipLaunchKernelGGL((k_norm_bwd<T, TW, decltype(v)::value, decltype(nv)::value, decltype(g)::value, decltype(waves)::value>),
                                           dim3((unsigned)blocks), dim3(256), 0, s, p);
                    });
                }
                hip_ok(hipGetLastError(), "launch");
                if (sums)
                    hipLaunchKernelGGL((k_norm_join<TW>), dim3((unsigned)((2 * dim + 15) / 16)), dim3(1024), 0, s, static_cast<const float*>(d_workspace),
                                       (int)parts, (int)dim, static_cast<TW*>(d_dweight), static_cast<TW*>(d_dbias));
            };
            if (weight_type == type) go(T{});
            else go(float{});
        });
        hip_ok(hipGetLastError(), "launch");
    });
}
