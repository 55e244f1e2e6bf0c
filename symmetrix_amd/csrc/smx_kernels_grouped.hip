// A product with a matrix of the row's own group, and its gradient.
//
//   y_i = W_g x_i + b_g,   dx_i = W_g^T dy_i,   dW_g = sum over the group's rows of dy_i x_i^T,   db_g = sum of dy_i
//
// Rows are taken in the order of their groups; a tile has rows of one group.
#include "smx_groups.hpp"

#include <limits>

namespace smx {

namespace {

// C(m, c) = sum over k of A(m, k) B(k, c) for the rows of a group
struct Product {
    const void* a;             // x or dy
    long a_stride;
    const void* b;             // the weights, or x for their gradient
    long b_each, b_k, b_c;
    const void* bias;          // [group][cols] or null
    const int *order, *offsets;
    int groups, k, cols;
    long rows;
    void* out;
    long out_stride;
};

// item -> group and its tile, where a group has ceil(rows / high) of them; false behind the last
__device__ __forceinline__ bool tile_of(const int* offsets, int groups, long rows, int item, int high, int& group, int& tile)
{
    for (int g = 0; g < groups + 2; ++g) {
        const int n = (int)((g == groups + 1 ? rows : offsets[g + 1]) - offsets[g]), tiles = (n + high - 1) / high;
        if (item < tiles) {
            group = g;
            tile = item;
            return true;
        }
        item -= tiles;
    }
    return false;
}

template <typename T>
__global__ __launch_bounds__(256) void k_rows(const Product p)
{
    __shared__ float as[16][65], bs[16][65];
    int g, tile;
    if (!tile_of(p.offsets, p.groups, p.rows, blockIdx.x, 64, g, tile)) return;
    const int begin = p.offsets[g] + 64 * tile, end = min((long)begin + 64, g == p.groups + 1 ? p.rows : (long)p.offsets[g + 1]), col0 = blockIdx.y * 64;
    const int tm = threadIdx.x / 16 * 4, tc = threadIdx.x % 16 * 4;
    float acc[4][4] = {};
    const bool real = g < p.groups;
    for (int k0 = 0; real && k0 < p.k; k0 += 16) {
        for (int u = threadIdx.x; u < 1024; u += 256) {
            const int m = u / 16, k = u % 16;
            as[k][m] = begin + m < end && k0 + k < p.k ? (float)static_cast<const T*>(p.a)[p.order[begin + m] * p.a_stride + k0 + k] : 0.0f;
            bs[k][m] = col0 + m < p.cols && k0 + k < p.k ? (float)static_cast<const T*>(p.b)[g * p.b_each + (k0 + k) * p.b_k + (col0 + m) * p.b_c] : 0.0f;
        }
        __syncthreads();
        for (int k = 0; k < 16; ++k)
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(as[k][tm + i], bs[k][tc + j], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            if (begin + tm + i >= end || col0 + tc + j >= p.cols) continue;
            float v = acc[i][j];
            if (real && p.bias) v += (float)static_cast<const T*>(p.bias)[(long)g * p.cols + col0 + tc + j];
            if (g == p.groups + 1) v = std::numeric_limits<float>::quiet_NaN();
            static_cast<T*>(p.out)[p.order[begin + tm + i] * p.out_stride + col0 + tc + j] = (T)v;
        }
}

// dW: m over columns of a (dy), k over the group's rows, c over columns of b (x)
template <typename T>
__global__ __launch_bounds__(256) void k_weights(const Product p)
{
    __shared__ float as[16][65], bs[16][65];
    const int g = blockIdx.z, begin = p.offsets[g], end = p.offsets[g + 1], m0 = blockIdx.x * 64, col0 = blockIdx.y * 64;
    const int tm = threadIdx.x / 16 * 4, tc = threadIdx.x % 16 * 4;
    float acc[4][4] = {};
    for (int k0 = begin; k0 < end; k0 += 16) {
        for (int u = threadIdx.x; u < 1024; u += 256) {
            const int m = u % 64, k = u / 64;
            const long row = p.order[min(k0 + k, end - 1)];
            as[k][m] = m0 + m < p.k && k0 + k < end ? (float)static_cast<const T*>(p.a)[row * p.a_stride + m0 + m] : 0.0f;
            bs[k][m] = col0 + m < p.cols && k0 + k < end ? (float)static_cast<const T*>(p.b)[row * p.b_k + col0 + m] : 0.0f;
        }
        __syncthreads();
        for (int k = 0; k < 16; ++k)
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(as[k][tm + i], bs[k][tc + j], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j)
            if (m0 + tm + i < p.k && col0 + tc + j < p.cols) static_cast<T*>(p.out)[((long)g * p.k + m0 + tm + i) * p.cols + col0 + tc + j] = (T)acc[i][j];
}
// db
template <typename T>
__global__ __launch_bounds__(256) void k_biases(const Product p)
{
    const int g = blockIdx.y, m = blockIdx.x * 256 + threadIdx.x;
    if (m >= p.k) return;
    float sum = 0.0f;
    for (int i = p.offsets[g]; i < p.offsets[g + 1]; ++i) sum += (float)static_cast<const T*>(p.a)[p.order[i] * p.a_stride + m];
    static_cast<T*>(p.out)[(long)g * p.k + m] = (T)sum;
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
    template <typename T>
    void rows(const T* a, long a_stride, long b_k, long b_c, const T* bias, int k, int cols, T* out, long out_stride)
    {
        Product q{a, a_stride, p.weight, p.weight_each, b_k, b_c, bias, groups.order, groups.offsets, p.num_groups, k, cols, p.rows, out, out_stride};
        start(k_rows<T>, (p.rows + 63) / 64 + p.num_groups + 2, (cols + 63) / 64, 1, 256, 0, q);
    }
    template <typename T>
    void forward(T* y, long y_stride)
    {
        sort();
        rows<T>(static_cast<const T*>(p.x), p.x_stride, 1, p.weight_stride, static_cast<const T*>(p.bias), p.d_in, p.d_out, y, y_stride);
    }
    template <typename T>
    void backward(const T* dy, long dy_stride, T* dx, long dx_stride, T* dW, T* db)
    {
        sort();
        if (dx && p.rows) rows<T>(dy, dy_stride, p.weight_stride, 1, nullptr, p.d_out, p.d_in, dx, dx_stride);
        if (!p.num_groups) return;
        Product q{dy, dy_stride, p.x, 0, p.x_stride, 1, nullptr, groups.order, groups.offsets, p.num_groups, p.d_out, p.d_in, p.rows, dW, 0};
        if (dW) start(k_weights<T>, (p.d_out + 63) / 64, (p.d_in + 63) / 64, p.num_groups, 256, 0, q);
        q.out = db;
        if (db) start(k_biases<T>, (p.d_out + 255) / 256, p.num_groups, 1, 256, 0, q);
    }
};

long workspace(const smx_grouped_linear* p, bool backward)
{
    Call c{{nullptr, true}, *p, {reinterpret_cast<char*>(256)}};
    with_type(p->type, [&](auto t) {
        using T = decltype(t);
        T* some = reinterpret_cast<T*>(256);
        if (backward) c.backward<T>(some, p->d_out, some, p->d_in, some, some);
        else if (p->rows > 0) c.forward<T>(some, p->d_out);
    });
    return c.arena.used;
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
