// A shared projection with a low-rank adapter per row beside it, and its gradient.
//
//   y = W x + c_a B_a (A_a x)
//   g = c_a B_a^T dy:   dx = W^T dy + A_a^T g,   dA_a = sum over the adapter's rows of g x^T,   dB_a = sum of dy (c_a A_a x)^T
#include "smx_finetune.hpp"

#include <algorithm>
#include <limits>

namespace smx {

namespace {

constexpr int kGood = 0, kNone = 1, kBad = 2;
__device__ __forceinline__ int state_of(int a, int n) { return a >= 0 && a < n ? kGood : (a == -1 ? kNone : kBad); }

// out[row][r] = scale_a sum over k of in[row][k] F_a(r, k), F_a(r, k) = F[a][r * fr + k * fk]; zero for rows without an adapter.
// A block per row, a wavefront per r.
template <typename T>
__global__ __launch_bounds__(256) void k_adapter_down(const T* in, long in_stride, const T* F, long f_adapter, long fr, long fk, const float* scale,
                                                      const int* index, int n, int rank, int d, float* out)
{
    const long row = blockIdx.x;
    const int a = index[row], lane = threadIdx.x & 63;
    const bool good = state_of(a, n) == kGood;
    for (int r = threadIdx.x >> 6; r < rank; r += 4) {
        float sum = 0.0f;
        if (good)
            for (int k = lane; k < d; k += 64) sum = fmaf((float)in[row * in_stride + k], (float)F[a * f_adapter + r * fr + k * fk], sum);
        sum = group_sum<64>(sum);
        if (lane == 0) out[row * rank + r] = good ? sum * (scale ? scale[a] : 1.0f) : 0.0f;
    }
}

// out[row][col] = sum over k of in[row][k] W(col, k) + sum over r of h[row][r] F_a(col, r).  A block takes 64 rows and 64 columns.
template <typename T>
__global__ __launch_bounds__(256) void k_adapter_product(const T* in, long in_stride, const T* W, long wc, long wk, const T* F, long f_adapter, long fc, long fr,
                                                         const float* h, const int* index, int n, int rank, long rows, int d, int cols, T* out, long out_stride)
{
    __shared__ float xs[64][17], ws[64][17];
    const long row0 = (long)blockIdx.x * 64;
    const int col0 = blockIdx.y * 64, tr = threadIdx.x / 16 * 4, tc = threadIdx.x % 16 * 4;
    float acc[4][4] = {};
    for (int k0 = 0; k0 < d; k0 += 16) {
        __syncthreads();
        for (int i = threadIdx.x; i < 64 * 16; i += 256) {
            const int r = i / 16, k = i % 16;
            xs[r][k] = row0 + r < rows && k0 + k < d ? (float)in[(row0 + r) * in_stride + k0 + k] : 0.0f;
            ws[r][k] = col0 + r < cols && k0 + k < d ? (float)W[(col0 + r) * wc + (k0 + k) * wk] : 0.0f;
        }
        __syncthreads();
        for (int k = 0; k < 16; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xs[tr + i][k], ws[tc + j][k], acc[i][j]);
    }
    for (int i = 0; i < 4; ++i) {
        const long row = row0 + tr + i;
        if (row >= rows) continue;
        const int a = index[row], state = state_of(a, n);
        for (int j = 0; j < 4; ++j) {
            const int col = col0 + tc + j;
            if (col >= cols) continue;
            float sum = acc[i][j];
            if (state == kGood)
                for (int r = 0; r < rank; ++r) sum = fmaf(h[row * rank + r], (float)F[a * f_adapter + col * fc + r * fr], sum);
            out[row * out_stride + col] = state == kBad ? (T)std::numeric_limits<float>::quiet_NaN() : (T)sum;
        }
    }
}

// out[a][r * orr + col * oc] = sum over the adapter's rows of h[row][r] in[row][col].  A block takes an adapter, 64 columns and four r.
template <typename T>
__global__ __launch_bounds__(256) void k_adapter_gradient(const T* in, long in_stride, const float* h, const int* index, int rank, long rows, int cols, T* out,
                                                          long o_adapter, long orr, long oc)
{
    const int a = blockIdx.x, col = blockIdx.y * 64 + (threadIdx.x & 63), r = blockIdx.z * 4 + (threadIdx.x >> 6);
    if (col >= cols || r >= rank) return;
    float sum = 0.0f;
    for (long row = 0; row < rows; ++row)
        if (index[row] == a) sum = fmaf(h[row * rank + r], (float)in[row * in_stride + col], sum);
    out[a * o_adapter + r * orr + col * oc] = (T)sum;
}

void check(const smx_adapted_linear* p)
{
    refuse_unless(p, "the description must not be null");
    (void)type_bytes(p->type);
    refuse_unless(p->rows >= 0 && p->rows <= 0x7fffffffL, "rows: 0 to 2^31 - 1");
    refuse_unless(p->d_in >= 1 && p->d_out >= 1 && p->d_in <= (1 << 20) && p->d_out <= (1 << 20), "d_in and d_out: 1 to 2^20");
    refuse_unless(p->rank >= 1 && p->rank <= SMX_ADAPTER_MAX_RANK, "rank: 1 to 128");
    refuse_unless(p->num_adapters >= 0 && p->num_adapters <= SMX_ADAPTER_MAX_COUNT, "num_adapters: 0 to 4096");
    refuse_unless(p->x_stride >= p->d_in && p->weight_stride >= p->d_in, "strides of x and weight: at least d_in");
    refuse_unless(p->weight && (p->num_adapters == 0 || (p->A && p->B)), "weight, A and B must not be null");
    refuse_unless(p->rows == 0 || (p->x && p->index), "x and index must not be null");
}
long workspace(const smx_adapted_linear* p, bool backward) { return p->rows * p->rank * 4 * (backward ? 2 : 1); }

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
        refuse_unless(d_workspace && workspace_bytes >= workspace(p, false), "the workspace is smaller than smx_adapted_linear_workspace says");
        require_gfx950();
        const hipStream_t s = static_cast<hipStream_t>(stream);
        float* h = static_cast<float*>(d_workspace);
        with_type(p->type, [&](auto t) {
            using T = decltype(t);
            const T *x = static_cast<const T*>(p->x), *w = static_cast<const T*>(p->weight), *A = static_cast<const T*>(p->A), *B = static_cast<const T*>(p->B);
            const long each_a = (long)p->rank * p->d_in, each_b = (long)p->rank * p->d_out;
            hipLaunchKernelGGL((k_adapter_down<T>), dim3((unsigned)p->rows), dim3(256), 0, s, x, p->x_stride, A, each_a, (long)p->d_in, 1L, p->scale, p->index,
                               p->num_adapters, p->rank, p->d_in, h);
            hipLaunchKernelGGL((k_adapter_product<T>), dim3((unsigned)((p->rows + 63) / 64), (p->d_out + 63) / 64), dim3(256), 0, s, x, p->x_stride, w,
                               p->weight_stride, 1L, B, each_b, (long)p->rank, 1L, h, p->index, p->num_adapters, p->rank, p->rows, p->d_in, p->d_out,
                               static_cast<T*>(d_y), y_stride);
        });
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
        refuse_unless(p->rows == 0 || (d_workspace && workspace_bytes >= workspace(p, true)), "the workspace is smaller than smx_adapted_linear_workspace says");
        require_gfx950();
        const hipStream_t s = static_cast<hipStream_t>(stream);
        float *h = static_cast<float*>(d_workspace), *g = h + p->rows * p->rank;
        with_type(p->type, [&](auto t) {
            using T = decltype(t);
            const T *x = static_cast<const T*>(p->x), *w = static_cast<const T*>(p->weight), *A = static_cast<const T*>(p->A), *B = static_cast<const T*>(p->B);
            const T* dy = static_cast<const T*>(d_dy);
            const long each_a = (long)p->rank * p->d_in, each_b = (long)p->rank * p->d_out;
            const int n = p->num_adapters, rank = p->rank;
            if (p->rows > 0) {
                hipLaunchKernelGGL((k_adapter_down<T>), dim3((unsigned)p->rows), dim3(256), 0, s, x, p->x_stride, A, each_a, (long)p->d_in, 1L, p->scale, p->index, n,
                                   rank, p->d_in, h);
                hipLaunchKernelGGL((k_adapter_down<T>), dim3((unsigned)p->rows), dim3(256), 0, s, dy, dy_stride, B, each_b, 1L, (long)rank, p->scale, p->index, n, rank,
                                   p->d_out, g);
                if (d_dx)
                    hipLaunchKernelGGL((k_adapter_product<T>), dim3((unsigned)((p->rows + 63) / 64), (p->d_in + 63) / 64), dim3(256), 0, s, dy, dy_stride, w, 1L,
                                       p->weight_stride, A, each_a, 1L, (long)p->d_in, g, p->index, n, rank, p->rows, p->d_out, p->d_in, static_cast<T*>(d_dx), dx_stride);
            }
            const unsigned rz = (rank + 3) / 4;
            if (d_dA && n)
                hipLaunchKernelGGL((k_adapter_gradient<T>), dim3(n, (p->d_in + 63) / 64, rz), dim3(256), 0, s, x, p->x_stride, g, p->index, rank, p->rows, p->d_in,
                                   static_cast<T*>(d_dA), each_a, (long)p->d_in, 1L);
            if (d_dB && n)
                hipLaunchKernelGGL((k_adapter_gradient<T>), dim3(n, (p->d_out + 63) / 64, rz), dim3(256), 0, s, dy, dy_stride, h, p->index, rank, p->rows, p->d_out,
                                   static_cast<T*>(d_dB), each_b, 1L, (long)rank);
        });
        hip_ok(hipGetLastError(), "launch");
    });
}
