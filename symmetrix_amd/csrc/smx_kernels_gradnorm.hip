// The norm of many tensors' numbers together, and the tensors brought to a norm at most as large as given.
//
//   norm = sqrt(sum g^2),   out = g min(1, max_norm / norm)
//
// Squares are formed and added in double precision: a product of two single-precision numbers is exact in it, and neither overflows
// nor vanishes.  A block sums neighbouring chunks and leaves one number; whoever needs the norm adds these numbers, at most about 1 024, in a
// fixed order.  That is the launch that writes the norm, or every block of the launch that clips, by itself.
//
// Bound by memory: 150 million numbers in bfloat16 are read for the norm in 47 us, 6.4 TB/s, and read and written clipped in 100, 6.0 TB/s.
#include "smx_finetune.hpp"

#include <algorithm>
#include <cmath>
#include <vector>

namespace smx {

namespace {

constexpr int kTensors = 96;         // of a launch: their descriptions are kernel arguments
constexpr int kChunkBytes = 16384;   // that a block takes at a time, the next ones on their way meanwhile
constexpr int kMostParts = SMX_GRAD_NORM_PARTS;     // blocks, four for every CU

struct NormTable {
    smx_grad_tensor tensor[kTensors];
    int first[kTensors + 1];         // chunks in front of each
    int count;
    double* part;                    // of the launch's blocks
};
static_assert(sizeof(NormTable) <= 4096, "kernel arguments");

__host__ __device__ __forceinline__ long chunk_numbers(int type) { return kChunkBytes / (type == SMX_TYPE_F32 ? 4 : 2); }

// sum over a block of 256, the same in all threads, in a fixed order
__device__ __forceinline__ double block_total(double x, double* lds)
{
#pragma unroll
    for (int d = 1; d < 64; d *= 2) x += __shfl_xor(x, d, 64);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 loose_u32x4 __attribute__((aligned(2)));
constexpr int kSteps = kChunkBytes / (256 * 16);
// 16 bytes a thread, kSteps times, of a chunk that is whole
struct Raw {
    u32x4 v[kSteps];
};
template <typename T>
__device__ __forceinline__ void numbers_of(const u32x4& raw, float (&v)[kRun<T>])
{
    const typename Operand<T>::type x = __builtin_bit_cast(typename Operand<T>::type, raw);
#pragma unroll
    for (int j = 0; j < kRun<T>; ++j) v[j] = (float)x[j];
}

// A block's chunks, neighbours: forwards or backwards, fn(tensor, base, whether it is whole, raw if it is).
template <bool BACKWARDS, typename Fn>
__device__ __forceinline__ void each_chunk(const NormTable& a, Fn&& fn)
{
    const int chunks = a.first[a.count];
    int chunk = (int)((long)chunks * blockIdx.x / gridDim.x), end = (int)((long)chunks * (blockIdx.x + 1) / gridDim.x);
    if (chunk >= end) return;
    int step = 1;
    if constexpr (BACKWARDS) {
        const int last = end - 1;
        end = chunk - 1;
        chunk = last;
        step = -1;
    }
    int low = 0, high = a.count;      // the tensor of the first (the same in all lanes)
    while (high - low > 1) {
        const int mid = (low + high) / 2;
        if (a.first[mid] <= chunk) low = mid;
        else high = mid;
    }
    struct At {
        int tensor;
        long base;
        bool whole;
    };
    auto place = [&](int c, int i) {
        if constexpr (BACKWARDS) {
            while (a.first[i] > c) --i;
        } else {
            while (a.first[i + 1] <= c) ++i;
        }
        const long n = chunk_numbers(a.tensor[i].type), base = (c - a.first[i]) * n;
        return At{i, base, base + n <= a.tensor[i].numel};
    };
    auto fetch = [&](const At& at, Raw& raw) {
        if (!at.whole) return;
        const char* from = static_cast<const char*>(a.tensor[at.tensor].grad) + at.base * (a.tensor[at.tensor].type == SMX_TYPE_F32 ? 4 : 2) + threadIdx.x * 16;
#pragma unroll
        for (int u = 0; u < kSteps; ++u) raw.v[u] = *reinterpret_cast<const loose_u32x4*>(from + u * 4096);
        asm volatile("" ::: "memory");      // (asked for here, not where they are used)
    };
    At now = place(chunk, low);
    Raw raw, next;
    fetch(now, raw);
    for (;;) {
        At then = now;
        const bool more = chunk + step != end;
        if (more) {
            then = place(chunk + step, now.tensor);
            fetch(then, next);
        }
        fn(a.tensor[now.tensor], now.base, now.whole, raw);
        if (!more) return;
        chunk += step;
        now = then;
        raw = next;
    }
}

template <typename T>
__device__ __forceinline__ double chunk_squares(const smx_grad_tensor& t, long base, bool whole, const Raw& raw)
{
    constexpr int V = kRun<T>;
    double sum[4] = {0.0, 0.0, 0.0, 0.0};
    float v[V];
    auto add = [&] {
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j % 4] = fma((double)v[j], (double)v[j], sum[j % 4]);
    };
    if (whole) {
#pragma unroll
        for (int u = 0; u < kSteps; ++u) {
            numbers_of<T>(raw.v[u], v);
            add();
        }
    } else {
        const long left = t.numel - base;
        for (long at = threadIdx.x * V; at < left; at += 256 * V) {
            load_run<V>(static_cast<const T*>(t.grad) + base + at, left - at, v);
            add();
        }
    }
    return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

__global__ __launch_bounds__(256) void k_squares(const NormTable a)
{
    __shared__ double lds[4];
    double sum = 0.0;
    each_chunk<false>(a, [&](const smx_grad_tensor& t, long base, bool whole, const Raw& raw) {
        if (t.type == SMX_TYPE_F32) sum += chunk_squares<float>(t, base, whole, raw);
        else if (t.type == SMX_TYPE_BF16) sum += chunk_squares<bf16>(t, base, whole, raw);
        else sum += chunk_squares<f16>(t, base, whole, raw);
    });
    sum = block_total(sum, lds);
    if (threadIdx.x == 0) a.part[blockIdx.x] = sum;
}

struct Norm {
    const double* part;
    int parts;
    double max_norm;
    float *norm, *factor;      // written by the first block; may be null
};
// the factor, the same in all threads and blocks
__device__ __forceinline__ float factor_of(const Norm& p, double* lds)
{
    double sum = 0.0;
#pragma unroll 8
    for (int i = threadIdx.x; i < p.parts; i += 256) sum += p.part[i];
    const double norm = sqrt(block_total(sum, lds));
    // (NaN fails the first comparison, infinity the second)
    const float factor = norm > p.max_norm && norm < __builtin_inf() ? (float)(p.max_norm / norm) : 1.0f;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        if (p.norm) *p.norm = (float)norm;
        if (p.factor) *p.factor = factor;
    }
    return factor;
}
__global__ __launch_bounds__(256) void k_norm(const Norm p)
{
    __shared__ double lds[4];
    factor_of(p, lds);
}

template <typename T>
__device__ __forceinline__ void scale_chunk(const smx_grad_tensor& t, long base, bool whole, const Raw& raw, float factor)
{
    constexpr int V = kRun<T>;
    T* out = static_cast<T*>(t.out) + base;
    float v[V];
    auto scale = [&] {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] *= factor;
    };
    if (whole) {
#pragma unroll
        for (int u = 0; u < kSteps; ++u) {
            numbers_of<T>(raw.v[u], v);
            scale();
            store_past<V>(out + (u * 256 + threadIdx.x) * V, v);
        }
    } else {
        const long left = t.numel - base;
        for (long at = threadIdx.x * V; at < left; at += 256 * V) {
            load_run<V>(static_cast<const T*>(t.grad) + base + at, left - at, v);
            scale();
            store_run<V>(out + at, left - at, v);
        }
    }
}
// Backwards: what the sums read last is in the caches; and past them with what is written (150 million numbers in bfloat16: 151 us a call,
// forwards and through the caches 195).
__global__ __launch_bounds__(256) void k_clip(const NormTable a, const Norm p)
{
    __shared__ double lds[4];
    const float factor = factor_of(p, lds);
    if (factor == 1.0f) {      // (nothing to do in place)
        bool all = true;
        for (int i = 0; i < a.count; ++i) all = all && a.tensor[i].grad == a.tensor[i].out;
        if (all) return;
    }
    each_chunk<true>(a, [&](const smx_grad_tensor& t, long base, bool whole, const Raw& raw) {
        if (t.type == SMX_TYPE_F32) scale_chunk<float>(t, base, whole, raw, factor);
        else if (t.type == SMX_TYPE_BF16) scale_chunk<bf16>(t, base, whole, raw, factor);
        else scale_chunk<f16>(t, base, whole, raw, factor);
    });
}

// ---- host side

long chunks_of(const smx_grad_tensor& t) { return (t.numel + chunk_numbers(t.type) - 1) / chunk_numbers(t.type); }
void check(const smx_grad_tensor* tensors, int count, bool sizes_only, bool outputs)
{
    refuse_unless(count >= 0 && (tensors || count == 0), "count must not be negative, tensors not null");
    for (int i = 0; i < count; ++i) {
        (void)type_bytes(tensors[i].type);
        refuse_unless(tensors[i].numel >= 0 && tensors[i].numel < (1L << 36), "numel: 0 less than 2^36");
        if (tensors[i].numel == 0 || sizes_only) continue;
        refuse_unless(tensors[i].grad, "gradients must not be null");
        refuse_unless(!outputs || tensors[i].out, "out must not be null");
    }
}

// What is written has memory of its own: none of another result's, none of another tensor's gradient, and of its own gradient all or none.
// (Blocks read gradients that others have written already, or will.)
void check_apart(const smx_grad_tensor* tensors, int count)
{
    struct Range {
        size_t from, to;
    };
    auto range = [](const void* at, const smx_grad_tensor& t) {
        const size_t from = reinterpret_cast<size_t>(at);
        return Range{from, from + t.numel * type_bytes(t.type)};
    };
    std::vector<Range> out;
    out.reserve(count);
    for (int i = 0; i < count; ++i)
        if (tensors[i].numel) out.push_back(range(tensors[i].out, tensors[i]));
    std::sort(out.begin(), out.end(), [](const Range& a, const Range& b) { return a.from < b.from; });
    for (size_t k = 1; k < out.size(); ++k) refuse_unless(out[k - 1].to <= out[k].from, "results of tensors share memory");
    for (int i = 0; i < count; ++i) {
        if (tensors[i].numel == 0 || tensors[i].grad == tensors[i].out) continue;
        const Range r = range(tensors[i].grad, tensors[i]);
        const auto behind = std::partition_point(out.begin(), out.end(), [&](const Range& o) { return o.to <= r.from; });
        refuse_unless(behind == out.end() || behind->from >= r.to, "a result shares memory with a gradient that is not its own, or with a part of it");
    }
}

// fn(table, its number of blocks) for as many tensors at a time as a launch takes; the answer: blocks in all, each of which has a part of
// the sum.
template <typename Fn>
int in_tables(const smx_grad_tensor* tensors, int count, Fn&& fn)
{
    long all = 0;
    for (int i = 0; i < count; ++i) all += chunks_of(tensors[i]);
    int parts = 0;
    NormTable a;
    a.count = a.first[0] = 0;
    auto flush = [&] {
        const long chunks = a.first[a.count];
        // of the parts, as many as its share of all chunks
        const int blocks = (int)(all <= kMostParts ? chunks : std::max(1L, kMostParts * chunks / all));
        fn(a, blocks, parts);
        parts += blocks;
        a.count = 0;
    };
    constexpr long kMostChunks = 1L << 30;
    for (int i = 0; i < count; ++i) {
        const long chunks = chunks_of(tensors[i]);
        if (chunks == 0) continue;
        if (a.count == kTensors || (a.count && a.first[a.count] + chunks > kMostChunks)) flush();
        a.tensor[a.count] = tensors[i];
        a.first[a.count + 1] = a.first[a.count] + (int)chunks;
        ++a.count;
    }
    if (a.count) flush();
    return parts;
}
long workspace(const smx_grad_tensor* tensors, int count)
{
    return up(8L * std::max(1, in_tables(tensors, count, [](const NormTable&, int, int) {})), 256);
}

void run(const smx_grad_tensor* tensors, int count, double max_norm, float* d_norm, float* d_factor, void* d_workspace, long workspace_bytes, void* stream, bool clip)
{
    check(tensors, count, false, clip);
    if (clip) check_apart(tensors, count);
    refuse_unless(max_norm >= 0, "max_norm: from 0 on");
    check_workspace(d_workspace, workspace_bytes, workspace(tensors, count), "smx_grad_norm_workspace");
    require_gfx950();
    const hipStream_t s = static_cast<hipStream_t>(stream);
    double* part = static_cast<double*>(d_workspace);
    const int parts = in_tables(tensors, count, [&](NormTable& a, int blocks, int first) {
        a.part = part + first;
        hipLaunchKernelGGL(k_squares, dim3(blocks), dim3(256), 0, s, a);
    });
    Norm n{part, parts, max_norm, d_norm, d_factor};
    if (!clip || parts == 0) hipLaunchKernelGGL(k_norm, dim3(1), dim3(256), 0, s, n);
    else
        in_tables(tensors, count, [&](const NormTable& a, int blocks, int first) {
            hipLaunchKernelGGL(k_clip, dim3(blocks), dim3(256), 0, s, a, n);
            n.norm = nullptr;
        });
    hip_ok(hipGetLastError(), "launch");
}

}  // namespace

}  // namespace smx

using namespace smx;

extern "C" int smx_grad_norm_workspace(const smx_grad_tensor* tensors, int count, long* bytes)
{
    return finetune_entry("smx_grad_norm_workspace", [&] {
        check(tensors, count, true, false);
        refuse_unless(bytes, "bytes must not be null");
        *bytes = workspace(tensors, count);
    });
}

extern "C" int smx_grad_norm(const smx_grad_tensor* tensors, int count, double max_norm, float* d_norm, float* d_factor, void* d_workspace, long workspace_bytes,
                             void* stream)
{
    return finetune_entry("smx_grad_norm", [&] { run(tensors, count, max_norm, d_norm, d_factor, d_workspace, workspace_bytes, stream, false); });
}

extern "C" int smx_clip_grads(const smx_grad_tensor* tensors, int count, double max_norm, float* d_norm, void* d_workspace, long workspace_bytes, void* stream)
{
    return finetune_entry("smx_clip_grads", [&] { run(tensors, count, max_norm, d_norm, nullptr, d_workspace, workspace_bytes, stream, true); });
}
