// One AdamW step over many tensors, with moments in 32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,   p = (1 - lr decay) p - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Moments in 8 bits: 256 numbers share a scale, the largest of them, which is held in single precision.  Codes run with the root of
// |m| and the fourth root of v, so that m and sqrt(v) have the same resolution, finest near zero:  m = scale c |c| / 127^2,
// v = scale (c / 255)^4.  The moments of a step are what was read, brought to single precision; the parameters see them before they
// are rounded.  Rounded to nearest, a moment that moves by less than half a code a step would never move, and v decays by a
// thousandth a step; so the place where a number is rounded up moves over [0, 1), by 0.046 from step to step (once around in 21.6
// steps) and by 0.618 from a number to the next.  What is lost at some is made up for at others: over the numbers of a tensor in every
// step, and for one number over some tens of steps, which a v of beta2 = 0.99 or more remembers.  An m of beta1 = 0.9 forgets in ten, and
// keeps a part of what it was rounded by.
// A v that is not zero keeps the code 1 at least (an m beside it that is not rounded to zero would be divided by eps).  There is no code
// for infinity or NaN: a scale that is one makes its 256 numbers NaN from the next step on.
//
// Every operation is rounded once, in the order written (no fused multiply-adds, IEEE division and root), so that the codes are those
// of the same formulas elsewhere.
//
// What bounds it is memory: 807 us for 150 million parameters in bfloat16 with masters and moments in 32 bits (28 bytes each, 5.2 TB/s).
// Moments in 8 bits are 2 + 1/32 bytes to read and as many to write; there the divisions and roots that make codes count as much as the bytes.
#include "smx_finetune.hpp"

#include <algorithm>
#include <cmath>
#include <cstdint>

namespace smx {

namespace {

constexpr int kTensors = 56;         // of a launch: their descriptions are kernel arguments
constexpr int kBlock = SMX_MOMENT_BLOCK;
constexpr int kChunk = 4096;         // numbers of a thread block: 16 scales, four per wavefront

struct AdamwTable {
    smx_adamw_tensor tensor[kTensors];
    int first[kTensors + 1];         // chunks in front of each
    int count;
    float beta1, beta2, rest1, rest2, keep, rate, root, eps;      // rest: 1 - beta; keep: 1 - lr decay; rate: lr / (1 - beta1^t); root: 1 / sqrt(1 - beta2^t)
    unsigned turn1, turn2;           // where the rounding of the moments' codes stands
};
static_assert(sizeof(AdamwTable) <= 4096, "kernel arguments");

struct Updated {
    float p, m, v;
};
__device__ __forceinline__ Updated update(const AdamwTable& a, float p, float g, float m, float v)
{
    m = m * a.beta1 + g * a.rest1;
    v = v * a.beta2 + g * a.rest2 * g;
    p = p * a.keep - m * a.rate / (sqrtf(v) * a.root + a.eps);
    return {p, m, v};
}

// tensor of a chunk (the same in all lanes)
__device__ __forceinline__ int tensor_of(const AdamwTable& a, int chunk)
{
    int low = 0, high = a.count;
    while (high - low > 1) {
        const int mid = (low + high) / 2;
        if (a.first[mid] <= chunk) low = mid;
        else high = mid;
    }
    return low;
}

template <typename T, typename TG, bool MASTERS>
__global__ __launch_bounds__(256) void k_adamw(const AdamwTable a)
{
    constexpr int V = 4;
    const int i = tensor_of(a, blockIdx.x);
    const smx_adamw_tensor& t = a.tensor[i];
    const long base = (long)(blockIdx.x - a.first[i]) * kChunk;
    T* param = static_cast<T*>(t.param);
    const TG* grad = static_cast<const TG*>(t.grad);
    float *master = t.master, *ms = static_cast<float*>(t.exp_avg), *vs = static_cast<float*>(t.exp_avg_sq);
    const long n = t.numel;
#pragma unroll
    for (int u = 0; u < kChunk / (256 * V); ++u) {
        const long at = base + (u * 256 + threadIdx.x) * V;
        if (at >= n) return;
        float p[V], g[V], m[V], v[V];
        if constexpr (MASTERS) load_run<V>(master + at, n - at, p);
        else load_run<V>(param + at, n - at, p);
        load_run<V>(grad + at, n - at, g);
        load_run<V>(ms + at, n - at, m);
        load_run<V>(vs + at, n - at, v);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const Updated x = update(a, p[j], g[j], m[j], v[j]);
            p[j] = x.p; m[j] = x.m; v[j] = x.v;
        }
        store_run<V>(param + at, n - at, p);
        if constexpr (MASTERS) store_run<V>(master + at, n - at, p);
        store_run<V>(ms + at, n - at, m);
        store_run<V>(vs + at, n - at, v);
    }
}

// largest of the wavefront's numbers, NaN if one of them is
__device__ __forceinline__ float wave_largest(float x)
{
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const float y = __shfl_xor(x, d, 64);
        x = (x != x || x > y) ? x : y;
    }
    return x;
}
__device__ __forceinline__ float first_moment(int c, float scale)
{
    const float q = (float)c * (1.0f / 127.0f);
    return q * fabsf(q) * scale;
}
__device__ __forceinline__ float second_moment(int c, float scale)
{
    const float q = (float)c * (1.0f / 255.0f), r = q * q;
    return r * r * scale;
}
__device__ __forceinline__ float turn_of(unsigned inside, unsigned turn)
{
    return (float)((inside * 0x9E3779B1u + turn) >> 8) * 0x1p-24f;
}

// A wavefront takes 256 numbers at a time: four neighbours a lane.
template <typename T, typename TG, bool MASTERS>
__global__ __launch_bounds__(256) void k_adamw_codes(const AdamwTable a)
{
    constexpr int V = 4, SCALES = kChunk / kBlock / 4;
    const int i = tensor_of(a, blockIdx.x), wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const smx_adamw_tensor& t = a.tensor[i];
    const long base = (long)(blockIdx.x - a.first[i]) * kChunk;
    T* param = static_cast<T*>(t.param);
    const TG* grad = static_cast<const TG*>(t.grad);
    float* master = t.master;
    int8_t* cm = static_cast<int8_t*>(t.exp_avg);
    uint8_t* cv = static_cast<uint8_t*>(t.exp_avg_sq);
    const long n = t.numel;
#pragma unroll 1
    for (int u = 0; u < SCALES; ++u) {
        const long start = base + (u * 4 + wave) * kBlock, at = start + lane * V;
        if (start >= n) return;
        const float sm = t.scale_avg[start / kBlock], sv = t.scale_avg_sq[start / kBlock];
        float p[V], g[V], m[V], v[V], c[V], d[V];
        if constexpr (MASTERS) load_run<V>(master + at, n - at, p);
        else load_run<V>(param + at, n - at, p);
        load_run<V>(grad + at, n - at, g);
        load_run<V>(cm + at, n - at, c);
        load_run<V>(cv + at, n - at, d);
        float most_m = 0.0f, most_v = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const Updated x = update(a, p[j], g[j], first_moment((int)c[j], sm), second_moment((int)d[j], sv));
            p[j] = x.p;
            // (behind the end of the tensor there is nothing, whatever the scales are)
            m[j] = at + j < n ? x.m : 0.0f;
            v[j] = at + j < n ? x.v : 0.0f;
            const float am = fabsf(m[j]);
            most_m = (most_m != most_m || most_m > am) ? most_m : am;
            most_v = (most_v != most_v || most_v > v[j]) ? most_v : v[j];
        }
        store_run<V>(param + at, n - at, p);
        if constexpr (MASTERS) store_run<V>(master + at, n - at, p);
        most_m = wave_largest(most_m);
        most_v = wave_largest(most_v);
        const float by_m = most_m > 0.0f ? most_m : 1.0f, by_v = most_v > 0.0f ? most_v : 1.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const unsigned inside = (unsigned)(at + j);
            // (NaN has no code: its scale says it)
            const float qm = fminf(floorf(sqrtf(fabsf(m[j]) / by_m) * 127.0f + turn_of(inside, a.turn1)), 127.0f);
            const float qv = fminf(floorf(sqrtf(sqrtf(v[j] / by_v)) * 255.0f + turn_of(inside, a.turn2)), 255.0f);
            c[j] = m[j] < 0.0f ? -qm : qm;
            d[j] = v[j] > 0.0f ? fmaxf(qv, 1.0f) : 0.0f;
        }
        store_run<V>(cm + at, n - at, c);
        store_run<V>(cv + at, n - at, d);
        if (lane == 0) {
            t.scale_avg[start / kBlock] = most_m;
            t.scale_avg_sq[start / kBlock] = most_v;
        }
    }
}

// what codes stand for
__global__ __launch_bounds__(256) void k_moment_values(long n, const int8_t* cm, const float* sm, const uint8_t* cv, const float* sv, float* m, float* v)
{
    constexpr int V = 4;
    const long at = ((long)blockIdx.x * 256 + threadIdx.x) * V;
    if (at >= n) return;
    float c[V];
    if (m) {
        load_run<V>(cm + at, n - at, c);
        const float s = sm[at / kBlock];
#pragma unroll
        for (int j = 0; j < V; ++j) c[j] = first_moment((int)c[j], s);
        store_run<V>(m + at, n - at, c);
    }
    if (v) {
        load_run<V>(cv + at, n - at, c);
        const float s = sv[at / kBlock];
#pragma unroll
        for (int j = 0; j < V; ++j) c[j] = second_moment((int)c[j], s);
        store_run<V>(v + at, n - at, c);
    }
}

}  // namespace

}  // namespace smx

using namespace smx;

extern "C" int smx_adamw_step(int param_type, int grad_type, int state_bits, const smx_adamw_tensor* tensors, int count, double lr, double beta1,
                              double beta2, double eps, double weight_decay, long step, void* stream)
{
    return finetune_entry("smx_adamw_step", [&] {
        (void)type_bytes(param_type);
        refuse_unless(grad_type == param_type || grad_type == SMX_TYPE_F32, "gradients: the parameters' type or single precision");
        refuse_unless(state_bits == 32 || state_bits == 8, "state_bits: 32 or 8");
        refuse_unless(count >= 0 && (tensors || count == 0), "count must not be negative, tensors not null");
        refuse_unless(step >= 1, "step: counted from 1");
        refuse_unless(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1, "betas: 0 up to, not including, 1");
        refuse_unless(std::isfinite(lr) && lr >= 0 && std::isfinite(weight_decay) && weight_decay >= 0 && std::isfinite(eps) && eps >= 0,
                      "lr, weight_decay and eps: numbers from 0 on");
        bool masters = false, first = true;
        for (int i = 0; i < count; ++i) {
            const smx_adamw_tensor& t = tensors[i];
            refuse_unless(t.numel >= 0 && t.numel < (1L << 36), "numel: 0 less than 2^36");
            if (t.numel == 0) continue;
            refuse_unless(t.param && t.grad && t.exp_avg && t.exp_avg_sq, "parameters, gradients and moments must not be null");
            refuse_unless(state_bits == 32 || (t.scale_avg && t.scale_avg_sq), "moments in 8 bits need their scales");
            refuse_unless(first || masters == (t.master != nullptr), "masters: for all tensors of a call or for none");
            masters = t.master != nullptr;
            first = false;
        }
        refuse_unless(!masters || param_type != SMX_TYPE_F32, "masters are for parameters in 16 bits");
        if (first) return;
        require_gfx950();
        AdamwTable a{};
        a.beta1 = (float)beta1; a.beta2 = (float)beta2; a.rest1 = (float)(1 - beta1); a.rest2 = (float)(1 - beta2);
        a.keep = (float)(1 - lr * weight_decay);
        a.rate = (float)(lr / (1 - std::pow(beta1, (double)step)));
        a.root = (float)(1 / std::sqrt(1 - std::pow(beta2, (double)step)));
        a.eps = (float)eps;
        a.turn1 = (unsigned)(2 * (unsigned long)step) * 0x85EBCA6Bu;
        a.turn2 = (unsigned)(2 * (unsigned long)step + 1) * 0x85EBCA6Bu;
        const hipStream_t s = static_cast<hipStream_t>(stream);
        auto launch = [&] {
            const dim3 grid((unsigned)a.first[a.count]);
            with_type(param_type, [&](auto t) {
                using T = decltype(t);
                auto go = [&](auto tg, auto with_masters) {
                    using TG = decltype(tg);
                    constexpr bool M = decltype(with_masters)::value;
                    if (state_bits == 32) hipLaunchKernelGGL((k_adamw<T, TG, M>), grid, dim3(256), 0, s, a);
                    else hipLaunchKernelGGL((k_adamw_codes<T, TG, M>), grid, dim3(256), 0, s, a);
                };
                if constexpr (std::is_same_v<T, float>) go(T{}, std::false_type{});
                else {
                    auto with = [&](auto tg) {
                        if (masters) go(tg, std::true_type{});
                        else go(tg, std::false_type{});
                    };
                    if (grad_type == param_type) with(T{});
                    else with(float{});
                }
            });
            hip_ok(hipGetLastError(), "launch");
            a.count = 0;
        };
        constexpr long kMostChunks = 1L << 23;      // (a launch takes fewer than 2^32 threads, a tensor at most 2^24 chunks)
        for (int i = 0; i < count; ++i) {
            if (tensors[i].numel == 0) continue;
            const long chunks = (tensors[i].numel + kChunk - 1) / kChunk;
            if (a.count == kTensors || (a.count && a.first[a.count] + chunks > kMostChunks)) launch();
            a.tensor[a.count] = tensors[i];
            a.first[a.count + 1] = a.first[a.count] + (int)chunks;
            ++a.count;
        }
        launch();
    });
}

extern "C" int smx_moment_values(long numel, const void* d_code_avg, const float* d_scale_avg, const void* d_code_avg_sq, const float* d_scale_avg_sq,
                                 float* d_exp_avg, float* d_exp_avg_sq, void* stream)
{
    return finetune_entry("smx_moment_values", [&] {
        refuse_unless(numel >= 0 && numel < (1L << 36), "numel: 0 less than 2^36");
        if (numel == 0 || (!d_exp_avg && !d_exp_avg_sq)) return;
        refuse_unless((!d_exp_avg || (d_code_avg && d_scale_avg)) && (!d_exp_avg_sq || (d_code_avg_sq && d_scale_avg_sq)), "codes and scales must not be null");
        require_gfx950();
        constexpr long kSlab = 1L << 30;      // (a launch takes fewer than 2^32 threads; whole blocks of a scale)
        for (long at = 0; at < numel; at += kSlab) {
            const long n = std::min(numel - at, kSlab);
            hipLaunchKernelGGL(k_moment_values, dim3((unsigned)((n + 1023) / 1024)), dim3(256), 0, static_cast<hipStream_t>(stream), n,
                               d_exp_avg ? static_cast<const int8_t*>(d_code_avg) + at : nullptr, d_exp_avg ? d_scale_avg + at / kBlock : nullptr,
                               d_exp_avg_sq ? static_cast<const uint8_t*>(d_code_avg_sq) + at : nullptr, d_exp_avg_sq ? d_scale_avg_sq + at / kBlock : nullptr,
                               d_exp_avg ? d_exp_avg + at : nullptr, d_exp_avg_sq ? d_exp_avg_sq + at : nullptr);
        }
        hip_ok(hipGetLastError(), "launch");
    });
}
