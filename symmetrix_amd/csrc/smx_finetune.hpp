// Shared by the operators for fine-tuned heads (layer norm, adapters beside a shared projection, AdamW, tables and
// products by group, norms of gradients): element types, loads and
// stores of runs of numbers at any alignment, sums over lanes, and what their C entry points check.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <new>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "../../include/symmetrix_amd.h"
#include "smx_internal.hpp"

namespace smx {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16;
typedef _Float16 f16;

// V numbers that need no more alignment than one of them (global memory takes such accesses; at an aligned address they cost no more)
template <typename T, int V>
struct Run {
    typedef T type __attribute__((ext_vector_type(V)));
    typedef type loose __attribute__((aligned(sizeof(T))));
};
template <typename T>
constexpr int kRun = 16 / (int)sizeof(T);      // numbers in 16 bytes

// left: numbers from p on that exist; zeros behind them
template <int V, typename T>
__device__ __forceinline__ void load_run(const T* p, long left, float (&v)[V])
{
    if (left >= V) {
        const typename Run<T, V>::type x = *reinterpret_cast<const typename Run<T, V>::loose*>(p);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = (float)x[j];
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = j < left ? (float)p[j] : 0.0f;
    }
}
// (all V of them, in 16 bytes, which nothing is expected to read soon)
template <int V, typename T>
__device__ __forceinline__ void store_past(T* p, const float (&v)[V])
{
    static_assert(V * sizeof(T) == 16, "16 bytes");
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    typedef u32x4 loose __attribute__((aligned(2)));
    typename Run<T, V>::type x;
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = (T)v[j];
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4, x), reinterpret_cast<loose*>(p));
}
template <int V, typename T>
__device__ __forceinline__ void store_run(T* p, long left, const float (&v)[V])
{
    if (left >= V) {
        typename Run<T, V>::type x;
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = (T)v[j];
        *reinterpret_cast<typename Run<T, V>::loose*>(p) = x;
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j < left) p[j] = (T)v[j];
    }
}


// 1 KB of a wavefront from global memory (16 bytes per lane, at base + offset, a multiple of 16) into LDS at `to` + 16 lane.
// In assembly: next to the compiler's own form of this load it lets every read of the LDS wait for all loads in flight; here
// wait_loads waits by count.  The LDS address goes through m0, which the load may read one wait state after the write (s_nop) and has
// read when it is issued; m0 belongs to the compiler and is given back as it was.
__device__ __forceinline__ void load_into_lds(const void* base, unsigned offset, unsigned to)
{
    unsigned m0;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0) : "v"(offset), "s"(base), "s"(to) : "memory");
}
// all but the N youngest loads have arrived, and every read and write of the LDS is done
template <int N>
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(N) : "memory"); }
// a barrier that waits for nothing but the wavefronts (__syncthreads would wait for loads in flight too)
__device__ __forceinline__ void barrier_only()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ unsigned lds_address(const void* p) { return (unsigned)(unsigned long)(__attribute__((address_space(3))) const void*)p; }

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

// sum over groups of G neighbouring lanes, the same in all of them
template <int G>
__device__ __forceinline__ float group_sum(float x)
{
#pragma unroll
    for (int d = 1; d < G; d *= 2) x += __shfl_xor(x, d, 64);
    return x;
}

// ---- host side

struct Refusal : std::runtime_error {
    int code;
    Refusal(int c, const std::string& what) : std::runtime_error(what), code(c) {}
};

// Runs a C entry point: no exception leaves it.
template <typename Fn>
int finetune_entry(const char* name, Fn&& fn) noexcept
{
    try {
        try {
            fn();
            return SMX_OK;
        } catch (const Refusal& e) {
            set_last_error(std::string(name) + ": " + e.what());
            return e.code;
        } catch (const std::bad_alloc&) {
            set_last_error("out of host memory");
            return SMX_ENOMEM;
        } catch (const std::exception& e) {
            set_last_error(std::string(name) + ": " + e.what());
            return SMX_EINVAL;
        }
    } catch (...) {      // (the message did not fit into memory either)
        return SMX_ENOMEM;
    }
}
inline void refuse_unless(bool holds, const char* what)
{
    if (!holds) throw Refusal(SMX_EINVAL, what);
}
inline void hip_ok(hipError_t e, const char* what)
{
    if (e != hipSuccess) throw Refusal(SMX_EHIP, std::string(what) + ": " + hipGetErrorString(e));
}
// the current device is one that the kernels are built for
inline void require_gfx950()
{
    static thread_local int checked = -1;
    int dev = -1;
    const bool known = hipGetDevice(&dev) == hipSuccess;
    if (known && dev == checked) return;
    int n = 0;
    if (!known || hipGetDeviceCount(&n) != hipSuccess || n <= 0)
        throw Refusal(SMX_ENODEVICE, "no HIP device available: there is no CPU path");
    hipDeviceProp_t prop;
    if (hipGetDeviceProperties(&prop, dev) != hipSuccess) throw Refusal(SMX_ENODEVICE, "hipGetDeviceProperties failed");
    if (std::string(prop.gcnArchName).rfind("gfx950", 0) != 0)
        throw Refusal(SMX_ENODEVICE, std::string("kernels are built for gfx950 only; found ") + prop.gcnArchName);
    checked = dev;
}
inline int type_bytes(int type)
{
    if (type == SMX_TYPE_F32) return 4;
    if (type == SMX_TYPE_BF16 || type == SMX_TYPE_F16) return 2;
    throw Refusal(SMX_EINVAL, "element type: SMX_TYPE_F32, SMX_TYPE_BF16 or SMX_TYPE_F16");
}
// fn(float{}), fn(bf16{}) or fn(f16{})
template <typename Fn>
void with_type(int type, Fn&& fn)
{
    if (type == SMX_TYPE_F32) fn(float{});
    else if (type == SMX_TYPE_BF16) fn(bf16{});
    else fn(f16{});
}

inline long up(long x, long m) { return (x + m - 1) / m * m; }

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

inline void check_workspace(const void* at, long bytes, long need, const char* who)
{
    if (need != 0 && !(at && bytes >= need)) throw Refusal(SMX_EINVAL, std::string("the workspace is smaller than ") + who + " says");
    refuse_unless((reinterpret_cast<size_t>(at) & 255) == 0, "the workspace: an address that is a multiple of 256");
}

template <int N>
using Int = std::integral_constant<int, N>;

// The launches of a call.
struct Launches {
    hipStream_t s;
    const bool dry;      // nothing is launched, the workspace is counted, and the sizes of the launches are looked at
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
};

}  // namespace smx
