// Shared by the operators for fine-tuned heads (layer norm, adapters beside a shared projection, AdamW): element types, loads and
// stores of runs of numbers at any alignment, sums over lanes, and what their C entry points check.
#pragma once

#include <hip/hip_runtime.h>

#include <new>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "../../include/symmetrix_amd.h"
#include "smx_internal.hpp"

namespace smx {

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

typedef float f32x4 __attribute__((ext_vector_type(4)));

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

}  // namespace smx
