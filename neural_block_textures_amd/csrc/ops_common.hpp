// What the operators of include/ntc_ops.h share: element types, loads of runs of them, wave reductions, refusals.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include <type_traits>

#include "ntc_ops.h"

namespace ntc_ops {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLowest = -3.402823466e38f;
#define NTC_INF __builtin_inff()

// ---------------------------------------------------------------- element types
using f32 = float;
using bf16 = __bf16;
using f16 = _Float16;
template <class T> constexpr int type_code = 0;
template <> inline constexpr int type_code<bf16> = NTC_BF16;
template <> inline constexpr int type_code<f16> = NTC_F16;

template <class T, int N> struct alignas(sizeof(T) * N) Run { T v[N]; };
// A run at any element's address: one wide access all the same (the hardware takes unaligned ones, at the cost of the lines it crosses).
template <class T, int N> struct __attribute__((packed, aligned(sizeof(T)))) LooseRun { T v[N]; };

inline size_t type_size(int t) { return t == NTC_F32 ? 4 : 2; }

// ---------------------------------------------------------------- lanes
__device__ __forceinline__ int lane_id() { return (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)); }
__device__ __forceinline__ float read_lane(float x, int l) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), l)); }
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }   // one instruction, 1 ulp; 2^-inf = 0
__device__ __forceinline__ float fast_log2(float x) { return __builtin_amdgcn_logf(x); }

// Between a wave's accesses to shared memory of which some lanes read what others wrote: the hardware keeps them in order by itself, the
// compiler does only across a fence (it takes a wave barrier alone for something that touches no memory). No instruction comes of it.
__device__ __forceinline__ void wave_shared() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Reductions over aligned groups of 4, 8, 16, 32 and 64 lanes: every lane gets the result, and no shared memory is used (lanes
// exchanged within a row of 16 on the way into the instruction, rows swapped). f is commutative and associative.
template <int kCtrl, class V> __device__ __forceinline__ V exchange(V x) {
    return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), kCtrl, 0xf, 0xf, false));
}
template <int kGroup, class V, class F> __device__ __forceinline__ V reduce(V x, F f) {
    x = f(x, exchange<0xb1>(x));                             // lane ^ 1
    x = f(x, exchange<0x4e>(x));                             // lane ^ 2
    if constexpr (kGroup >= 8) x = f(x, exchange<0x141>(x)); // the other four of eight, mirrored
    if constexpr (kGroup >= 16) x = f(x, exchange<0x140>(x));
    if constexpr (kGroup >= 32) {
        const uint32_t b = __builtin_bit_cast(uint32_t, x);
        const auto p = __builtin_amdgcn_permlane16_swap(b, b, false, false);
        x = f(__builtin_bit_cast(V, (uint32_t)p[0]), __builtin_bit_cast(V, (uint32_t)p[1]));
    }
    if constexpr (kGroup >= 64) {
        const uint32_t b = __builtin_bit_cast(uint32_t, x);
        const auto p = __builtin_amdgcn_permlane32_swap(b, b, false, false);
        x = f(__builtin_bit_cast(V, (uint32_t)p[0]), __builtin_bit_cast(V, (uint32_t)p[1]));
    }
    return x;
}
template <class V, class F> __device__ __forceinline__ V reduce16(V x, F f) { return reduce<16>(x, f); }
template <class V, class F> __device__ __forceinline__ V reduce64(V x, F f) { return reduce<64>(x, f); }
// of lanes l, l ^ 16, l ^ 32 and l ^ 48
template <class V, class F> __device__ __forceinline__ V reduce_rows(V x, F f) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    const auto p = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    x = f(__builtin_bit_cast(V, (uint32_t)p[0]), __builtin_bit_cast(V, (uint32_t)p[1]));
    const uint32_t c = __builtin_bit_cast(uint32_t, x);
    const auto q = __builtin_amdgcn_permlane32_swap(c, c, false, false);
    return f(__builtin_bit_cast(V, (uint32_t)q[0]), __builtin_bit_cast(V, (uint32_t)q[1]));
}

// ---------------------------------------------------------------- launches
// A grid of n blocks and a block's number in it: a dimension's threads have to stay below 2^32. (Numbers may pass n.)
inline dim3 grid_of(int64_t n) { return n <= 1 << 22 ? dim3((unsigned)n) : dim3(1u << 22, (unsigned)((n + (1 << 22) - 1) >> 22)); }
__device__ __forceinline__ long long block_number() { return blockIdx.x + (long long)blockIdx.y * gridDim.x; }

// ---------------------------------------------------------------- refusals
inline int refuse(char* why, size_t cap, const char* text) {
    if (why && cap) snprintf(why, cap, "%s", text);
    return 1;
}
inline int launched(char* why, size_t cap) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return 0;
    if (why && cap) snprintf(why, cap, "launch failed: %s", hipGetErrorString(e));
    return 2;
}

}  // namespace ntc_ops
