// What the operators of include/ntc_ops.h share: element types, loads of runs of them, wave reductions, refusals.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>

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
