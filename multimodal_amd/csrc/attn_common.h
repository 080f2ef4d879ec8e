// attn_common.h - small device helpers shared by the attention kernels.
#pragma once
#include "common.h"

namespace mm {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Make a register-resident operand "used" here: the compiler must finish its global load before this point instead of
// sinking the load to the first MFMA inside the tile loop (where its pending vmcnt would serialise every iteration's
// prefetch behind the MFMAs).
template <typename V> __device__ __forceinline__ void pin(V& v) {
    static_assert(sizeof(V) == 16, "a 16-byte operand");
    u32x4 t;
    __builtin_memcpy(&t, &v, 16);
    asm volatile("" : "+v"(t));
    __builtin_memcpy(&v, &t, 16);
}
__device__ __forceinline__ void pin(float& v) { asm volatile("" : "+v"(v)); }

// Combine a value with the one held by the lane 32 away (the other half of the wave) without the LDS round trip of
// ds_bpermute: v_permlane32_swap exchanges the upper 32 lanes of its first operand with the lower 32 of its second, so with
// both operands = x every lane ends up holding (lower-half value, upper-half value) of its lane pair.
__device__ __forceinline__ void half_pair(float x, float& lo, float& hi) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    lo = __uint_as_float(r[0]);
    hi = __uint_as_float(r[1]);
}
__device__ __forceinline__ float half_max(float x) {
    float lo, hi;
    half_pair(x, lo, hi);
    return fmaxf(lo, hi);
}
__device__ __forceinline__ float half_sum(float x) {
    float lo, hi;
    half_pair(x, lo, hi);
    return lo + hi;
}

}  // namespace mm
