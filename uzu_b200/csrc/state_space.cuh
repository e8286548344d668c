// What the kernels of a state space mixer share: rows of 16 and 32 bits, a step's size, the gate.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "row_sequences.h"

namespace uzu {

inline uint32_t ss_size(uint32_t data_type) { return data_type == UZU_DT_F32 ? 4u : 2u; }
inline bool ss_data_type(uint32_t data_type) { return data_type == UZU_DT_BF16 || data_type == UZU_DT_F32 || data_type == UZU_DT_F16; }

// the scan of a call on tcgen05 (state_space_umma.cu): whether it takes the call, the scratch that lets it cut long sequences into parts
bool scan_umma_applicable(const uzu_state_space_scan_args& a);
bool encode_scan_umma(uzu_command_buffer* cmd, const uzu_state_space_scan_args& a);
size_t scan_umma_scratch_bytes(const uzu_context* ctx, const uzu_state_space_scan_args& a);

#ifdef __CUDACC__
__device__ __forceinline__ float ss_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float ss_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float ss_f(float v) { return v; }
template <typename T>
__device__ __forceinline__ T ss_t(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 ss_t<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half ss_t<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float ss_t<float>(float v) { return v; }

// 2^x, 1 / x: to a few 2^-24 of the value, below 2^-126 zero
__device__ __forceinline__ float ss_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float ss_rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// pairs of f32 in one instruction
__device__ __forceinline__ float2 ss_fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
    return d;
}
__device__ __forceinline__ float2 ss_mul2(float2 a, float2 b) {
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return d;
}
__device__ __forceinline__ float2 ss_add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return d;
}
// x sigmoid(x), to about 2^-21 of its value (the exponent's rounding: 2^-24 |x| more) down to x = -87; 0 below, where the value is less than 2^-119
__device__ __forceinline__ float ss_silu(float x) { return x * ss_rcp(1.0f + ss_exp2(-1.4426950408889634f * x)); }
__device__ __forceinline__ float2 ss_silu2(float2 x) {
    const float2 e = ss_mul2(x, make_float2(-1.4426950408889634f, -1.4426950408889634f));
    const float2 d = ss_add2(make_float2(ss_exp2(e.x), ss_exp2(e.y)), make_float2(1.0f, 1.0f));
    return ss_mul2(x, make_float2(ss_rcp(d.x), ss_rcp(d.y)));
}
// a token's step (log1p: steps of 1e-3 keep their digits); not a number stays so
__device__ __forceinline__ float ss_step(float dt, float bias, uint32_t softplus, float lo, float hi) {
    float s = dt + bias;
    if (softplus) s = s > 20.0f ? s : log1pf(expf(s));
    return s < lo ? lo : s > hi ? hi : s;
}
// the sequence of a launch's tile
__device__ __forceinline__ uint32_t ss_find(const SequenceTable& t, uint32_t tile) {
    uint32_t lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const uint32_t mid = (lo + hi + 1) >> 1;
        if (t.s[mid].tile0 <= tile) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
#endif

}  // namespace uzu
