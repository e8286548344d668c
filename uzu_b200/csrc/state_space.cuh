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

// x sigmoid(x), to about 2^-21 of its value
__device__ __forceinline__ float ss_silu(float x) { return __fdividef(x, 1.0f + __expf(-x)); }
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
