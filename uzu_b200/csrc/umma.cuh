// Barriers with bounded waits, tiled copies, tcgen05 products and tensor memory, as the kernels of the state space scan and of the experts' layer use them.
// A wait that runs out (about a second) reports its code to the context (wait_errors.h) and makes every role of the CTA leave.
#pragma once

#include <cuda.h>

#include "common.cuh"

namespace uzu {

#ifdef __CUDACC__
__device__ __forceinline__ uint32_t um_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void um_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void um_fence_init() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
// (a whole warp, for all its lanes)
__device__ __forceinline__ void um_arrive(uint32_t bar) {
    __syncwarp();
    if ((threadIdx.x & 31u) == 0) asm volatile("{ .reg .b64 st; mbarrier.arrive.shared::cta.b64 st, [%0]; }" ::"r"(bar) : "memory");
}
// ... once what was loaded into `seen` is there. An arrival takes another way than loads from shared memory and does not wait for them: behind many global accesses
// they came back after the place had been given away (rows of x two chunks on were found). `zero` is 0, which the compiler does not know: the barrier's address then
// depends on the loads, and a warp issues in order.
__device__ __forceinline__ void um_arrive_after(uint32_t bar, uint32_t seen, uint32_t zero) {
    __syncwarp();
    if ((threadIdx.x & 31u) == 0) asm volatile("{ .reg .b64 st; mbarrier.arrive.shared::cta.b64 st, [%0]; }" ::"r"(bar + (seen & zero)) : "memory");
}
__device__ __forceinline__ uint4 um_lds(uint32_t at) {
    uint4 v;
    asm volatile("ld.volatile.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ float4 um_ldf4(const float* p) {
    float4 v;
    asm volatile("ld.volatile.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(um_smem(p)) : "memory");
    return v;
}
__device__ __forceinline__ float um_ldf(const float* p) { return *reinterpret_cast<const volatile float*>(p); }
__device__ __forceinline__ bool um_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3; selp.u32 %0, 1, 0, p; }" : "=r"(ok) : "r"(bar), "r"(parity), "r"(20000u) : "memory");
    return ok != 0;
}
// after a wait that ran out: what is in flight ends before the CTA does
__device__ __forceinline__ void um_settle(uint32_t bar, uint32_t parity) {
    for (uint32_t n = 0; n < 4096 && !um_try(bar, parity); ++n) {}
}
__device__ __forceinline__ uint64_t um_now() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
// By whole warps. false: the phase did not complete within about a second; gave_up then holds the code, which the CTA reports at its end (um_report), and the roles that wait for
// this one run out the same way. As few instructions as it takes: a call would hold its caller's registers down, and what many roles run has to fit the instruction caches.
__device__ __forceinline__ bool um_wait(uint32_t bar, uint32_t parity, volatile uint32_t* gave_up, uint32_t code) {
    uint32_t ok;
    asm volatile(
        "{ .reg .pred p, q; .reg .u64 t, e;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 20000;\n"
        "@p bra DONE_%=;\n"
        "mov.u64 e, %%globaltimer;\n"
        "add.u64 e, e, 1000000000;\n"
        "WAIT_%=: mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 20000;\n"
        "@p bra DONE_%=;\n"
        "mov.u64 t, %%globaltimer;\n"
        "setp.lt.u64 q, t, e;\n"
        "@q bra WAIT_%=;\n"
        "DONE_%=: selp.u32 %0, 1, 0, p; }"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (__all_sync(0xffffffffu, ok)) return true;
    *gave_up = code;
    return false;
}
__device__ __forceinline__ void um_report(volatile uint32_t* gave_up, unsigned int* error) {
    if (*gave_up) report_wait_error(error, *gave_up);
}
__device__ __forceinline__ bool um_elect() {
    uint32_t p = 0;
    asm volatile("{ .reg .pred q; .reg .b32 r; elect.sync r|q, 0xffffffff; @q mov.u32 %0, 1; }" : "+r"(p));
    return p != 0;
}
__device__ __forceinline__ void um_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("{ .reg .b64 st; mbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1; }" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void um_tma(uint32_t dst, const CUtensorMap* map, uint32_t x, uint32_t y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
// rows of shared memory to global memory; the group of them is read when um_store_read returns
__device__ __forceinline__ void um_tma_store(const CUtensorMap* map, uint32_t src, uint32_t x, uint32_t y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];\n\tcp.async.bulk.commit_group;" ::"l"(map), "r"(x), "r"(y), "r"(src) : "memory");
}
__device__ __forceinline__ void um_store_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void um_store_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void um_commit(uint32_t bar) { asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void um_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void um_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void um_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void um_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void um_fence_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// 16 columns of the warp's lanes. The wait is part of it: between a load and its wait the registers hold nothing, and the compiler may move or spill what it takes for a value.
__device__ __forceinline__ void um_ld16(uint32_t taddr0, uint32_t (&v0)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=&r"(v0[0]), "=&r"(v0[1]), "=&r"(v0[2]), "=&r"(v0[3]), "=&r"(v0[4]), "=&r"(v0[5]), "=&r"(v0[6]), "=&r"(v0[7]), 
          "=&r"(v0[8]), "=&r"(v0[9]), "=&r"(v0[10]), "=&r"(v0[11]), "=&r"(v0[12]), "=&r"(v0[13]), "=&r"(v0[14]), "=&r"(v0[15])
        : "r"(taddr0)
        : "memory");
}
// twice 16 (8) columns under way together
__device__ __forceinline__ void um_ld16x2(uint32_t taddr0, uint32_t taddr1, uint32_t (&v0)[16], uint32_t (&v1)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%32];\n\ttcgen05.ld.sync.aligned.32x32b.x16.b32 {%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%33];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=&r"(v0[0]), "=&r"(v0[1]), "=&r"(v0[2]), "=&r"(v0[3]), "=&r"(v0[4]), "=&r"(v0[5]), "=&r"(v0[6]), "=&r"(v0[7]), 
          "=&r"(v0[8]), "=&r"(v0[9]), "=&r"(v0[10]), "=&r"(v0[11]), "=&r"(v0[12]), "=&r"(v0[13]), "=&r"(v0[14]), "=&r"(v0[15]), 
          "=&r"(v1[0]), "=&r"(v1[1]), "=&r"(v1[2]), "=&r"(v1[3]), "=&r"(v1[4]), "=&r"(v1[5]), "=&r"(v1[6]), "=&r"(v1[7]), 
          "=&r"(v1[8]), "=&r"(v1[9]), "=&r"(v1[10]), "=&r"(v1[11]), "=&r"(v1[12]), "=&r"(v1[13]), "=&r"(v1[14]), "=&r"(v1[15])
        : "r"(taddr0), "r"(taddr1)
        : "memory");
}
__device__ __forceinline__ void um_ld8x2(uint32_t taddr0, uint32_t taddr1, uint32_t (&v0)[8], uint32_t (&v1)[8]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%16];\n\ttcgen05.ld.sync.aligned.32x32b.x8.b32 {%8,%9,%10,%11,%12,%13,%14,%15}, [%17];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=&r"(v0[0]), "=&r"(v0[1]), "=&r"(v0[2]), "=&r"(v0[3]), "=&r"(v0[4]), "=&r"(v0[5]), "=&r"(v0[6]), "=&r"(v0[7]), 
          "=&r"(v1[0]), "=&r"(v1[1]), "=&r"(v1[2]), "=&r"(v1[3]), "=&r"(v1[4]), "=&r"(v1[5]), "=&r"(v1[6]), "=&r"(v1[7])
        : "r"(taddr0), "r"(taddr1)
        : "memory");
}
__device__ __forceinline__ void um_st8(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
__device__ __forceinline__ void um_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// a warpgroup's registers (of every thread; the warpgroups' shares together are what the block was launched with)
template <uint32_t R>
__device__ __forceinline__ void um_fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R)); }
template <uint32_t R>
__device__ __forceinline__ void um_more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R)); }
__device__ __forceinline__ uint32_t um_pack(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float um_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float um_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
#endif

inline decltype(&cuTensorMapEncodeTiled) um_encoder() {
    static decltype(&cuTensorMapEncodeTiled) fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) f = nullptr;
        cudaGetLastError();
        return (decltype(&cuTensorMapEncodeTiled))f;
    }();
    return fn;
}
// rows of bf16, `pitch` elements apart, in boxes of 64 elements (128-byte swizzled rows) by `box_rows`
inline bool um_map(CUtensorMap* map, uint64_t addr, uint64_t width, uint64_t rows, uint64_t pitch, uint32_t box_rows) {
    const cuuint64_t dims[2] = {width, rows}, strides[1] = {pitch * 2};
    const cuuint32_t box[2] = {64, box_rows}, steps[2] = {1, 1};
    return um_encoder() && um_encoder()(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, (void*)addr, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace uzu
