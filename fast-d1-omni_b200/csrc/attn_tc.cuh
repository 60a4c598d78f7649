// Building blocks shared by the tcgen05 attention kernels (attn.cu, kv4_attn.cu): exponentials and packed fp32 arithmetic
// of the softmax, the MMA with its A operand in tensor memory, bulk stores of output tiles, waits with a time limit, and
// the tensor maps.
#pragma once
#include "common.cuh"

namespace d1 {

__device__ __forceinline__ void fence_async_smem_cta() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Bulk tensor store of a staged O tile and its completion waits (issued and awaited by one thread).
__device__ __forceinline__ void o_tile_store(const CUtensorMap* map, uint32_t src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"((uint64_t)map),
                 "r"(src), "r"(x), "r"(y)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void o_store_read_done() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void o_store_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

__device__ __forceinline__ void record_err(int* err, volatile int* abort_flag, int code) {
    *abort_flag = 1;
    if (err) atomicExch(err, code);
}

__device__ __forceinline__ bool mbar_wait_timed2(uint32_t bar, uint32_t parity) {
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(bar, parity))
        if (globaltimer_ns() - t0 > kWaitLimitNs) return false;
    return true;
}

__device__ __forceinline__ void cp_async16z(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// 2^x with the hardware approximation (relative error ~2^-22, far below the fp16 rounding of P).
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two fp32 lanes in one 64-bit register for the packed sm_100 instructions: d = a * b + c and d = a + b, per lane.
__device__ __forceinline__ uint64_t f2_pack(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void f2_unpack(uint64_t v, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// 2^x of two lanes on the FMA pipe (Cody-Waite style): n = round(x) by the 1.5 * 2^23 shifter, f = x - n in
// [-0.5, 0.5], 2^f by a cubic fitted for relative error on that interval (7.5e-5 max, below the fp16 rounding of
// P), 2^n added into the exponent field. x is clamped to -126 first (masked keys give ~1e-38, zero in fp16).
__device__ __forceinline__ void ex2_poly2(float x0, float x1, float& p0, float& p1) {
    const uint64_t x = f2_pack(fmaxf(x0, -126.f), fmaxf(x1, -126.f));
    const uint64_t t = f2_add(x, f2_pack(12582912.f, 12582912.f));
    const uint64_t n = f2_add(t, f2_pack(-12582912.f, -12582912.f));
    const uint64_t f = f2_fma(n, f2_pack(-1.f, -1.f), x);
    uint64_t q = f2_fma(f2_pack(0.0551716685f, 0.0551716685f), f, f2_pack(0.24261114f, 0.24261114f));
    q = f2_fma(q, f, f2_pack(0.69326097f, 0.69326097f));
    q = f2_fma(q, f, f2_pack(0.99992806f, 0.99992806f));
    float q0, q1, t0, t1;
    f2_unpack(q, q0, q1);
    f2_unpack(t, t0, t1);
    p0 = __uint_as_float(__float_as_uint(q0) + (__float_as_uint(t0) << 23));
    p1 = __uint_as_float(__float_as_uint(q1) + (__float_as_uint(t1) << 23));
}

// max(a, b, c) in one instruction (sm_100).
__device__ __forceinline__ float fmax3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// D[tmem] (+)= A[tmem] . B[smem]: A (M=128 rows = TMEM lanes, K fp16 values packed two per 32-bit column) in
// tensor memory, B through a shared-memory descriptor, fp32 accumulate; shape from the instruction descriptor.
__device__ __forceinline__ void tc_mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                              uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(0u)
        : "memory");
}

// A 2-D fp16 tensor map over rows x cols (row pitch ld elements) with 64-column x box_rows boxes in the 128-byte
// swizzle; rows past `rows` read as zeros.
inline bool attn_tmap(CUtensorMap* m, const void* base, int cols, int rows, int ld, uint32_t box_rows) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return false;
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
    cuuint32_t box[2] = {64, box_rows};
    cuuint32_t estr[2] = {1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(base), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace d1
