// The 4-bit key/value cache format of include/d1kernels.h (D1Kv4Seq) on the device: expansion of codes to fp16 pairs
// and the checks of a table entry, shared by kv4.cu (append, load, evict) and kv4_attn.cu (attention, mass).
#pragma once
#include "common.cuh"

namespace d1 {

// Error codes of the d1_kv4_* kernels beyond those of the waits.
enum : int { kErrTable = 6 };  // a table entry that breaks the header's rules; it was skipped

constexpr int kKv4MaxRows = 1 << 30;  // of a cache: row counters that step by a grid's rows stay inside 32 bits

// Device address of the error word on the current device, or NULL.
int* kv4_err_addr();

// SMs of the current device, or 0.
inline int sm_count() {
    static int sms[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (!sms[dev & 63] && cudaDeviceGetAttribute(&sms[dev & 63], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return 0;
    return sms[dev & 63];
}

__device__ __forceinline__ bool kv4_cache_ok(int len, int cap, const void* k4, const void* v4, const void* kp,
                                             const void* vp) {
    if (len < 0 || len > cap || cap > kKv4MaxRows || (cap & 7)) return false;
    if (cap == 0) return true;
    if (!k4 || !v4 || !kp || !vp) return false;
    return (((uintptr_t)k4 | (uintptr_t)v4 | (uintptr_t)kp | (uintptr_t)vp) & 15) == 0;
}

__device__ __forceinline__ bool kv4_seq_ok(const D1Kv4Seq& s) {
    return kv4_cache_ok(s.ext_len, s.ext_cap, s.k4, s.v4, s.kp, s.vp);
}

// Rows [start, start + len) lie inside [0, rows); none do, wherever they start.
__device__ __forceinline__ bool rows_ok(int start, int len, int rows) {
    return len == 0 || (start >= 0 && len > 0 && (long long)start + len <= rows);
}

__device__ __forceinline__ uint32_t h2_sub(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t h2_mul(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
template <int OP>
__device__ __forceinline__ uint32_t lop3(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, %4;" : "=r"(d) : "r"(a), "r"(b), "r"(c), "n"(OP));
    return d;
}

// The zero points of two parameters (one in each half) as the fp16 pairs that the expansion subtracts: 1024 + zero for
// codes at bits 0-3 of a half, 64 + zero for codes at bits 4-7.
__device__ __forceinline__ void kv4_zero(uint32_t par2, uint32_t& z0, uint32_t& z1) {
    constexpr int kAndOr = (0xf0 & 0xcc) | 0xaa;
    z0 = lop3<kAndOr>(par2, 0x000f000fu, 0x64006400u);
    z1 = lop3<kAndOr>(par2 << 4, 0x00f000f0u, 0x54005400u);
}
__device__ __forceinline__ uint32_t kv4_step2(uint32_t par2) { return par2 & 0xfff0fff0u; }
__device__ __forceinline__ float kv4_step(uint32_t par) { return __half2float(__ushort_as_half(par & 0xfff0u)); }

// The expansion of 4-bit weights by or-ing codes into the mantissa of 1024 (Kim et al., "Who Says Elephants Can't Run:
// Bringing Large Scale MoE Models into Cloud Scale Production", 2022), here with 64 for the upper nibbles.
// A word's eight codes as fp16 pairs of (code - zero): out[i] holds the codes at bits 4i (low half) and 16 + 4i (high
// half). A code at bits 0-3 of a half, or-ed into the fp16 pattern of 1024, is 1024 + code; at bits 4-7, into that of
// 64, it is 64 + code; the differences are whole numbers in -15 .. 15, exact. One shift for the upper two codes.
__device__ __forceinline__ void kv4_expand(uint32_t w, uint32_t z0, uint32_t z1, uint32_t (&out)[4]) {
    const uint32_t h = w >> 8;
    constexpr int kAndOr = (0xf0 & 0xcc) | 0xaa;
    out[0] = h2_sub(lop3<kAndOr>(w, 0x000f000fu, 0x64006400u), z0);
    out[1] = h2_sub(lop3<kAndOr>(w, 0x00f000f0u, 0x54005400u), z1);
    out[2] = h2_sub(lop3<kAndOr>(h, 0x000f000fu, 0x64006400u), z0);
    out[3] = h2_sub(lop3<kAndOr>(h, 0x00f000f0u, 0x54005400u), z1);
}

}  // namespace d1
