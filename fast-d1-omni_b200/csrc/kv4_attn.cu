// Attention over key/value caches held in 4 bits (format: include/d1kernels.h, D1Kv4Seq), and the attention weight that
// every cached key received. Head dim 64, packed variable-length sequences, bidirectional.
#include "attn_tc.cuh"
#include "kv4.cuh"
#include "warp_mma.cuh"

using namespace d1;

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kMaxHeads = 0x7fffffff / 64;  // their columns are counted in 32 bits
constexpr float kLazyRescale = 8.f;  // log2: how far scores may exceed the reference of a running softmax

struct Kv4Args {
    const __half* Q;
    const __half* K;
    const __half* V;
    __half* O;
    float* lse;
    const D1Kv4Seq* seqs;
    int* err;
    int ldq, ldkv, ldo, lse_ld, n_seqs, heads, group, q_rows, kv_rows, accumulate, ranks;
    float scale_log2;
};

__device__ __forceinline__ float fmax_nan(float a, float b) {  // NaN if either is
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float fmin_nan(float a, float b) {
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// 2^x of two numbers without the SFU: x = n + f, n whole by adding and taking away 1.5 * 2^23 (the sum's low bits, with
// 127 added, are 2^n's exponent), |f| <= 1/2, 2^f by a polynomial of degree 5 fitted here for the smallest relative error,
// 2.1e-7 evaluated in fp32. x below -126.5 gives 0, above 127.5 infinity; NaN stays.
__device__ __forceinline__ void ex2_fma2(float x0, float x1, float& p0, float& p1) {
    const uint64_t x = f2_pack(fmin_nan(fmax_nan(x0, -127.f), 128.f), fmin_nan(fmax_nan(x1, -127.f), 128.f));
    const uint64_t t = f2_add(x, f2_pack(12583039.f, 12583039.f));
    const uint64_t f = f2_fma(f2_add(t, f2_pack(-12583039.f, -12583039.f)), f2_pack(-1.f, -1.f), x);
    auto c2 = [](float c) { return f2_pack(c, c); };
    uint64_t q = f2_fma(c2(0.00132764725f), f, c2(0.00967554096f));
    q = f2_fma(q, f, c2(0.0555071309f));
    q = f2_fma(q, f, c2(0.240221202f));
    q = f2_fma(q, f, c2(0.693146944f));
    q = f2_fma(q, f, c2(1.00000012f));
    float t0, t1;
    f2_unpack(t, t0, t1);
    f2_unpack(f2_mul(q, f2_pack(__uint_as_float(__float_as_uint(t0) << 23), __uint_as_float(__float_as_uint(t1) << 23))), p0, p1);
}

// ------------------------------------------------------------------------------------------------ attention, few rows
// The query rows of a kv head's group are packed: packed row p is row p / group of the sequence, head p % group of the
// group. A cluster of 1 to 8 CTAs takes 8 * NT packed rows of one (sequence, kv head); the CTAs share out its tiles of 64
// keys, and the warps of a CTA take theirs in turn, each with its own running maximum, sum and output. They are joined
// through shared memory, and the CTAs of a cluster through distributed shared memory, always in the same order.
//
// Everything is transposed, S^T = K Q^T and O^T = V^T P^T on m16n8k16, so that 8 rows fill an MMA's n. The codes go from
// global memory to the registers of the A operands directly. An MMA's k index may run over the dimensions in any order as
// long as both operands use the same: for S^T lane (r, t) = (lane / 4, lane % 4) holds dimensions 16t .. 16t+15 of keys r
// and r + 8 of each 16: 8 bytes of codes, and 32 bytes of a query row. The MMA sees the whole numbers code - zero; a key's
// step multiplies its scores afterwards, in fp32, with the softmax scale. For O^T lane (r, t) holds word r (dimensions
// 8r .. 8r+7) of keys 2t, 2t+1, 2t+8, 2t+9 of each 16; byte permutes bring two keys' codes of one dimension together, and
// the values are (code - zero) * step, exact in fp16. Row r of the j-th m tile is dimension 8r + 2j, row r + 8 dimension
// 8r + 2j + 1, so that a lane ends with dimensions 8r .. 8r+7 of packed rows 2t and 2t + 1. P^T turns from the result's
// layout into the B operand's by movmatrix.
// Bound: latency, and unequal sequences. 32 tokens over 8346 to 16151 keys, 89 us: the SMs are busy for 0.81 of the time and
// issue in 0.52 of those cycles (about 800 instructions a tile, half of them for the expansion of codes), 16 warps an SM
// waiting for each other's results and for memory. Of 9 to 64 packed rows the time is about five times that of the bytes
// (16 x 32 packed rows over 8000 keys: 55 us). Tried and dropped: the codes as fp16 subnormals (code * 2^-24 or * 2^-20, no
// subtraction), with zeros and steps taken care of by the sums: an eighth fewer instructions, but the MMA aligns its fp32
// sums to the operands' exponent, and their last 10 bits are lost.
constexpr int R_KEYS = 64, R_CLUSTER = 8, R_LD = 68;  // padded row of the joining buffers (floats)

template <int NT, int W>
constexpr int rows_smem() {
    return (W + 1) * 8 * NT * (R_LD + 2) * 4;
}

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

template <int NT, int W>
__global__ void __launch_bounds__(W * 32, (NT == 1 ? 16 : 8) / W) k_kv4_attn_rows(const Kv4Args a) {
    extern __shared__ __align__(16) float r_smem[];
    constexpr int NR = 8 * NT;
    float* sO = r_smem;                               // [warp][NR][R_LD]
    float* cO = sO + W * NR * R_LD;             // [NR][R_LD]: the CTA's sum, read by the cluster
    float* sM = cO + NR * R_LD;                       // [warp][NR]
    float* cM = sM + W * NR;                    // [NR]
    float* sL = cM + NR;                              // [warp][NR]
    float* cL = sL + W * NR;                    // [NR]
    pdl_entry();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = lane >> 2, t = lane & 3, g = blockIdx.y;
    const int rank = (int)cluster_ctarank(), ranks = a.ranks;
    for (int sq = blockIdx.z; sq < a.n_seqs; sq += gridDim.z) {
        const D1Kv4Seq s = a.seqs[sq];
        if (!kv4_seq_ok(s) || !rows_ok(s.q_start, s.q_len, a.q_rows) || !rows_ok(s.kv_start, s.kv_len, a.kv_rows)) {
            if (tid == 0) atomicExch(a.err, kErrTable);
            continue;
        }
        const uint32_t group = a.group, n_rows = (uint32_t)s.q_len * group;  // (2^31 rows would exceed the memory)
        const int ext_tiles = (s.ext_len + R_KEYS - 1) / R_KEYS, tiles = ext_tiles + (s.kv_len + R_KEYS - 1) / R_KEYS;
        // this CTA's tiles
        const int per = (tiles + ranks - 1) / ranks, tile0 = min(tiles, rank * per), tile1 = min(tiles, tile0 + per);
        const uint8_t* k4 = s.k4 + (size_t)g * s.ext_cap * 32 + 8 * t;
        const uint8_t* v4 = s.v4 + (size_t)g * s.ext_cap * 32 + 4 * r;
        const uint16_t* kp = reinterpret_cast<const uint16_t*>(s.kp) + (size_t)g * s.ext_cap;
        const uint16_t* vp = reinterpret_cast<const uint16_t*>(s.vp) + (size_t)g * s.ext_cap;
        for (uint32_t base = blockIdx.x / ranks * NR; base < n_rows; base += gridDim.x / ranks * NR) {
            // ---- the query rows, as B operands: [n tile][k step][2]
            uint32_t qb[NT][4][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const uint32_t p = base + nt * 8 + r;
                uint4 x0 = make_uint4(0, 0, 0, 0), x1 = x0;
                if (p < n_rows) {
                    const uint32_t row = p / group, h = g * group + p % group;
                    const uint4* src =
                        reinterpret_cast<const uint4*>(a.Q + (size_t)(s.q_start + row) * a.ldq + h * 64 + 16 * t);
                    x0 = __ldg(src);
                    x1 = __ldg(src + 1);
                }
                const uint32_t w[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
#pragma unroll
                for (int i = 0; i < 8; i++) qb[nt][i >> 1][i & 1] = w[i];
            }
            float o[NT][4][4], m[NT][2], l[NT][2];  // rows 2t and 2t + 1 of each n tile
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int c = 0; c < 4; c++) o[nt][j][c] = 0.f;
                m[nt][0] = m[nt][1] = 0.f;
                l[nt][0] = l[nt][1] = 0.f;
            }
            bool started = false;  // this warp has had a tile
            uint2 kw[8];       // cached: this lane's codes of keys 8i + r
            uint32_t pk = 0;   // K parameters of keys 2 lane, 2 lane + 1
            auto fetch_k = [&](int tile) {
                const int key0 = tile * R_KEYS, last = min(s.ext_len - key0, R_KEYS) - 1;
                const uint8_t* src = k4 + (size_t)key0 * 32;
                if (last == R_KEYS - 1) {
#pragma unroll
                    for (int i = 0; i < 8; i++) kw[i] = __ldg(reinterpret_cast<const uint2*>(src + r * 32 + i * 256));
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++) kw[i] = __ldg(reinterpret_cast<const uint2*>(src + min(8 * i + r, last) * 32));
                }
                // whole pairs are inside the cache's arrays: ext_cap is a multiple of 8
                pk = __ldg(reinterpret_cast<const uint32_t*>(kp + key0 + (min(2 * lane, last) & ~1)));
            };
            int tile = tile0 + warp;
            if (tile < tile1 && tile < ext_tiles) fetch_k(tile);
            for (; tile < tile1; tile += W) {
                const bool ext = tile < ext_tiles;
                const int key0 = (ext ? tile : tile - ext_tiles) * R_KEYS;
                const int left = (ext ? s.ext_len : s.kv_len) - key0;  // keys of this tile: min(left, 64), at least 1
                const int last = min(left, R_KEYS) - 1;
                float sc[NT][4][4];  // keys 16i + r (0, 1) and 16i + 8 + r (2, 3), rows 2t and 2t + 1
                uint32_t vw[4][4];   // cached: the words of V
                uint32_t pv = 0;     // cached: V parameters of keys 2 lane, 2 lane + 1
                if (ext) {
                    const uint8_t* src = v4 + (size_t)key0 * 32;
                    if (last == R_KEYS - 1) {
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            vw[i >> 2][i & 3] = __ldg(reinterpret_cast<const uint32_t*>(
                                src + t * 64 + ((i >> 2) * 16 + (i & 1) + (i & 2) * 4) * 32));
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            vw[i >> 2][i & 3] = __ldg(reinterpret_cast<const uint32_t*>(
                                src + min((i >> 2) * 16 + 2 * t + (i & 1) + (i & 2) * 4, last) * 32));
                    }
                    pv = __ldg(reinterpret_cast<const uint32_t*>(vp + key0 + (min(2 * lane, last) & ~1)));
                    // rows behind the cached ones hold anything: step 0 there, so that 0 * V is 0
                    if (2 * lane + 1 > last) pv = 2 * lane > last ? 0 : pv & 0xffffu;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        uint32_t ka[4][4];
                        float st[2];
#pragma unroll
                        for (int hf = 0; hf < 2; hf++) {
                            const int n = 2 * i + hf;
                            const uint32_t both = __shfl_sync(D1_FULL_MASK, pk, 4 * n + (r >> 1));
                            const uint32_t par = __byte_perm(both, 0, r & 1 ? 0x3232 : 0x1010);
                            uint32_t z0, z1, x[4], y[4];
                            kv4_zero(par, z0, z1);
                            kv4_expand(kw[n].x, z0, z1, x);
                            kv4_expand(kw[n].y, z0, z1, y);
                            ka[0][hf] = x[0];
                            ka[0][2 + hf] = x[1];
                            ka[1][hf] = x[2];
                            ka[1][2 + hf] = x[3];
                            ka[2][hf] = y[0];
                            ka[2][2 + hf] = y[1];
                            ka[3][hf] = y[2];
                            ka[3][2 + hf] = y[3];
                            st[hf] = kv4_step(par & 0xffffu) * a.scale_log2;
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            float c[4];
                            mma16816_first(c, ka[0], qb[nt][0][0], qb[nt][0][1]);
#pragma unroll
                            for (int ks = 1; ks < 4; ks++) mma16816(c, ka[ks], qb[nt][ks][0], qb[nt][ks][1]);
                            const uint64_t m2 = f2_pack(-m[nt][0], -m[nt][1]);
#pragma unroll
                            for (int hf = 0; hf < 2; hf++)
                                f2_unpack(f2_fma(f2_pack(c[2 * hf], c[2 * hf + 1]), f2_pack(st[hf], st[hf]), m2),
                                          sc[nt][i][2 * hf], sc[nt][i][2 * hf + 1]);
                        }
                    }
                    if (tile + W < tile1 && tile + W < ext_tiles) fetch_k(tile + W);
                } else {
                    const __half* kr = a.K + (size_t)(s.kv_start + key0) * a.ldkv + g * 64 + 16 * t;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        uint32_t ka[4][4];
#pragma unroll
                        for (int hf = 0; hf < 2; hf++) {
                            const uint4* src =
                                reinterpret_cast<const uint4*>(kr + (size_t)min(16 * i + 8 * hf + r, last) * a.ldkv);
                            const uint4 x0 = __ldg(src), x1 = __ldg(src + 1);
                            const uint32_t w[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
#pragma unroll
                            for (int q = 0; q < 8; q++) ka[q >> 1][(q & 1) * 2 + hf] = w[q];
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            float c[4];
                            mma16816_first(c, ka[0], qb[nt][0][0], qb[nt][0][1]);
#pragma unroll
                            for (int ks = 1; ks < 4; ks++) mma16816(c, ka[ks], qb[nt][ks][0], qb[nt][ks][1]);
#pragma unroll
                            for (int q = 0; q < 4; q++) sc[nt][i][q] = c[q] * a.scale_log2 - m[nt][q & 1];
                        }
                    }
                }
                if (left < R_KEYS) {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
#pragma unroll
                            for (int q = 0; q < 4; q++)
                                if (16 * i + 8 * (q >> 1) + r >= left) sc[nt][i][q] = -INFINITY;
                }
                // ---- running softmax, in the exp2 domain. The scores are taken against the reference m as it was before
                // this tile; only where one exceeds it by more than 2^8 (and in the first tile) does m move, and what was
                // summed so far is rescaled: P stays below 2^8, well inside fp16, to which it is rounded for the product with
                // V, as in the fp16 attention; the row's sum is of P in fp32 (O is 2.4e-4 to 2.9e-4 off, and 2.1e-4 by its own
                // rounding alone). P^T as B operands: keys 16i + 2t, 16i + 2t + 1 and 8 above
                uint32_t pb[NT][4][2];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float over[2];
#pragma unroll
                    for (int q = 0; q < 2; q++) {
                        over[q] = fmaxf(sc[nt][0][q], sc[nt][0][q + 2]);
#pragma unroll
                        for (int i = 1; i < 4; i++) over[q] = fmax3(over[q], sc[nt][i][q], sc[nt][i][q + 2]);
                    }
                    if (!started || __any_sync(D1_FULL_MASK, fmaxf(over[0], over[1]) > kLazyRescale)) {
#pragma unroll
                        for (int q = 0; q < 2; q++) {
                            float up = over[q];
                            up = fmaxf(up, __shfl_xor_sync(D1_FULL_MASK, up, 4));
                            up = fmaxf(up, __shfl_xor_sync(D1_FULL_MASK, up, 8));
                            up = fmaxf(up, __shfl_xor_sync(D1_FULL_MASK, up, 16));
                            if (started) up = fmaxf(up, 0.f);
                            const float alpha = started ? ex2(-up) : 0.f;
                            m[nt][q] += up;
                            l[nt][q] *= alpha;
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                o[nt][i][q] *= alpha;
                                o[nt][i][q + 2] *= alpha;
                                sc[nt][i][q] -= up;
                                sc[nt][i][q + 2] -= up;
                            }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int hf = 0; hf < 2; hf++) {
                            const float p0 = ex2(sc[nt][i][2 * hf]), p1 = ex2(sc[nt][i][2 * hf + 1]);
                            l[nt][0] += p0;
                            l[nt][1] += p1;
                            pb[nt][i][hf] = movmatrix_trans(pack_h2(p0, p1));
                        }
                }
                started = true;
                // ---- O^T += V^T P^T
#pragma unroll
                for (int ks = 0; ks < 4; ks++) {
                    uint32_t va[4][4];  // [m tile][dimensions 8r + 2j, 8r + 2j + 1 of keys 2t, 2t+1; of 2t+8, 2t+9]
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        if (ext) {
                            const uint32_t par = __shfl_sync(D1_FULL_MASK, pv, 8 * ks + 4 * i + t);
                            const uint32_t st = kv4_step2(par);
                            uint32_t z0, z1, ev[4], od[4];
                            kv4_zero(par, z0, z1);
                            kv4_expand(__byte_perm(vw[ks][2 * i], vw[ks][2 * i + 1], 0x5410), z0, z1, ev);
                            kv4_expand(__byte_perm(vw[ks][2 * i], vw[ks][2 * i + 1], 0x7632), z0, z1, od);
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                va[j][2 * i] = h2_mul(ev[j], st);
                                va[j][2 * i + 1] = h2_mul(od[j], st);
                            }
                        } else {
                            const __half* vr = a.V + (size_t)(s.kv_start + key0) * a.ldkv + g * 64 + 8 * r;
                            const int k = 16 * ks + 8 * i + 2 * t;
                            const uint4 x = __ldg(reinterpret_cast<const uint4*>(vr + (size_t)min(k, last) * a.ldkv));
                            const uint4 y = __ldg(reinterpret_cast<const uint4*>(vr + (size_t)min(k + 1, last) * a.ldkv));
                            const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                va[j][2 * i] = __byte_perm(xs[j], ys[j], 0x5410);
                                va[j][2 * i + 1] = __byte_perm(xs[j], ys[j], 0x7632);
                            }
                        }
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int j = 0; j < 4; j++) mma16816(o[nt][j], va[j], pb[nt][ks][0], pb[nt][ks][1]);
                }
            }
            // ---- join the warps, weights 2^(m - M), in their order; a warp without tiles has m = -inf and l = 0
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    float sum = l[nt][q];
                    sum += __shfl_xor_sync(D1_FULL_MASK, sum, 4);
                    sum += __shfl_xor_sync(D1_FULL_MASK, sum, 8);
                    sum += __shfl_xor_sync(D1_FULL_MASK, sum, 16);
                    const int row = warp * NR + nt * 8 + 2 * t + q;
                    if (r == 0) {
                        sM[row] = started ? m[nt][q] : -INFINITY;
                        sL[row] = sum;
                    }
                    float4* dst = reinterpret_cast<float4*>(sO + row * R_LD + 8 * r);
                    dst[0] = make_float4(o[nt][0][q], o[nt][0][q + 2], o[nt][1][q], o[nt][1][q + 2]);
                    dst[1] = make_float4(o[nt][2][q], o[nt][2][q + 2], o[nt][3][q], o[nt][3][q + 2]);
                }
            __syncthreads();
            auto finish = [&](uint32_t p, int d, float M, float L, const float4& x) {
                const float il = tiles ? 1.f / L : 0.f;
                const int q = s.q_start + (int)(p / group), h = g * a.group + (int)(p % group);
                *reinterpret_cast<uint2*>(a.O + (size_t)q * a.ldo + h * 64 + d) =
                    make_uint2(pack_h2(x.x * il, x.y * il), pack_h2(x.z * il, x.w * il));
                if (a.lse && d == 0) a.lse[(size_t)h * a.lse_ld + q] = tiles ? (M + log2f(L)) * kLn2 : -INFINITY;
            };
            const int warps = min(W, tile1 - tile0);  // those with tiles
            for (int i = tid; i < NR * 16; i += W * 32) {
                const int row = i >> 4, d = (i & 15) * 4;
                if (base + row >= n_rows) break;
                float M = -INFINITY, L = 0.f;
                for (int w = 0; w < warps; w++) M = fmaxf(M, sM[w * NR + row]);
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int w = 0; w < warps; w++) {
                    const float f = ex2(sM[w * NR + row] - M);
                    const float4 v = *reinterpret_cast<const float4*>(sO + (w * NR + row) * R_LD + d);
                    L += f * sL[w * NR + row];
                    x.x += f * v.x;
                    x.y += f * v.y;
                    x.z += f * v.z;
                    x.w += f * v.w;
                }
                if (ranks == 1) {
                    finish(base + row, d, M, L, x);
                    continue;
                }
                *reinterpret_cast<float4*>(cO + row * R_LD + d) = x;
                if (d == 0) {
                    cM[row] = M;
                    cL[row] = L;
                }
            }
            if (ranks == 1) {
                __syncthreads();  // before the next rows
                continue;
            }
            // ---- join the CTAs; each writes its share of the output
            __syncwarp();
            cluster_sync();
            const int parts = tiles == 0 ? 0 : (tiles - 1) / per + 1;  // CTAs with tiles
            for (int i = rank * W * 32 + tid; i < NR * 16; i += ranks * W * 32) {
                const int row = i >> 4, d = (i & 15) * 4;
                if (base + row >= n_rows) break;
                float cm[R_CLUSTER], cl[R_CLUSTER];
                float4 v[R_CLUSTER];
#pragma unroll
                for (int c = 0; c < R_CLUSTER; c++) {
                    cm[c] = -INFINITY;
                    cl[c] = 0.f;
                    v[c] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (c < parts) {
                        cm[c] = ld_cluster_f32(mapa_shared(smem_u32(cM + row), c));
                        cl[c] = ld_cluster_f32(mapa_shared(smem_u32(cL + row), c));
                        v[c] = ld_cluster_f32x4(mapa_shared(smem_u32(cO + row * R_LD + d), c));
                    }
                }
                float M = -INFINITY, L = 0.f;
#pragma unroll
                for (int c = 0; c < R_CLUSTER; c++) M = fmaxf(M, cm[c]);
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int c = 0; c < R_CLUSTER; c++) {
                    if (c >= parts) break;
                    const float f = ex2(cm[c] - M);
                    L += f * cl[c];
                    x.x += f * v[c].x;
                    x.y += f * v[c].y;
                    x.z += f * v[c].z;
                    x.w += f * v[c].w;
                }
                finish(base + row, d, M, L, x);
            }
            __syncwarp();
            cluster_sync();  // the other CTAs have read this one's sums
        }
    }
}

// ------------------------------------------------------------------------------------------------ attention, many rows
// tcgen05 form. Persistent CTAs (one per SM) loop over units. A unit is, by the length of its sequence,
//   packed  up to 128 packed query rows (row p / group, head p % group) of one kv head; the two softmax warpgroups take
//           its key tiles in turn and are joined at the end, each for half of the dimensions
//   pair    128 rows of two heads of one kv head (an even group), a warpgroup each
//   single  256 rows of one head (an odd group), a warpgroup for each 128
// Keys come in tiles of 128, first the cached ones, then the own ones; the last tile of either kind is filled up with
// zeros and masked.
// Warps:
//   0-3, 4-7   softmax: thread = query row = TMEM lane. S is copied to registers and released at once, P goes to TMEM as
//              fp16, O is rescaled only when a row's maximum grows by more than 2^8. Warps whose rows are all behind the
//              sequence's end leave the work out.
//   8          fetches the query rows by TMA (packed ones from a view of [row][head][64]) and, by bulk copies into a ring
//              of their own, the codes and parameters of the cached tiles, from one thread
//   10-13      expand them to fp16 (exact) into the swizzled layout that the MMAs read. Own rows come by
//              TMA. (A tile takes the four warps 1700 clocks, most of it latency; 3200 with the
//              codes loaded straight into their registers, a tile ahead; 2200 with two warps to a tile, in turn.)
//   9, 14      MMA issuers of warpgroups 0 and 1, one thread each: S = Q K^T (both in shared memory), O += P V (P in
//              TMEM). Warp 9 also keeps the TMEM. (One issuer for both: each warpgroup then waits for the other's P.)
// The softmax warps take 200 registers, the others 56 (four documents of 2048 rows over 4096 keys: 253.5 us; 256.7 with
// 192 and 64, 254 with 208 and 48, 272 with 184 and 72; 252.5 now).
// TMEM (512 columns), warpgroup w at 256 w: S in 128 columns, P in 64, O in 64. Both warpgroups' columns share the lanes,
// so that a packed unit is joined by each reading the other's O.
constexpr int TQ = 128, TKV = 128, T_QSLOTS = 2, T_STAGES = 4, T_RAW_STAGES = 3, T_EXPANDERS = 128, T_THREADS = 512;
constexpr int T_QT_BYTES = TQ * 128, T_KV_BYTES = TKV * 128;
constexpr int T_RAW_V = TKV * 32, T_RAW_KP = 2 * TKV * 32, T_RAW_VP = T_RAW_KP + TKV * 2, T_RAW_BYTES = T_RAW_VP + TKV * 2;
constexpr int T_ENTRIES = 256;  // of the table of units
constexpr int T_SOFTMAX_REGS = 200, T_OTHER_REGS = 56;
static_assert(T_SOFTMAX_REGS + T_OTHER_REGS <= 2 * 128, "what the launch of 512 threads, 128 registers each, has");
constexpr uint32_t T_TMEM_COLS = 512, T_WG_COLS = 256, T_P_COL = TKV, T_O_COL = TKV + TKV / 2;
enum : int {
    B_QFULL = 0,
    B_QEMPTY = B_QFULL + T_QSLOTS,
    B_KVFULL = B_QEMPTY + T_QSLOTS,
    B_KVEMPTY = B_KVFULL + T_STAGES,
    B_SFULL = B_KVEMPTY + T_STAGES,  // [w]: S of the warpgroup's next keys is in TMEM
    B_SFREE = B_SFULL + 2,           // [w]: it is in registers (4 warps)
    B_PFULL = B_SFREE + 2,           // [w]: P is in TMEM (4 warps)
    B_ODONE = B_PFULL + 2,           // [w]: P V has completed
    B_OFREE = B_ODONE + 2,           // [w]: O has been read (8 warps of a packed unit, otherwise 4, twice)
    B_RAWFULL = B_OFREE + 2,         // [raw stage]: a tile's codes and parameters are in shared memory
    B_RAWEMPTY = B_RAWFULL + T_RAW_STAGES,  // [raw stage] (4 warps)
    B_OWN = B_RAWEMPTY + T_RAW_STAGES,  // [stage]: a partial tile of own rows has landed
    B_JOIN = B_OWN + T_STAGES,       // a packed unit's maxima and sums are in shared memory, its O's complete (8 warps)
    B_DRAIN = B_JOIN + 1,            // [issuer]
    T_NBARS = B_DRAIN + 2
};
constexpr int T_SMEM = T_QSLOTS * 2 * T_QT_BYTES + T_STAGES * 2 * T_KV_BYTES + T_RAW_STAGES * T_RAW_BYTES + T_NBARS * 8 + 16 + TQ * 16 +
                       (T_ENTRIES * 6 + 1) * 4;
static_assert(T_SMEM <= 232448 && T_O_COL + 64 <= T_WG_COLS, "shared memory and TMEM of the tcgen05 attention");

enum : int { kPacked, kPair, kSingle };

__device__ __forceinline__ int unit_mode(const Kv4Args& a, int q_len) {
    return (long long)q_len * a.group <= TQ ? kPacked : a.group % 2 == 0 ? kPair : kSingle;
}
// Units of sequence sq; none of a sequence without rows or with a bad entry (report: tell).
__device__ __forceinline__ int seq_units(const Kv4Args& a, int sq, bool report) {
    const D1Kv4Seq s = a.seqs[sq];
    if (!kv4_seq_ok(s) || !rows_ok(s.q_start, s.q_len, a.q_rows) || !rows_ok(s.kv_start, s.kv_len, a.kv_rows)) {
        if (report) atomicExch(a.err, kErrTable);
        return 0;
    }
    if (s.q_len == 0) return 0;
    const int mode = unit_mode(a, s.q_len);
    return mode == kPacked ? a.heads / a.group
                           : mode == kPair ? ((s.q_len - 1) / TQ + 1) * (a.heads / 2) : ((s.q_len - 1) / (2 * TQ) + 1) * a.heads;
}
// The table of units: cum[e] = units of the sequences before the e-th run of `run` sequences, and behind it, for runs of
// one, what a unit needs of its sequence, five words each. Ends with a barrier.
__device__ __forceinline__ void build_units(const Kv4Args& a, int* cum, int run) {
    for (int e = threadIdx.x; e < T_ENTRIES; e += blockDim.x) {
        int n = 0;
        for (int i = e * run; i < min(a.n_seqs, (e + 1) * run); i++) n += seq_units(a, i, true);
        cum[e + 1] = n;
        if (run == 1 && e < a.n_seqs) {
            const D1Kv4Seq& s = a.seqs[e];
            int* info = cum + T_ENTRIES + 1 + e;
            info[0] = s.q_start;
            info[T_ENTRIES] = s.q_len;
            info[2 * T_ENTRIES] = s.kv_start;
            info[3 * T_ENTRIES] = s.kv_len;
            info[4 * T_ENTRIES] = s.ext_len;
        }
    }
    if (threadIdx.x == 0) cum[0] = 0;
    __syncthreads();
    if (threadIdx.x < 32) {
        constexpr int PER = T_ENTRIES / 32;
        int v[PER], sum = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) sum += v[i] = cum[1 + threadIdx.x * PER + i];
        int upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(D1_FULL_MASK, upto, o);
            if ((int)threadIdx.x >= o) upto += x;
        }
        upto -= sum;
#pragma unroll
        for (int i = 0; i < PER; i++) cum[1 + threadIdx.x * PER + i] = upto += v[i];
    }
    __syncthreads();
}

template <bool SPLIT>
struct Unit {
    int sq, q_start, q_len, kv_start, kv_len, ext_len;
    int mode, block, h;  // h: first head; of a packed unit the first of its kv head
    int entry = 0;       // of the table
    int t0, t1;          // SPLIT: its key tiles

    // unit u of the table, at or behind the one found before (a CTA's units ascend). Little code, and no loop of fixed
    // length: it runs once a unit, mostly from outside the instruction cache, in every role
    __device__ void find(const Kv4Args& a, const int* cum, int run, int u) {
        while (cum[entry + 1] <= u) entry++;
        int rest = u - cum[entry];
        sq = entry * run;
        if (run > 1)
            for (int n; rest >= (n = seq_units(a, sq, false)); sq++) rest -= n;
        if (run == 1) {
            const int* info = cum + T_ENTRIES + 1 + sq;
            q_start = info[0];
            q_len = info[T_ENTRIES];
            kv_start = info[2 * T_ENTRIES];
            kv_len = info[3 * T_ENTRIES];
            ext_len = info[4 * T_ENTRIES];
        } else {
            const D1Kv4Seq& s = a.seqs[sq];
            q_start = s.q_start;
            q_len = s.q_len;
            kv_start = s.kv_start;
            kv_len = s.kv_len;
            ext_len = s.ext_len;
        }
        mode = unit_mode(a, q_len);
        block = 0;
        if (mode != kPacked) {
            const int hu = mode == kPair ? a.heads / 2 : a.heads;
            block = rest / hu;
            rest -= block * hu;
        }
        h = rest * (mode == kPacked ? a.group : mode == kPair ? 2 : 1);
        t0 = 0;
        t1 = all_tiles();
    }
    __device__ void part(int rank, int ranks) {  // the rank's share of the key tiles
        const int per = (all_tiles() + ranks - 1) / ranks;
        t0 = min(all_tiles(), rank * per);
        t1 = min(all_tiles(), t0 + per);
    }
    __device__ int all_ext_tiles() const { return (ext_len + TKV - 1) / TKV; }
    __device__ int all_tiles() const { return all_ext_tiles() + (kv_len + TKV - 1) / TKV; }
    __device__ int first() const { return SPLIT ? t0 : 0; }
    __device__ int ext_tiles() const { return SPLIT ? max(0, min(t1, all_ext_tiles()) - t0) : all_ext_tiles(); }
    __device__ int tiles() const { return SPLIT ? t1 - t0 : all_tiles(); }
    __device__ int valid(int i) const {  // keys of its tile i, at least 1; 128 or more: all
        const int e = all_ext_tiles(), j = first() + i;
        return j < e ? ext_len - j * TKV : kv_len - (j - e) * TKV;
    }
    __device__ int q_tiles() const { return mode == kPacked ? 1 : mode == kPair || q_len > row0(1) ? 2 : 1; }
    __device__ int row0(int w) const {  // of the sequence; not of a packed unit
        return mode == kPair ? block * TQ : (2 * block + w) * TQ;
    }
    __device__ int head(int w) const { return h + (mode == kPair ? w : 0); }
    __device__ int rows(const Kv4Args& a, int w) const { return mode == kPacked ? q_len * a.group : q_len - row0(w); }
    // key tiles that warpgroup w takes: all, or of a packed unit every other one, from w
    __device__ int first_of(int w) const { return mode == kPacked ? w : 0; }
    __device__ int tiles_of(int w) const {
        return mode == kPacked ? (tiles() - first_of(w) + 1) / 2 : w < q_tiles() ? tiles() : 0;
    }
    __device__ int tile_of(int w, int i) const { return mode == kPacked ? 2 * i + first_of(w) : i; }
};

// Whether the phase of `parity` has completed, at once; and after half a microsecond's wait at most.
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool mbar_try_wait_brief(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 500;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            dst),
        "l"((uint64_t)map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}

// A run of bytes global -> shared (addresses and size multiples of 16), completing on the mbarrier.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

template <bool SPLIT>
__global__ void __launch_bounds__(T_THREADS, 1)
    k_kv4_attn_tc(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmQp,
                  const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const Kv4Args a) {
    constexpr uint32_t IDESC_S = idesc_f16_f32(TQ, TKV);
    constexpr uint32_t IDESC_O = idesc_f16_f32(TQ, 64) | (1u << 16);  // B (= V) MN-major
    extern __shared__ __align__(1024) uint8_t t_smem[];
    uint8_t* sQ = t_smem;                                   // slot q: tile 0 at q * 2 * T_QT_BYTES, tile 1 behind it
    uint8_t* sKV = sQ + T_QSLOTS * 2 * T_QT_BYTES;          // stage s: K at s * 2 * T_KV_BYTES, V behind it
    uint8_t* sRaw = sKV + T_STAGES * 2 * T_KV_BYTES;        // raw stage r at r * T_RAW_BYTES: K, V, parameters of K, of V
    uint64_t* bars = reinterpret_cast<uint64_t*>(sRaw + T_RAW_STAGES * T_RAW_BYTES);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + T_NBARS);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    float* join = reinterpret_cast<float*>(tmem_slot + 4);  // [w][128][2]: maximum and sum of a row
    int* cum = reinterpret_cast<int*>(join + 4 * TQ);       // [T_ENTRIES + 1]
    auto bar = [&](int i) { return smem_u32(bars + i); };
    if (smem_u32(t_smem) & 1023) {  // never expected: dynamic shared memory starts at the window's base
        pdl_wait();
        if (threadIdx.x == 0) atomicExch(a.err, kErrDrain);
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < T_QSLOTS; i++) {
            mbar_init(bar(B_QFULL + i), 1);
            mbar_init(bar(B_QEMPTY + i), 2);
        }
        for (int i = 0; i < T_STAGES; i++) {
            mbar_init(bar(B_KVFULL + i), T_EXPANDERS);
            mbar_init(bar(B_KVEMPTY + i), 2);
            mbar_init(bar(B_OWN + i), 1);
        }
        for (int w = 0; w < 2; w++) {
            mbar_init(bar(B_SFULL + w), 1);
            mbar_init(bar(B_SFREE + w), 4);
            mbar_init(bar(B_PFULL + w), 4);
            mbar_init(bar(B_ODONE + w), 1);
            mbar_init(bar(B_OFREE + w), 8);
            mbar_init(bar(B_DRAIN + w), 1);
        }
        for (int i = 0; i < T_RAW_STAGES; i++) {
            mbar_init(bar(B_RAWFULL + i), 1);
            mbar_init(bar(B_RAWEMPTY + i), T_EXPANDERS / 32);
        }
        mbar_init(bar(B_JOIN), 8);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 9) {
        tmem_alloc(smem_u32(tmem_slot), T_TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_entry();  // barriers and TMEM are set up; global memory is touched only after this
    const int run = (a.n_seqs + T_ENTRIES - 1) / T_ENTRIES;
    build_units(a, cum, run);
    const int n_units = cum[T_ENTRIES];
    Unit<SPLIT> un;
    // SPLIT: the CTAs of a cluster share out the key tiles of the cluster's first unit. Should there be more units than
    // clusters (max_q was too small), the first CTA goes on alone. Every warp passes the three barriers behind the first unit.
    const int ranks = SPLIT ? a.ranks : 1, rank = SPLIT ? (int)cluster_ctarank() : 0;
    const int u0 = blockIdx.x / ranks, u_step = gridDim.x / ranks;
    auto find_unit = [&](int u) {
        un.find(a, cum, run, u);
        if (SPLIT && u == u0) un.part(rank, ranks);
    };
    auto pass_barriers = [&]() {
        __syncwarp();
        for (int i = 0; i < 3; i++) cluster_sync();
    };

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(T_OTHER_REGS));
        if (warp == 8) {
            // ------------------------------------------------------------------ fetching (one thread)
            if (SPLIT || lane == 0) {
                int qi = 0, ri = 0;
                bool ok = true;
                auto unit = [&](int u) {
                    find_unit(u);
                    const int g = un.h / a.group, e_tiles = un.ext_tiles();
                    if (un.tiles() == 0) return;
                    const int qs = qi % T_QSLOTS;
                    if (!(ok = mbar_wait(bar(B_QEMPTY + qs), ((qi / T_QSLOTS) & 1) ^ 1, abort_flag))) return;
                    // whole tiles always: rows behind the sequence's end are other sequences', or zeros behind the buffer's;
                    // the lanes that they fall to are not used
                    const uint32_t dq = smem_u32(sQ + qs * 2 * T_QT_BYTES), full = bar(B_QFULL + qs);
                    const int row = un.q_start + (un.mode == kPacked ? 0 : un.row0(0));
                    if (un.mode == kPacked) {
                        mbar_arrive_expect_tx(full, TQ / a.group * a.group * 128);
                        tma_load_3d(dq, &tmQp, 0, un.h, row, full);
                    } else {
                        const int nq = un.q_tiles();
                        mbar_arrive_expect_tx(full, nq * T_QT_BYTES);
                        tma_load_2d(dq, &tmQ, un.head(0) * 64, row, full);
                        if (nq == 2) tma_load_2d(dq + T_QT_BYTES, &tmQ, un.head(1) * 64, un.q_start + un.row0(1), full);
                    }
                    qi++;
                    const size_t at = (size_t)g * a.seqs[un.sq].ext_cap;
                    const uint8_t *k4 = a.seqs[un.sq].k4 + at * 32, *v4 = a.seqs[un.sq].v4 + at * 32;
                    const d1_half *kp = a.seqs[un.sq].kp + at, *vp = a.seqs[un.sq].vp + at;
                    for (int j = 0; j < e_tiles; j++, ri++) {
                        const int rs = ri % T_RAW_STAGES;
                        if (!(ok = mbar_wait(bar(B_RAWEMPTY + rs), ((ri / T_RAW_STAGES) & 1) ^ 1, abort_flag))) return;
                        // whole 16-byte runs: up to 8 parameters, which the arrays hold (ext_cap is a multiple of 8)
                        const int n = min(un.valid(j), TKV);
                        const uint32_t codes = n * 32, pars = ((n + 7) & ~7) * 2;
                        const uint32_t dst = smem_u32(sRaw + rs * T_RAW_BYTES), landed = bar(B_RAWFULL + rs);
                        const size_t key = (size_t)(un.first() + j) * TKV;
                        mbar_arrive_expect_tx(landed, 2 * (codes + pars));
                        bulk_load(dst, k4 + key * 32, codes, landed);
                        bulk_load(dst + T_RAW_V, v4 + key * 32, codes, landed);
                        bulk_load(dst + T_RAW_KP, kp + key, pars, landed);
                        bulk_load(dst + T_RAW_VP, vp + key, pars, landed);
                    }
                };
                for (int u = u0; ok && u < n_units; u += u_step) {
                    if (lane == 0) unit(u);
                    if (SPLIT && u == u0) {
                        pass_barriers();
                        if (rank > 0) break;
                    }
                }
                if (lane == 0) {
                    if (!ok) record_err(a.err, abort_flag, kErrWaitEmpty);
                    // copies still in flight (only after an abort) land before the CTA exits
                    for (int i = ri > T_RAW_STAGES ? ri - T_RAW_STAGES : 0; i < ri; i++)
                        if (!mbar_wait_timed2(bar(B_RAWFULL + i % T_RAW_STAGES), (i / T_RAW_STAGES) & 1)) break;
                    for (int i = qi > T_QSLOTS ? qi - T_QSLOTS : 0; i < qi; i++)
                        if (!mbar_wait_timed2(bar(B_QFULL + i % T_QSLOTS), (i / T_QSLOTS) & 1)) break;
                }
            }
            __syncwarp();
        } else if (warp >= 10 && warp < 14) {
            // ------------------------------------------------------------------ expanding
            const int lt = (warp - 10) * 32 + lane;
            int ri = 0, ki = 0;  // cached tiles and tiles so far
            uint32_t own = 0;    // of each stage, the parity of its next partial tile of own rows
            bool ok = true;
            auto unit = [&](int u) {
                find_unit(u);
                const int g = un.h / a.group, nt = un.tiles(), e_tiles = un.ext_tiles();
                for (int j = 0; j < nt; j++, ki++) {
                    const int st = ki % T_STAGES, n = un.valid(j);
                    uint8_t* dK = sKV + st * 2 * T_KV_BYTES;
                    if (j < e_tiles) {
                        // the thread's 16-byte pieces: of K, then of V, those of keys lt / 2 and 64 more, half lt % 2
                        const int rs = ri % T_RAW_STAGES;
                        const uint8_t* raw = sRaw + rs * T_RAW_BYTES;
                        if (!(ok = __all_sync(D1_FULL_MASK, mbar_wait(bar(B_RAWFULL + rs), (ri / T_RAW_STAGES) & 1, abort_flag))))
                            return;
                        uint4 piece[4];
                        uint32_t par[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int r = (lt >> 1) + (i & 1) * 64;
                            piece[i] = *reinterpret_cast<const uint4*>(raw + (i >> 1) * T_RAW_V + r * 32 + (lt & 1) * 16);
                            par[i] = *reinterpret_cast<const uint16_t*>(raw + T_RAW_KP + (i >> 1) * (TKV * 2) + r * 2);
                            if (r >= n) {  // behind the cached keys: zeros
                                piece[i] = make_uint4(0, 0, 0, 0);
                                par[i] = 0;
                            }
                        }
                        __syncwarp();
                        if (lane == 0) mbar_arrive(bar(B_RAWEMPTY + rs));
                        ri++;
                        if (!(ok = __all_sync(D1_FULL_MASK, mbar_wait(bar(B_KVEMPTY + st), ((ki / T_STAGES) & 1) ^ 1, abort_flag))))
                            return;
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int r = (lt >> 1) + (i & 1) * 64;
                            uint8_t* row = dK + (i >> 1) * T_KV_BYTES + r * 128;
                            const uint32_t p2 = par[i] * 0x00010001u, step = kv4_step2(p2);
                            uint32_t z0, z1;
                            kv4_zero(p2, z0, z1);
                            const uint32_t word[4] = {piece[i].x, piece[i].y, piece[i].z, piece[i].w};
#pragma unroll
                            for (int q = 0; q < 4; q++) {
                                uint32_t x[4];
                                kv4_expand(word[q], z0, z1, x);
                                *reinterpret_cast<uint4*>(row + ((((lt & 1) * 4 + q) ^ (r & 7)) << 4)) =
                                    make_uint4(h2_mul(x[0], step), h2_mul(x[1], step), h2_mul(x[2], step), h2_mul(x[3], step));
                            }
                        }
                        fence_async_smem_cta();
                        mbar_arrive(bar(B_KVFULL + st));
                        continue;
                    }
                    if (!(ok = __all_sync(D1_FULL_MASK, mbar_wait(bar(B_KVEMPTY + st), ((ki / T_STAGES) & 1) ^ 1, abort_flag))))
                        return;
                    // own rows: a whole tile by TMA. Rows behind the sequence's end are others', or zeros behind the buffer's:
                    // their scores are masked, and their values, which P = 0 multiplies, are overwritten with zeros
                    const int row0 = un.kv_start + (un.first() + j - un.all_ext_tiles()) * TKV;
                    // (a barrier to each stage, so that it is armed again only when every thread has seen its phase before)
                    const uint32_t landed = bar((n >= TKV ? B_KVFULL : B_OWN) + st);
                    if (lt == 0) {
                        mbar_arrive_expect_tx(landed, 2 * T_KV_BYTES);
                        tma_load_2d(smem_u32(dK), &tmK, g * 64, row0, landed);
                        tma_load_2d(smem_u32(dK + T_KV_BYTES), &tmV, g * 64, row0, landed);
                    }
                    if (n >= TKV) {
                        if (lt != 0) mbar_arrive(landed);
                        continue;
                    }
                    if (!(ok = __all_sync(D1_FULL_MASK, mbar_wait(landed, (own >> st) & 1, abort_flag)))) return;
                    own ^= 1u << st;
                    for (int c = n * 8 + lt; c < TKV * 8; c += T_EXPANDERS)
                        *reinterpret_cast<uint4*>(dK + T_KV_BYTES + c * 16) = make_uint4(0, 0, 0, 0);
                    fence_async_smem_cta();
                    mbar_arrive(bar(B_KVFULL + st));
                }
            };
            for (int u = u0; ok && u < n_units; u += u_step) {
                unit(u);
                if (SPLIT && u == u0) {
                    pass_barriers();
                    if (rank > 0) break;
                }
            }
            if (!ok && lane == 0) record_err(a.err, abort_flag, kErrWaitEmpty);
            if (lt == 0 && !ok)  // copies still in flight land before the CTA exits
                mbar_wait_timed2(bar(B_OWN + ki % T_STAGES), (own >> ki % T_STAGES) & 1);
            if (lt == 0)
                for (int i = ki > T_STAGES ? ki - T_STAGES : 0; i < ki; i++)
                    if (!mbar_wait_timed2(bar(B_KVFULL + i % T_STAGES), (i / T_STAGES) & 1)) break;
            __syncwarp();
        } else if (warp == 9 || warp == 14) {
            // ------------------------------------------------------------------ MMA issuer of warpgroup w
            const int w = warp == 9 ? 0 : 1;
            if (SPLIT || lane == 0) {
                const uint32_t tS = tmem + w * T_WG_COLS, tP = tS + T_P_COL, tO = tS + T_O_COL;
                int cnt = 0, units = 0;  // key tiles and units of the warpgroup so far
                int qi = 0, ki = 0;
                bool ok = true;
                auto unit = [&](int u) {
                    find_unit(u);
                    const int nt = un.tiles(), mine = un.tiles_of(w);
                    if (nt == 0) return;
                    const int step = un.mode == kPacked ? 2 : 1, first = un.first_of(w);  // its key tiles
                    const int qs = qi % T_QSLOTS;
                    if (!(ok = mbar_wait(bar(B_QFULL + qs), (qi / T_QSLOTS) & 1, abort_flag))) return;
                    const uint64_t dq = smem_desc_k128(smem_u32(sQ + qs * 2 * T_QT_BYTES) + (un.mode == kPacked ? 0 : w * T_QT_BYTES));
                    auto kv_addr = [&](int j) { return smem_u32(sKV + ((ki + j) % T_STAGES) * 2 * T_KV_BYTES); };
                    // Sees its tiles up to j full, one after the other (wait: or only those that are, at once). Both issuers see
                    // every tile and give B_KVEMPTY an arrival for each, so that no stage's phase passes unseen: by its parity
                    // a phase cannot be told from the one two before it. A tile without MMAs of this issuer goes back at once.
                    int seen = 0;
                    auto see = [&](int j, bool wait) {
                        for (; seen <= j; seen++) {
                            const int x = ki + seen, st = x % T_STAGES;
                            if (!(wait ? mbar_wait(bar(B_KVFULL + st), (x / T_STAGES) & 1, abort_flag)
                                       : mbar_test(bar(B_KVFULL + st), (x / T_STAGES) & 1)))
                                return false;
                            if (mine == 0 || (step == 2 && (seen & 1) != w)) mbar_arrive(bar(B_KVEMPTY + st));
                        }
                        return true;
                    };
                    // S of its i-th tile, once the softmax has read the one before
                    auto issue_s = [&](int i) {
                        const int c = cnt + i;
                        if (!see(first + i * step, true)) return false;
                        if (c > 0 && !mbar_wait(bar(B_SFREE + w), (c - 1) & 1, abort_flag)) return false;
                        tc_fence_after();
                        const uint64_t dk = smem_desc_k128(kv_addr(first + i * step));
#pragma unroll
                        for (int k = 0; k < 4; k++) tc_mma_f16(tS, dq + 2 * k, dk + 2 * k, IDESC_S, k != 0);
                        tc_commit(bar(B_SFULL + w));
                        return true;
                    };
                    if (mine > 0) ok = issue_s(0);
                    for (int i = 0; i < mine && ok; i++) {
                        const int j = first + i * step, c = cnt + i;
                        // the next S computes while the softmax works on tile i; where its keys are late, P V goes first (it
                        // frees a stage that they may be waiting for)
                        bool s_next = i + 1 == mine;
                        const int next = s_next ? nt - 1 : j + step;  // meanwhile it sees the tiles up to its next, or the last ones
                        const uint64_t t0 = globaltimer_ns();
                        while (true) {
                            if (see(next, false) && !s_next) {
                                if (!(ok = issue_s(i + 1))) break;
                                s_next = true;
                            }
                            if (mbar_try_wait_brief(bar(B_PFULL + w), c & 1)) break;
                            if (*abort_flag || globaltimer_ns() - t0 > kWaitLimitNs) {
                                ok = false;
                                break;
                            }
                        }
                        if (!ok) break;
                        // the first P V of a unit overwrites O: the unit before must have been read
                        if (i == 0 && units > 0 && !(ok = mbar_wait(bar(B_OFREE + w), (units - 1) & 1, abort_flag))) break;
                        tc_fence_after();
                        const uint64_t dv = smem_desc_k128(kv_addr(j) + T_KV_BYTES);
#pragma unroll
                        for (int k = 0; k < TKV / 16; k++)
                            tc_mma_f16_ts(tO, tP + k * 8, dv + k * (2048 >> 4), IDESC_O, (i | k) != 0);
                        tc_commit(bar(B_ODONE + w));
                        tc_commit(bar(B_KVEMPTY + (ki + j) % T_STAGES));
                        if (!s_next && !(ok = issue_s(i + 1))) break;
                    }
                    if (!ok) return;
                    tc_commit(bar(B_QEMPTY + qs));
                    if (!(ok = see(nt - 1, true))) return;
                    ki += nt;
                    qi++;
                    cnt += mine;
                    units += mine > 0;
                };
                for (int u = u0; ok && u < n_units; u += u_step) {
                    if (lane == 0) unit(u);
                    if (SPLIT && u == u0) {
                        pass_barriers();
                        if (rank > 0) break;
                    }
                }
                if (lane == 0) {
                    if (!ok) record_err(a.err, abort_flag, kErrWaitFull);
                    tc_commit(bar(B_DRAIN + w));  // every issued MMA has completed before TMEM is released
                    if (!mbar_wait_timed2(bar(B_DRAIN + w), 0)) record_err(a.err, abort_flag, kErrDrain);
                }
            }
            __syncwarp();
        } else if (SPLIT) {  // the warp without a role
            if (u0 < n_units) pass_barriers();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(T_SOFTMAX_REGS));
        // ------------------------------------------------------------------ softmax
        const int w = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tS = tmem + w * T_WG_COLS + lane_off, tP = tS + T_P_COL, tO = tS + T_O_COL;
        // SPLIT: sums [w][row][R_LD], and maxima and weights [w][row][2], where the key tiles were
        float *part_o = reinterpret_cast<float*>(sKV), *part_ml = part_o + 2 * TQ * R_LD;
        int cnt = 0, njoin = 0;  // key tiles and packed units joined so far
        bool ok = true;
        for (int u = u0; ok && u < n_units; u += u_step) {
            find_unit(u);
            const bool packed = un.mode == kPacked, split = SPLIT && u == u0;
            if (!SPLIT && w == 1 && !packed && un.q_tiles() == 1) continue;
            // this thread's row: of the sequence and the head
            const int rows = un.rows(a, w), nt = un.tiles_of(w);
            const bool there = row < rows;
            const int q = packed ? row / a.group : un.row0(w) + row, h = packed ? un.h + row % a.group : un.head(w);
            const size_t grow = (size_t)(un.q_start + q);
            if (un.all_tiles() == 0) {  // no keys: zeros
                if (there && rank == 0 && !(packed && w == 1)) {
                    for (int i = 0; i < 8; i++)
                        *reinterpret_cast<uint4*>(a.O + grow * a.ldo + h * 64 + i * 8) = make_uint4(0, 0, 0, 0);
                    if (a.lse) a.lse[(size_t)h * a.lse_ld + grow] = -INFINITY;
                }
                if (split) {
                    pass_barriers();
                    if (rank > 0) break;
                }
                continue;
            }
            const bool idle = (warp & 3) * 32 >= rows;  // none of the warp's rows is there
            float m = -INFINITY, l = 0.f;
            for (int j = 0; j < nt; j++) {
                const int c = cnt + j;
                if (!(ok = __all_sync(D1_FULL_MASK, mbar_wait(bar(B_SFULL + w), c & 1, abort_flag)))) break;
                if (idle) {
                    // in step with the others, through every phase of B_ODONE: a wait for the last one alone could pass on the
                    // parity of the one before it, and O would be given back while the other warpgroup still reads it
                    if (lane == 0) mbar_arrive(bar(B_SFREE + w));
                    if (c > 0 && !(ok = __all_sync(D1_FULL_MASK, mbar_wait(bar(B_ODONE + w), (c - 1) & 1, abort_flag)))) break;
                    if (lane == 0) mbar_arrive(bar(B_PFULL + w));
                    continue;
                }
                tc_fence_after();
                uint32_t sr[TKV];
#pragma unroll
                for (int c32 = 0; c32 < TKV / 32; c32++)
                    tmem_ld32(tS + c32 * 32, *reinterpret_cast<uint32_t(*)[32]>(sr + c32 * 32));
                tc_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(B_SFREE + w));
                const int n = un.valid(un.tile_of(w, j));
                if (n < TKV) {
#pragma unroll
                    for (int i = 0; i < TKV; i++)
                        if (i >= n) sr[i] = __float_as_uint(-INFINITY);
                }
                // maximum of the raw scores (the scale is positive) in eight chains, scaled once
                float mx8[8];
#pragma unroll
                for (int e = 0; e < 8; e++) mx8[e] = fmaxf(__uint_as_float(sr[2 * e]), __uint_as_float(sr[2 * e + 1]));
#pragma unroll
                for (int i = 16; i < TKV; i += 16) {
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        mx8[e] = fmax3(mx8[e], __uint_as_float(sr[i + 2 * e]), __uint_as_float(sr[i + 2 * e + 1]));
                }
                const float mx = fmaxf(fmax3(mx8[0], mx8[1], mx8[2]), fmax3(mx8[3], mx8[4], fmax3(mx8[5], mx8[6], mx8[7]))) *
                                 a.scale_log2;
                float m_use = m, alpha = 1.f;
                if (j == 0) {
                    m_use = mx;
                } else if (mx > m + kLazyRescale) {
                    m_use = mx;
                    alpha = ex2(m - mx);
                }
                if (j > 0 && __any_sync(D1_FULL_MASK, alpha < 1.f)) {  // rare: O must hold P V up to the tile before
                    if (!(ok = __all_sync(D1_FULL_MASK, mbar_wait(bar(B_ODONE + w), (c - 1) & 1, abort_flag)))) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int o8 = 0; o8 < 8; o8++) {
                        uint32_t o[8];
                        tmem_ld8(tO + o8 * 8, o);
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < 8; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                        tmem_st8(tO + o8 * 8, o);
                    }
                }
                // P = 2^(s * scale - m), two scores at a time, and the row's sum in fp32. For the MMA, whose operands have 16
                // bits, P is rounded to fp16 (O is 2.9e-4 off, and 2.1e-4 by its own rounding alone). Nothing for the upper
                // half of a tile without keys there (26 x 176 rows over 7 keys 18.4 -> 17.5 us; in quarters 17.3, but
                // documents 252 -> 256).
                // (An eighth of the exponentials on the FMA pipe: documents 258 -> 253 us with a polynomial of degree 3, whose
                // 7.5e-5 showed in the log-sum-exp; 259 with degree 5.)
                const uint64_t sc2 = f2_pack(a.scale_log2, a.scale_log2), nm2 = f2_pack(-m_use, -m_use);
                uint64_t rs2[4];
#pragma unroll
                for (int e = 0; e < 4; e++) rs2[e] = f2_pack(0.f, 0.f);
                uint32_t pr[TKV / 2];
#pragma unroll
                for (int c64 = 0; c64 < 2; c64++) {
                    if (c64 == 1 && n <= 64) {  // none of these keys is there
#pragma unroll
                        for (int i = 32; i < 64; i++) pr[i] = 0;
                        break;
                    }
#pragma unroll
                    for (int i = 32 * c64; i < 32 * c64 + 32; i++) {
                        float x0, x1;
                        f2_unpack(f2_fma(f2_pack(__uint_as_float(sr[2 * i]), __uint_as_float(sr[2 * i + 1])), sc2, nm2), x0, x1);
                        const float p0 = ex2(x0), p1 = ex2(x1);
                        rs2[i & 3] = f2_add(rs2[i & 3], f2_pack(p0, p1));
                        pr[i] = pack_h2(p0, p1);
                    }
                }
                if (c > 0) {  // P V of the tile before has read the P columns
                    if (!(ok = __all_sync(D1_FULL_MASK, mbar_wait(bar(B_ODONE + w), (c - 1) & 1, abort_flag)))) break;
                    tc_fence_after();
                }
#pragma unroll
                for (int c32 = 0; c32 < TKV / 64; c32++)
                    tmem_st32(tP + c32 * 32, *reinterpret_cast<uint32_t(*)[32]>(pr + c32 * 32));
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(B_PFULL + w));
                float rs[8];
#pragma unroll
                for (int e = 0; e < 4; e++) f2_unpack(rs2[e], rs[2 * e], rs[2 * e + 1]);
                l = l * alpha + (((rs[0] + rs[1]) + (rs[2] + rs[3])) + ((rs[4] + rs[5]) + (rs[6] + rs[7])));
                m = m_use;
            }
            if (!SPLIT && !ok) break;
            cnt += nt;
            const bool mine = packed ? un.tiles() > 0 : nt > 0;  // this warpgroup finishes rows of the unit
            if (ok && nt > 0) ok = __all_sync(D1_FULL_MASK, mbar_wait(bar(B_ODONE + w), (cnt - 1) & 1, abort_flag));
            if (!SPLIT && !ok) break;
            if (split) {
                __syncwarp();
                cluster_sync();  // both warpgroups have done with the key tiles: their shared memory is free
            }
            // A packed unit's rows are in both warpgroups: they tell each other their maxima and sums, and each finishes half
            // of the dimensions. The shared memory is written again only behind a P V of a later unit, which waits for
            // B_OFREE, or not read (a warpgroup without tiles)
            float f0 = 1.f, f1 = 0.f;
            const bool two = packed && un.tiles_of(1) > 0;
            if (ok && mine && packed) {
                if (nt > 0) {
                    join[2 * (w * TQ + row)] = m;
                    join[2 * (w * TQ + row) + 1] = l;
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(B_JOIN));
                ok = __all_sync(D1_FULL_MASK, mbar_wait(bar(B_JOIN), njoin & 1, abort_flag));
                njoin++;
                m = join[2 * row];
                l = join[2 * row + 1];
                if (two) {
                    const float m1 = join[2 * (TQ + row)], l1 = join[2 * (TQ + row) + 1], both = fmaxf(m, m1);
                    f0 = ex2(m - both);
                    f1 = ex2(m1 - both);
                    l = l * f0 + l1 * f1;
                    m = both;
                }
            }
            if (!SPLIT && !ok) break;
            if (SPLIT && !split && !mine) continue;
            if (!SPLIT || (ok && mine)) {
                tc_fence_after();
                const float il = 1.f / l;
#pragma unroll 1
                for (int hd = packed ? w : 0; hd < (packed ? w + 1 : 2); hd++) {  // dimensions 32 hd .. 32 hd + 31
                    const uint32_t from = (packed ? tO - w * T_WG_COLS : tO) + 32 * hd;
                    uint32_t o[32];
                    tmem_ld32(from, o);
                    if (two) {
                        uint32_t o1[32];
                        tmem_ld32(from + T_WG_COLS, o1);
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; i++)
                            o[i] = __float_as_uint(__uint_as_float(o[i]) * f0 + __uint_as_float(o1[i]) * f1);
                    } else {
                        tc_wait_ld();
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0 && (packed || hd == 1)) {  // eight arrivals for either
                        mbar_arrive(bar(B_OFREE + (packed ? 0 : w)));
                        if (!packed) mbar_arrive(bar(B_OFREE + w));
                        if (two) mbar_arrive(bar(B_OFREE + 1));
                    }
                    if (!there) continue;
                    if (split) {  // unscaled sums, for the cluster
                        float* dst = part_o + ((packed ? 0 : w) * TQ + row) * R_LD + 32 * hd;
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            *reinterpret_cast<float4*>(dst + 4 * i) =
                                make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                                            __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
                    } else {
                        uint4* dst = reinterpret_cast<uint4*>(a.O + grow * a.ldo + h * 64 + 32 * hd);
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            uint32_t oh[4];
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                oh[e] = pack_h2(__uint_as_float(o[8 * i + 2 * e]) * il, __uint_as_float(o[8 * i + 2 * e + 1]) * il);
                            dst[i] = make_uint4(oh[0], oh[1], oh[2], oh[3]);
                        }
                    }
                }
                if (there && !(packed && w == 1)) {
                    if (split) {
                        part_ml[2 * (w * TQ + row)] = m;
                        part_ml[2 * (w * TQ + row) + 1] = l;
                    } else if (a.lse) {
                        a.lse[(size_t)h * a.lse_ld + grow] = (m + log2f(l)) * kLn2;
                    }
                }
            }
            if (split) {
                fence_async_smem_cta();  // (the next unit's copies come to the same place)
                __syncwarp();
                cluster_sync();  // the sums of every CTA are in its shared memory
                // join them, in their order: each CTA writes its share of the rows
                const int per = (un.all_tiles() + ranks - 1) / ranks, parts = (un.all_tiles() - 1) / per + 1, share = TQ / ranks;
                if (packed || w < un.q_tiles()) {
                    const int wp = packed ? 0 : w, team = packed ? 2 * TQ : TQ;
                    for (int i = packed ? w * TQ + row : row; i < share * 16; i += team) {
                        const int r = rank * share + (i >> 4), d = (i & 15) * 4;
                        if (r >= rows) break;
                        float pm[R_CLUSTER], pl[R_CLUSTER];
                        float4 v[R_CLUSTER];
#pragma unroll
                        for (int c = 0; c < R_CLUSTER; c++) {
                            pm[c] = -INFINITY;
                            pl[c] = 0.f;
                            v[c] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (c < parts) {
                                pm[c] = ld_cluster_f32(mapa_shared(smem_u32(part_ml + 2 * (wp * TQ + r)), c));
                                pl[c] = ld_cluster_f32(mapa_shared(smem_u32(part_ml + 2 * (wp * TQ + r) + 1), c));
                                v[c] = ld_cluster_f32x4(mapa_shared(smem_u32(part_o + (wp * TQ + r) * R_LD + d), c));
                            }
                        }
                        float M = -INFINITY, L = 0.f;
#pragma unroll
                        for (int c = 0; c < R_CLUSTER; c++) M = fmaxf(M, pm[c]);
                        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                        for (int c = 0; c < R_CLUSTER; c++) {
                            if (c >= parts) break;
                            const float f = ex2(pm[c] - M);
                            L += f * pl[c];
                            x.x += f * v[c].x;
                            x.y += f * v[c].y;
                            x.z += f * v[c].z;
                            x.w += f * v[c].w;
                        }
                        const float il = 1.f / L;
                        const int qr = un.q_start + (packed ? r / a.group : un.row0(w) + r);
                        const int hr = packed ? un.h + r % a.group : un.head(w);
                        *reinterpret_cast<uint2*>(a.O + (size_t)qr * a.ldo + hr * 64 + d) =
                            make_uint2(pack_h2(x.x * il, x.y * il), pack_h2(x.z * il, x.w * il));
                        if (a.lse && d == 0) a.lse[(size_t)hr * a.lse_ld + qr] = (M + log2f(L)) * kLn2;
                    }
                }
                __syncwarp();
                cluster_sync();  // the other CTAs have read this one's sums
                if (rank > 0) break;
            }
        }
        if (!ok && lane == 0) record_err(a.err, abort_flag, kErrWaitAccFull);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem, T_TMEM_COLS);
    }
}

// ------------------------------------------------------------------------------------------------ mass, few rows
// S^T = K Q^T on m16n8k16: a warp holds 16 * MT keys as A operands (whole numbers code - zero, as above) and goes over the
// packed query rows 8 at a time, adding exp(s - lse) into its keys' sums; four lanes share a key at the end. The sequences
// that share a mass array are taken by the first of them whose cache is in order, in the table's order. What bounds it are
// latencies: of the table, of the codes (both at once where the table has 256 entries at most), and of 8 rows after 8 rows.
template <int MT>
__global__ void __launch_bounds__(256, 2) k_kv4_mass_rows(const Kv4Args a) {
    constexpr int KEYS = 16 * MT * 8;   // of a CTA of 8 warps
    constexpr bool AHEAD = MT < 4;      // the next 8 rows on their way meanwhile; of 64 keys the registers do not hold them
    __shared__ int2 peers[256];         // of 256 sequences: first row and rows
    __shared__ uint32_t same[8];        // and which are of this mass array
    pdl_entry();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = lane >> 2, t = lane & 3, g = blockIdx.y;
    const int q_first = r / a.group, h_first = g * a.group + r % a.group, q_step = 8 / a.group, h_step = 8 % a.group;
    const int h_end = (g + 1) * a.group;
    for (int sq = blockIdx.z; sq < a.n_seqs; sq += gridDim.z) {
        const D1Kv4Seq s = a.seqs[sq];
        if (!s.mass) continue;
        if (!kv4_seq_ok(s) || ((uintptr_t)s.mass & 3)) {
            if (tid == 0) atomicExch(a.err, kErrTable);
            continue;
        }
        int listed = -1;  // which 256 sequences the list holds
        // lists sequences b0 .. b0 + 255; whether one before sq with a cache in order, which then takes the mass array, is
        // among them
        auto list = [&](int b0) {
            if (listed == b0) return false;
            if (listed >= 0) __syncthreads();  // the list has been read
            listed = b0;
            const int j = b0 + tid;
            bool mine = false, before = false;
            if (j < a.n_seqs) {
                const D1Kv4Seq p = a.seqs[j];
                mine = p.mass == s.mass;
                before = mine && j < sq && kv4_seq_ok(p);
                if (mine && (!kv4_seq_ok(p) || p.k4 != s.k4 || p.ext_len != s.ext_len || p.ext_cap != s.ext_cap ||
                             !rows_ok(p.q_start, p.q_len, a.q_rows))) {
                    atomicExch(a.err, kErrTable);
                    mine = false;
                }
                peers[tid] = make_int2(p.q_start, p.q_len);
            }
            const uint32_t v = __ballot_sync(D1_FULL_MASK, mine);
            if (lane == 0) same[warp] = v;
            return __syncthreads_or(before) != 0;
        };
        const uint16_t* kp = reinterpret_cast<const uint16_t*>(s.kp) + (size_t)g * s.ext_cap;
        const uint8_t* k4 = s.k4 + (size_t)g * s.ext_cap * 32;
        bool others = false;
        for (int k0 = blockIdx.x * KEYS; k0 < s.ext_len && !others; k0 += gridDim.x * KEYS) {
            const int key0 = k0 + warp * (16 * MT);
            uint2 code[MT][2];
            uint32_t par[MT][2];
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const int key = min(key0 + mt * 16 + hf * 8 + r, s.ext_len - 1);
                    code[mt][hf] = __ldg(reinterpret_cast<const uint2*>(k4 + (size_t)key * 32) + t);
                    par[mt][hf] = __ldg(kp + key);
                }
            others = list(0);
            if (others) break;
            uint32_t ka[MT][4][4];
            float st[MT][2], sum[MT][2];
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    uint32_t z0, z1, x[4], y[4];
                    kv4_zero(par[mt][hf] * 0x00010001u, z0, z1);
                    kv4_expand(code[mt][hf].x, z0, z1, x);
                    kv4_expand(code[mt][hf].y, z0, z1, y);
                    ka[mt][0][hf] = x[0];
                    ka[mt][0][2 + hf] = x[1];
                    ka[mt][1][hf] = x[2];
                    ka[mt][1][2 + hf] = x[3];
                    ka[mt][2][hf] = y[0];
                    ka[mt][2][2 + hf] = y[1];
                    ka[mt][3][hf] = y[2];
                    ka[mt][3][2 + hf] = y[3];
                    st[mt][hf] = kv4_step(par[mt][hf]) * a.scale_log2;
                    sum[mt][hf] = 0.f;
                }
            bool any = false;
            for (int b0 = 0; b0 < a.n_seqs && !others; b0 += 256) {  // the sequences of this mass array, in order
                others = list(b0);
                for (int i = 0; i < 8 && !others; i++)
                    for (uint32_t left = same[i]; left; left &= left - 1) {
                        const int2 p = peers[32 * i + __ffs(left) - 1];
                        any = true;
                        const uint32_t n_rows = (uint32_t)p.y * (uint32_t)a.group;
                        int q = p.x + q_first, h = h_first;  // of the packed row fetched next
                        uint4 n0, n1;
                        float nl;
                        auto fetch = [&](uint32_t row) {
                            n0 = n1 = make_uint4(0, 0, 0, 0);
                            nl = -INFINITY;
                            if (row < n_rows) {
                                const uint4* src = reinterpret_cast<const uint4*>(a.Q + (size_t)q * a.ldq + h * 64 + 16 * t);
                                n0 = __ldg(src);
                                n1 = __ldg(src + 1);
                                nl = __ldg(a.lse + (size_t)h * a.lse_ld + q);
                            }
                            q += q_step;
                            h += h_step;
                            if (h >= h_end) {
                                h -= a.group;
                                q++;
                            }
                        };
                        if (AHEAD) fetch(r);
                        for (uint32_t base = 0; base < n_rows; base += 8) {
                            if (!AHEAD) fetch(base + r);
                            uint4 x0 = n0, x1 = n1;
                            float lse = nl * kLog2e;  // in log2; +inf: adds nothing
                            if (lse == -INFINITY) {   // whatever the row holds
                                lse = INFINITY;
                                x0 = x1 = make_uint4(0, 0, 0, 0);
                            }
                            if (AHEAD) fetch(base + 8 + r);
                            const float l0 = __shfl_sync(D1_FULL_MASK, lse, 8 * t), l1 = __shfl_sync(D1_FULL_MASK, lse, 8 * t + 4);
#pragma unroll
                            for (int mt = 0; mt < MT; mt++) {
                                float c[4];
                                mma16816_first(c, ka[mt][0], x0.x, x0.y);
                                mma16816(c, ka[mt][1], x0.z, x0.w);
                                mma16816(c, ka[mt][2], x1.x, x1.y);
                                mma16816(c, ka[mt][3], x1.z, x1.w);
                                sum[mt][0] += ex2(c[0] * st[mt][0] - l0) + ex2(c[1] * st[mt][0] - l1);
                                sum[mt][1] += ex2(c[2] * st[mt][1] - l0) + ex2(c[3] * st[mt][1] - l1);
                            }
                        }
                    }
            }
            if (others) break;
            float* mass = s.mass + (size_t)g * s.ext_cap;
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    float v = sum[mt][hf];
                    v += __shfl_xor_sync(D1_FULL_MASK, v, 1);
                    v += __shfl_xor_sync(D1_FULL_MASK, v, 2);
                    const int key = key0 + mt * 16 + hf * 8 + r;
                    if (any && t == 0 && key < s.ext_len) mass[key] = a.accumulate ? mass[key] + v : v;
                }
        }
        if (sq + (int)gridDim.z < a.n_seqs) __syncthreads();  // the list has been read, before the next sequence's is written
    }
}

// ------------------------------------------------------------------------------------------------ mass, many rows
// tcgen05 form: S^T = K Q^T, so that a key is a TMEM lane and its sum over the query rows stays in one thread. Persistent
// CTAs loop over units of 128 keys of one (cache, kv head): the keys are expanded once into shared memory, then tiles of
// up to 256 query columns (a block of rows of every head of the kv head) pass by. The bound is the exponentials: 1 per
// key and column, some of them on the FMA pipe.
// Warps:
//   0-15       four warpgroups share every tile (two of its eight 32-column pieces each): S from TMEM, where the next
//              tile's S is computed meanwhile, exp2(s * scale - lse), summed in fp32; one pair of exponentials in eight on
//              the FMA pipe. At the unit's end three pass their sums to the first through shared memory. (Two documents of
//              2048 rows over 8192 keys: 78 us. Compared while it took 91: 98 with two warpgroups and the next piece's
//              load on its way, 97 with both pieces loaded at once, 93 without the FMA pipe, 94 and 99 with a quarter and
//              three eighths there)
//   16, 18, 19 loaders: the keys' codes, expanded; query tiles by TMA from a view of [row][head][64], always whole; the
//              columns' -lse (behind the end and for rows that add nothing: -inf). Such rows are wiped out in shared
//              memory, so that a NaN in padding stays there (masking their scores instead cost the exponentials' loop its
//              schedule: 85 us)
//   17         TMEM, and the MMAs from one thread
constexpr int MQ = 256, MK = 128, M_STAGES = 4, M_LOADERS = 3, M_WGS = 4, M_THREADS = 128 * M_WGS + 128;
constexpr int M_Q_BYTES = MQ * 128, M_K_BYTES = MK * 128;
enum : int {
    MB_KFULL = 0,                    // [2] the unit's keys
    MB_KEMPTY = MB_KFULL + 2,        // [2]
    MB_QFULL = MB_KEMPTY + 2,        // [stage]
    // [stage] the tile has been read: its lse by 16 warps, which wait for S, and so for the MMA, before they arrive. (A
    // loader looks at every third tile's phase only. As the warps arrive tile after tile, the phase of the stage's use
    // before is then over, and the parity that it waits on is not that one's.)
    MB_QEMPTY = MB_QFULL + M_STAGES,
    MB_SFULL = MB_QEMPTY + M_STAGES, // [buffer] S of a tile is in TMEM
    MB_SFREE = MB_SFULL + 2,         // [buffer] (16 warps)
    MB_SUM = MB_SFREE + 2,           // [2] the other warpgroups' sums are in shared memory (12 warps)
    MB_SUMFREE = MB_SUM + 2,         // [2] (4 warps)
    MB_LANDED = MB_SUMFREE + 2,      // [loader] a query tile with rows to wipe out
    MB_DRAIN = MB_LANDED + M_LOADERS,
    M_NBARS = MB_DRAIN + 1
};

// What the roles need of up to M_SEQS sequences, in shared memory: units (key tiles of 128 of the caches that belong to a
// sequence, for each kv head) before each, query rows, cached keys, and the next sequence of the same mass array. The
// sequences that share a mass array belong to the first of them whose cache is in order, which they must share, too.
constexpr int M_SEQS = 256;
struct MassTable {
    const float* mass[M_SEQS];
    int cum[M_SEQS + 1], q_start[M_SEQS], q_len[M_SEQS], ext_len[M_SEQS], next[M_SEQS];
};

constexpr int M_SMEM = 2 * M_K_BYTES + M_STAGES * (M_Q_BYTES + MQ * 4) + (2 * (M_WGS - 1) + 1) * MK * 4 + (int)sizeof(MassTable) +
                       M_NBARS * 8 + 16;
static_assert(M_SMEM <= 232448 && sizeof(MassTable) % 8 == 0, "shared memory of the tcgen05 mass kernel");

// Fills the table; ends with a barrier. Every thread of the CTA takes part.
__device__ __forceinline__ void build_mass_table(const Kv4Args& a, MassTable& tb, int n) {
    const int tid = threadIdx.x, kv_heads = a.heads / a.group;
    for (int i = tid; i < n; i += blockDim.x) {
        const D1Kv4Seq& s = a.seqs[i];
        tb.mass[i] = s.mass;
        tb.q_start[i] = s.q_start;
        tb.q_len[i] = s.q_len;
        tb.ext_len[i] = s.ext_len;
    }
    __syncthreads();
    for (int i = tid; i < M_SEQS; i += blockDim.x) {
        int units = 0;
        if (i < n && tb.mass[i]) {
            const D1Kv4Seq s = a.seqs[i];
            bool owner = true;
            int first = i, next = n;
            for (int j = 0; j < i && owner; j++)
                if (tb.mass[j] == s.mass && kv4_seq_ok(a.seqs[j])) {
                    owner = false;
                    first = j;
                }
            for (int j = n - 1; j > i; j--)
                if (tb.mass[j] == s.mass) next = j;
            tb.next[i] = next;
            const D1Kv4Seq& o = a.seqs[first];
            const bool bad = !kv4_seq_ok(s) || ((uintptr_t)s.mass & 3);
            if (bad || !rows_ok(s.q_start, s.q_len, a.q_rows) ||
                (!owner && (o.k4 != s.k4 || o.ext_len != s.ext_len || o.ext_cap != s.ext_cap))) {
                atomicExch(a.err, kErrTable);
                tb.q_len[i] = -1;  // its rows do not count
            }
            if (owner && !bad) units = (s.ext_len + MK - 1) / MK * kv_heads;
        }
        tb.cum[i + 1] = units;
    }
    if (tid == 0) tb.cum[0] = 0;
    __syncthreads();
    if (tid < 32) {
        constexpr int PER = M_SEQS / 32;
        int v[PER], sum = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) sum += v[i] = tb.cum[1 + tid * PER + i];
        int upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(D1_FULL_MASK, upto, o);
            if (tid >= o) upto += x;
        }
        upto -= sum;
#pragma unroll
        for (int i = 0; i < PER; i++) tb.cum[1 + tid * PER + i] = upto += v[i];
    }
    __syncthreads();
}

// The units of a CTA and, within each, its query tiles, walked alike by every role: unit u is a sequence, a tile of its
// keys and a kv head, the heads fastest.
struct MassWalk {
    int sq, g, kt;
    int peer, q_start, q_len, row0;  // the tile: rows row0 .. row0 + rows() - 1 of sequence `peer`, every head of g
    int block, kv_heads;             // rows of a whole tile
    bool any;                        // a sequence counted, be it without rows
    int entry;
    int rank, ranks;                 // every ranks-th tile, from the rank's

    __device__ MassWalk(const Kv4Args& a) : block(MQ / a.group), kv_heads(a.heads / a.group), entry(0) {}
    __device__ void find(const MassTable& tb, int u, int rank_, int ranks_) {  // u at or behind the one before
        rank = rank_;
        ranks = ranks_;
        while (tb.cum[entry + 1] <= u) entry++;
        sq = entry;
        const int rest = u - tb.cum[entry];
        kt = rest / kv_heads;
        g = rest - kt * kv_heads;
        peer = -1;
        q_len = row0 = 0;
        any = false;
    }
    __device__ bool next_tile(const MassTable& tb, int n) {
        int ahead = peer < 0 ? rank : ranks - 1;  // tiles of the others before it
        row0 += block;
        while (true) {
            while (row0 >= q_len) {
                peer = peer < 0 ? sq : tb.next[peer];
                if (peer >= n) return false;
                q_start = tb.q_start[peer];
                q_len = tb.q_len[peer];
                row0 = 0;
                any |= q_len >= 0;
            }
            if (ahead-- == 0) return true;
            row0 += block;
        }
    }
    __device__ int rows() const { return min(block, q_len - row0); }
};

template <bool SPLIT>
__global__ void __launch_bounds__(M_THREADS, 1) k_kv4_mass_tc(const __grid_constant__ CUtensorMap tmQp, const Kv4Args a) {
    extern __shared__ __align__(1024) uint8_t m_smem[];
    uint8_t* sK = m_smem;                                                          // [2][128 keys]
    uint8_t* sQ = sK + 2 * M_K_BYTES;                                              // [stage][256 columns]
    float* sL = reinterpret_cast<float*>(sQ + M_STAGES * M_Q_BYTES);               // [stage][256]: -lse in log2
    float* sSum = sL + M_STAGES * MQ;                                              // [2][warpgroup - 1][128]
    float* sPart = sSum + 2 * (M_WGS - 1) * MK;                                    // [128] SPLIT: the CTA's sums
    MassTable& tb = *reinterpret_cast<MassTable*>(sPart + MK);
    uint64_t* bars = reinterpret_cast<uint64_t*>(&tb + 1);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + M_NBARS);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    auto bar = [&](int i) { return smem_u32(bars + i); };
    if (smem_u32(m_smem) & 1023) {  // never expected: dynamic shared memory starts at the window's base
        pdl_wait();
        if (threadIdx.x == 0) atomicExch(a.err, kErrDrain);
        return;
    }
    constexpr int M_WARP = 4 * M_WGS + 1;  // the MMA warp
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(bar(MB_KFULL + i), 32 * M_LOADERS);
            mbar_init(bar(MB_KEMPTY + i), 1);
            mbar_init(bar(MB_SFULL + i), 1);
            mbar_init(bar(MB_SFREE + i), 4 * M_WGS);
            mbar_init(bar(MB_SUM + i), 4 * (M_WGS - 1));
            mbar_init(bar(MB_SUMFREE + i), 4);
        }
        for (int i = 0; i < M_STAGES; i++) {
            mbar_init(bar(MB_QFULL + i), 32);
            mbar_init(bar(MB_QEMPTY + i), 4 * M_WGS);
        }
        for (int i = 0; i < M_LOADERS; i++) mbar_init(bar(MB_LANDED + i), 1);
        mbar_init(bar(MB_DRAIN), 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == M_WARP) {
        tmem_alloc(smem_u32(tmem_slot), T_TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_entry();  // barriers and TMEM are set up; global memory is touched only after this
    const int n = a.n_seqs;
    build_mass_table(a, tb, n);
    const int n_units = tb.cum[M_SEQS];
    MassWalk wk(a);
    int nu = 0, ti = 0;  // units and tiles so far
    bool ok = true;
    auto wait = [&](int b, uint32_t parity) {
        return __all_sync(D1_FULL_MASK, mbar_wait(bar(b), parity, abort_flag)) != 0;
    };
    // SPLIT: the CTAs of a cluster share out the query tiles of the cluster's first unit. Should there be more units than
    // clusters (max_len was too small), the first CTA goes on alone. Every warp passes the two barriers behind that unit.
    const int ranks = SPLIT ? a.ranks : 1, rank = SPLIT ? (int)cluster_ctarank() : 0;
    const int u0 = blockIdx.x / ranks, u_step = gridDim.x / ranks;
    auto find_unit = [&](int u) {
        const bool split = SPLIT && u == u0;
        wk.find(tb, u, split ? rank : 0, split ? ranks : 1);
    };
    auto each_unit = [&](auto&& unit) {
        for (int u = u0; ok && u < n_units; u += u_step, nu++) {
            unit(u);
            if (SPLIT && u == u0) {
                __syncwarp();
                cluster_sync();  // the CTAs' sums are in their shared memory
                if (rank == 0 && warp < 4 && ok) {
                    const int row = warp * 32 + lane;
                    float all = sPart[row];
                    for (int c = 1; c < ranks; c++) all += ld_cluster_f32(mapa_shared(smem_u32(sPart + row), c));
                    const long long key = (long long)wk.kt * MK + row;
                    if (wk.any && key < tb.ext_len[wk.sq]) {
                        float* m = a.seqs[wk.sq].mass + (size_t)wk.g * a.seqs[wk.sq].ext_cap + key;
                        *m = a.accumulate ? *m + all : all;
                    }
                }
                __syncwarp();
                cluster_sync();  // and have been read
                if (rank > 0) break;
            }
        }
    };

    if (warp == M_WARP - 1 || warp > M_WARP) {
        // ------------------------------------------------------------------ loaders
        const int lw = warp < M_WARP ? 0 : warp - M_WARP, lt = lw * 32 + lane;
        int wiped = 0;  // tiles with rows wiped out so far
        const int inv = (65536 + a.group - 1) / a.group;  // c / group = c * inv >> 16 for c < 256: off by less than 1 / group
        each_unit([&](int u) {
            find_unit(u);
            const size_t at = (size_t)wk.g * a.seqs[wk.sq].ext_cap;
            const uint8_t* k4 = a.seqs[wk.sq].k4 + at * 32;
            const uint16_t* kp = reinterpret_cast<const uint16_t*>(a.seqs[wk.sq].kp) + at;
            const int ext_len = tb.ext_len[wk.sq];
            constexpr int PIECES = (2 * MK + 32 * M_LOADERS - 1) / (32 * M_LOADERS);
            uint4 piece[PIECES];
            uint32_t par[PIECES];
#pragma unroll
            for (int i = 0; i < PIECES; i++) {
                const int c = lt + i * 32 * M_LOADERS, key = wk.kt * MK + (c >> 1);
                piece[i] = make_uint4(0, 0, 0, 0);
                par[i] = 0;  // step 0: zeros
                if (c < 2 * MK && key < ext_len) {
                    piece[i] = __ldg(reinterpret_cast<const uint4*>(k4 + (size_t)key * 32) + (c & 1));
                    par[i] = __ldg(kp + key);
                }
            }
            if (!(ok = wait(MB_KEMPTY + (nu & 1), ((nu >> 1) & 1) ^ 1))) return;
            uint8_t* dK = sK + (nu & 1) * M_K_BYTES;
#pragma unroll
            for (int i = 0; i < PIECES; i++) {
                const int c = lt + i * 32 * M_LOADERS, r = c >> 1;
                if (c >= 2 * MK) continue;
                const uint32_t p2 = par[i] * 0x00010001u, step = kv4_step2(p2);
                uint32_t z0, z1;
                kv4_zero(p2, z0, z1);
                const uint32_t word[4] = {piece[i].x, piece[i].y, piece[i].z, piece[i].w};
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    uint32_t v[4];
                    kv4_expand(word[q], z0, z1, v);
                    *reinterpret_cast<uint4*>(dK + r * 128 + ((((c & 1) * 4 + q) ^ (r & 7)) << 4)) =
                        make_uint4(h2_mul(v[0], step), h2_mul(v[1], step), h2_mul(v[2], step), h2_mul(v[3], step));
                }
            }
            fence_async_smem_cta();
            mbar_arrive(bar(MB_KFULL + (nu & 1)));
            for (; wk.next_tile(tb, n); ti++) {
                if (ti % M_LOADERS != lw) continue;  // the warps take the tiles in turn: their latencies overlap
                const int st = ti % M_STAGES, cols = wk.rows() * a.group, pad = (cols + 31) & ~31;
                const int row = wk.q_start + wk.row0, h0 = wk.g * a.group;
                float l[MQ / 32];
#pragma unroll
                for (int i = 0; i < MQ / 32; i++) {
                    const int c = lane + 32 * i, r = c * inv >> 16;
                    l[i] = -INFINITY;
                    if (c < cols) l[i] = __ldg(a.lse + (size_t)(h0 + c - r * a.group) * a.lse_ld + row + r);
                }
                bool wipe = false;  // rows that add nothing, whatever they hold: zeros in their place
#pragma unroll
                for (int i = 0; i < MQ / 32; i++) wipe |= lane + 32 * i < cols && l[i] == -INFINITY;
                wipe = __any_sync(D1_FULL_MASK, wipe);
                if (!(ok = wait(MB_QEMPTY + st, ((ti / M_STAGES) & 1) ^ 1))) return;
#pragma unroll
                for (int i = 0; i < MQ / 32; i++)
                    if (32 * i < pad) sL[st * MQ + lane + 32 * i] = l[i] == -INFINITY ? -INFINITY : -l[i] * kLog2e;
                const uint32_t full = bar(MB_QFULL + st), landed = wipe ? bar(MB_LANDED + lw) : full;
                if (lane == 0) {
                    mbar_arrive_expect_tx(landed, wk.block * a.group * 128);
                    tma_load_3d(smem_u32(sQ + st * M_Q_BYTES), &tmQp, 0, h0, row, landed);
                }
                if (wipe) {
                    if (!(ok = wait(MB_LANDED + lw, wiped & 1))) return;
                    wiped++;
#pragma unroll
                    for (int i = 0; i < MQ / 32; i++)
                        if (lane + 32 * i < cols && l[i] == -INFINITY)
                            for (int q = 0; q < 8; q++)
                                *reinterpret_cast<uint4*>(sQ + st * M_Q_BYTES + (lane + 32 * i) * 128 + q * 16) =
                                    make_uint4(0, 0, 0, 0);
                    fence_async_smem_cta();
                }
                if (wipe || lane != 0) mbar_arrive(full);
            }
        });
        if (!ok && lane == 0) record_err(a.err, abort_flag, kErrWaitEmpty);
        if (lane == 0 && !ok) mbar_wait_timed2(bar(MB_LANDED + lw), wiped & 1);
        if (lane == 0)  // TMA copies still in flight (only after an abort) land before the CTA exits
            for (int i = ti > M_STAGES ? ti - M_STAGES : 0; i < ti; i++)
                if (!mbar_wait_timed2(bar(MB_QFULL + i % M_STAGES), (i / M_STAGES) & 1)) break;
    } else if (warp == M_WARP) {
        // ------------------------------------------------------------------ MMA issuer (lane 0)
        each_unit([&](int u) {
            find_unit(u);
            if (!(ok = wait(MB_KFULL + (nu & 1), (nu >> 1) & 1))) return;
            const uint32_t k_addr = smem_u32(sK + (nu & 1) * M_K_BYTES);
            for (; wk.next_tile(tb, n); ti++) {
                const int st = ti % M_STAGES, w = ti & 1, pad = (wk.rows() * a.group + 31) & ~31;
                if (!(ok = wait(MB_QFULL + st, (ti / M_STAGES) & 1))) return;
                if (ti > 1 && !(ok = wait(MB_SFREE + w, ((ti >> 1) - 1) & 1))) return;
                tc_fence_after();
                if (lane == 0) {
                    const uint32_t q_addr = smem_u32(sQ + st * M_Q_BYTES), idesc = idesc_f16_f32(MK, pad);
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        tc_mma_f16(tmem + w * MQ, smem_desc_k128(k_addr + k * 32), smem_desc_k128(q_addr + k * 32), idesc, k != 0);
                    tc_commit(bar(MB_SFULL + w));
                }
                __syncwarp();
            }
            if (lane == 0) tc_commit(bar(MB_KEMPTY + (nu & 1)));
            __syncwarp();
        });
        if (lane == 0) {
            if (!ok) record_err(a.err, abort_flag, kErrWaitFull);
            tc_commit(bar(MB_DRAIN));  // every issued MMA has completed before TMEM is released
            if (!mbar_wait_timed2(bar(MB_DRAIN), 0)) record_err(a.err, abort_flag, kErrDrain);
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------------ exponentials and sums
        const int wg = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t tS = tmem + 32 * wg + ((uint32_t)((warp & 3) * 32) << 16);
        const uint64_t sc2 = f2_pack(a.scale_log2, a.scale_log2);
        each_unit([&](int u) {
            find_unit(u);
            uint64_t sum[4];
#pragma unroll
            for (int e = 0; e < 4; e++) sum[e] = f2_pack(0.f, 0.f);
            for (; wk.next_tile(tb, n); ti++) {
                const int st = ti % M_STAGES, b = ti & 1, pad = (wk.rows() * a.group + 31) & ~31;
                if (!(ok = wait(MB_QFULL + st, (ti / M_STAGES) & 1))) return;  // the lse
                if (!(ok = wait(MB_SFULL + b, (ti >> 1) & 1))) return;
                tc_fence_after();
                const int cols = wk.rows() * a.group;
                for (int c0 = 32 * wg; c0 < pad; c0 += 32 * M_WGS) {
                    const float4* l4 = reinterpret_cast<const float4*>(sL + st * MQ + c0);
                    uint32_t y[32];
                    tmem_ld32(tS + b * MQ + (c0 - 32 * wg), y);
                    tc_wait_ld();
                    if (c0 + 32 > cols) {  // columns of other sequences' rows, or of none: whatever they hold, a score of 0
#pragma unroll
                        for (int i = 0; i < 32; i++)
                            if (c0 + i >= cols) y[i] = 0;
                    }
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float4 l = l4[i];
                        float x[4], p[4];
                        f2_unpack(f2_fma(f2_pack(__uint_as_float(y[4 * i]), __uint_as_float(y[4 * i + 1])), sc2,
                                         f2_pack(l.x, l.y)), x[0], x[1]);
                        f2_unpack(f2_fma(f2_pack(__uint_as_float(y[4 * i + 2]), __uint_as_float(y[4 * i + 3])), sc2,
                                         f2_pack(l.z, l.w)), x[2], x[3]);
                        p[0] = ex2(x[0]);
                        p[1] = ex2(x[1]);
                        if (i % 4 == 3) {
                            ex2_fma2(x[2], x[3], p[2], p[3]);
                        } else {
                            p[2] = ex2(x[2]);
                            p[3] = ex2(x[3]);
                        }
                        sum[(2 * i) & 3] = f2_add(sum[(2 * i) & 3], f2_pack(p[0], p[1]));
                        sum[(2 * i + 1) & 3] = f2_add(sum[(2 * i + 1) & 3], f2_pack(p[2], p[3]));
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(bar(MB_SFREE + b));
                    mbar_arrive(bar(MB_QEMPTY + st));
                }
            }
            float v[8];
#pragma unroll
            for (int e = 0; e < 4; e++) f2_unpack(sum[e], v[2 * e], v[2 * e + 1]);
            const float mine = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
            const int slot = nu & 1;
            if (wg > 0) {
                if (!(ok = wait(MB_SUMFREE + slot, ((nu >> 1) & 1) ^ 1))) return;
                sSum[(slot * (M_WGS - 1) + wg - 1) * MK + row] = mine;
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(MB_SUM + slot));
            } else {
                if (!(ok = wait(MB_SUM + slot, (nu >> 1) & 1))) return;
                const float* other = sSum + slot * (M_WGS - 1) * MK + row;
                const float all = (mine + other[0]) + (other[MK] + other[2 * MK]);
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(MB_SUMFREE + slot));
                const long long key = (long long)wk.kt * MK + row;
                if (SPLIT && u == u0) {
                    sPart[row] = all;
                } else if (wk.any && key < tb.ext_len[wk.sq]) {
                    float* m = a.seqs[wk.sq].mass + (size_t)wk.g * a.seqs[wk.sq].ext_cap + key;
                    *m = a.accumulate ? *m + all : all;
                }
            }
        });
        if (!ok && lane == 0) record_err(a.err, abort_flag, kErrWaitAccFull);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == M_WARP) {
        tc_fence_after();
        tmem_dealloc(tmem, T_TMEM_COLS);
    }
}

// The shared-memory opt-in is per function and device: set on the first launch on each device (`done`: its bits).
template <typename F>
bool smem_opt_in(F* kernel, int bytes, unsigned long long* done) {
    int dev = 0;
    cudaGetDevice(&dev);
    const unsigned long long bit = 1ull << (dev & 63);
    if (__atomic_load_n(done, __ATOMIC_ACQUIRE) & bit) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
    __atomic_fetch_or(done, bit, __ATOMIC_RELEASE);
    return true;
}

// How many clusters of `ranks` CTAs (1, 2, 4 or 8) of a kernel the GPU holds at once: the GPCs' sizes decide (of 8 CTAs, one
// to an SM, fewer than 148 / 8). Found on the first call for a device and kept in `found`, the kernel's own.
template <typename F>
int clusters_at_once(F* kernel, int threads, int smem, int ranks, int (*found)[R_CLUSTER + 1]) {
    int dev = 0;
    cudaGetDevice(&dev);
    int& n = found[dev & 63][ranks];
    if (!n) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(ranks);
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = ranks;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        int v = 0;
        if (cudaOccupancyMaxActiveClusters(&v, kernel, &cfg) != cudaSuccess) {
            cudaGetLastError();
            return 0;
        }
        n = v;
    }
    return n;
}

// kernel<<<...>>>(args...) in clusters of `ranks` CTAs along x, with programmatic stream serialization.
template <typename... KP, typename... A>
int launch_clusters(void (*kernel)(KP...), dim3 grid, int block, size_t smem, int ranks, cudaStream_t st, const A&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ranks;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    cudaLaunchKernelEx(&cfg, kernel, args...);
    return (int)cudaGetLastError();
}

template <int NT, int W>
bool rows_opt_in() {
    static unsigned long long done = 0;
    return smem_opt_in(k_kv4_attn_rows<NT, W>, rows_smem<NT, W>(), &done);
}

template <int NT, int W>
int launch_rows_ranks(Kv4Args& a, long long x, int kv_heads, int z, int ranks, cudaStream_t st) {
    if (!rows_opt_in<NT, W>()) return -1;
    a.ranks = ranks;
    return launch_clusters(k_kv4_attn_rows<NT, W>, dim3((unsigned)x * ranks, kv_heads, z), W * 32, rows_smem<NT, W>(), ranks, st,
                           (const Kv4Args)a);
}

template <int NT, int W>
int rows_clusters_at_once() {
    static int found[64][R_CLUSTER + 1];
    if (!rows_opt_in<NT, W>()) return 0;
    return clusters_at_once(k_kv4_attn_rows<NT, W>, W * 32, rows_smem<NT, W>(), R_CLUSTER, found);
}

template <int NT>
int launch_rows(Kv4Args& a, int max_q, int max_keys, int kv_heads, cudaStream_t st) {
    long long x = ((long long)max_q * a.group + 8 * NT - 1) / (8 * NT);
    x = x < 1 ? 1 : x > 65536 ? 65536 : x;
    const int z = a.n_seqs < 65535 ? a.n_seqs : 65535;
    // CTAs to a cluster: as many as are resident at once, and no more than the keys give a tile to every warp (16
    // sequences of 8 rows, 4096 keys, 2 CTAs to an SM: 24 us with 2, 33 with 1, 31 with 4 and 46 with 8; one token over
    // 4097 keys, 4 warps to a CTA: 8.5 us with 8, 11, 17 and 27 with 4, 2 and 1)
    int ranks = R_CLUSTER;
    const int sms = sm_count();
    if (!sms) return -1;
    const long long tiles = ((long long)max_keys + R_KEYS - 1) / R_KEYS, slots = sms * (NT == 1 ? 4 : 2);
    const long long ctas = x * kv_heads * z;
    while (ranks > 1 && ((ranks / 2) * 4 >= tiles || ctas * ranks > slots)) ranks /= 2;
    // where they leave more than a quarter of the room empty and the keys are long, twice as many, the rest of them as room
    // comes free (10, 20 and 40 tokens over 8192 to 16384 keys: 32, 72 and 123 us, otherwise 40, 82 and 164; but of 16
    // tiles a CTA 10 x 16 rows over 4096 keys: 31 us, otherwise 28; and of a fuller GPU, 32 tokens over 16384: 103 and 97)
    if (ranks < R_CLUSTER && ctas * ranks * 4 < slots * 3 && tiles >= 2 * ranks * 24) ranks *= 2;
    // more warps to a CTA where there are tiles for them and the GPU holds all of these clusters at once (one token: over 4097
    // keys 6.8 us with 16 warps, 7.4 with 8, 8.3 with 4; over 60000 24, 31 and 48; two tokens, whose 16 clusters of 16 warps
    // do not fit: over 4500 keys 8.3 with 8, 12.3 with 16)
    if (ranks == R_CLUSTER) {
        constexpr int MOST = NT == 1 ? 16 : 8;
        if (NT == 1 && tiles > 8 * R_CLUSTER && ctas <= rows_clusters_at_once<NT, MOST>())
            return launch_rows_ranks<NT, MOST>(a, x, kv_heads, z, ranks, st);
        if (tiles > 4 * R_CLUSTER && ctas <= rows_clusters_at_once<NT, 8>())
            return launch_rows_ranks<NT, 8>(a, x, kv_heads, z, ranks, st);
    }
    return launch_rows_ranks<NT, 4>(a, x, kv_heads, z, ranks, st);
}

// Q as [row][head][64], in boxes of the group's heads of `most` / group rows: the packed rows of a tile in their order, in
// the 128-byte swizzle; rows behind the buffer read as zeros.
bool packed_tmap(CUtensorMap* m, const Kv4Args& a, int most) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return false;
    cuuint64_t dims[3] = {64, (cuuint64_t)a.heads, (cuuint64_t)a.q_rows};
    cuuint64_t strides[2] = {128, (cuuint64_t)a.ldq * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)a.group, (cuuint32_t)(most / a.group)};
    cuuint32_t estr[3] = {1, 1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(a.Q), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int launch_tc(Kv4Args& a, int max_q, int max_keys, cudaStream_t st) {
    static unsigned long long done = 0, done_split = 0;
    if (!smem_opt_in(k_kv4_attn_tc<false>, T_SMEM, &done) || !smem_opt_in(k_kv4_attn_tc<true>, T_SMEM, &done_split)) return -1;
    const int sms = sm_count();
    if (!sms) return -1;
    // no more CTAs than units, were every sequence max_q rows long
    const long long hu = (long long)max_q * a.group <= TQ ? a.heads / a.group : a.group % 2 == 0 ? a.heads / 2 : a.heads;
    const int per = a.group % 2 == 0 ? TQ : 2 * TQ;
    const long long units = a.n_seqs * hu * (max_q > per ? (max_q - 1) / per + 1 : 1);
    const int kv_cols = a.heads / a.group * 64;
    CUtensorMap tq, tqp, tk, tv;
    if (!attn_tmap(&tq, a.Q, a.heads * 64, a.q_rows, a.ldq, TQ)) return -1;
    if (a.group > TQ)
        tqp = tq;  // no packed units: never read
    else if (!packed_tmap(&tqp, a, TQ))
        return -1;
    if (a.kv_rows > 0) {
        if (!attn_tmap(&tk, a.K, kv_cols, a.kv_rows, a.ldkv, TKV) || !attn_tmap(&tv, a.V, kv_cols, a.kv_rows, a.ldkv, TKV))
            return -1;
    } else {
        tk = tv = tq;  // no own rows: never read
    }
    // few units: a cluster of CTAs to each, as many as the GPU has room for at once, with two key tiles or more for each
    // (8 heads, 128 packed rows over 4097 keys: 17 us, and 69 without; two such sequences: 21 us in clusters of 4, and 32 of 8)
    int ranks = R_CLUSTER;
    static int found[64][R_CLUSTER + 1];
    while (ranks > 1 && ((long long)(ranks - 1) * 2 * TKV >= max_keys ||
                         units > clusters_at_once(k_kv4_attn_tc<true>, T_THREADS, T_SMEM, ranks, found)))
        ranks /= 2;
    // the clusters' barriers and joins cost as much as five key tiles (100 packed rows: over 600 keys 11.8 us alone and 14.6
    // in twos, over 800 13.6 and in fours 13.0, over 1600 19.5, in twos 18.3 and in fours 15.0)
    const long long key_tiles = ((long long)max_keys + TKV - 1) / TKV;
    if (key_tiles * (ranks - 1) < 5 * ranks) ranks = 1;
    a.ranks = ranks;
    if (ranks == 1) {
        launch_pdl(k_kv4_attn_tc<false>, (int)(units < sms ? units : sms), T_THREADS, T_SMEM, st, tq, tqp, tk, tv, a);
        return (int)cudaGetLastError();
    }
    return launch_clusters(k_kv4_attn_tc<true>, dim3((unsigned)units * ranks), T_THREADS, T_SMEM, ranks, st, tq, tqp, tk, tv,
                           (const Kv4Args)a);
}

int launch_mass_tc(Kv4Args& a, int max_q, int max_len, cudaStream_t st) {
    static unsigned long long done = 0, done_split = 0;
    if (!smem_opt_in(k_kv4_mass_tc<false>, M_SMEM, &done) || !smem_opt_in(k_kv4_mass_tc<true>, M_SMEM, &done_split)) return -1;
    const int sms = sm_count();
    if (!sms) return -1;
    // no more CTAs than units, were every sequence's cache its own and max_len long
    const long long units = (long long)a.n_seqs * (max_len > 0 ? (max_len - 1) / MK + 1 : 1) * (a.heads / a.group);
    CUtensorMap tq;
    if (!packed_tmap(&tq, a, MQ)) return -1;
    // few units: a cluster of CTAs to each, as many as the GPU has room for at once, with a query tile for each (8 heads, one
    // sequence of 4000 rows, 500 keys: 18 us, and 42 without; 16 units in clusters of 8, which do not all fit: 17 us, of 4: 10)
    int ranks = R_CLUSTER;
    static int found[64][R_CLUSTER + 1];
    while (ranks > 1 && ((long long)max(2, ranks - 1) * (MQ / a.group) >= max_q ||  // (two tiles alone: 7.5 us, and 8.0)
                         units > clusters_at_once(k_kv4_mass_tc<true>, M_THREADS, M_SMEM, ranks, found)))
        ranks /= 2;
    a.ranks = ranks;
    if (ranks == 1) {
        launch_pdl(k_kv4_mass_tc<false>, (int)(units < sms ? units : sms), M_THREADS, M_SMEM, st, tq, a);
        return (int)cudaGetLastError();
    }
    return launch_clusters(k_kv4_mass_tc<true>, dim3((unsigned)units * ranks), M_THREADS, M_SMEM, ranks, st, tq, (const Kv4Args)a);
}

}  // namespace

extern "C" int d1_flash_attn_kv4(const d1_half* Q, int ldq, const d1_half* K, const d1_half* V, int ldkv, d1_half* O,
                                 int ldo, float* lse, int lse_ld, const D1Kv4Seq* seqs, int n_seqs, int max_q,
                                 int max_keys, int heads, int group, float scale, int q_rows, int kv_rows,
                                 cudaStream_t st) {
    if (n_seqs <= 0) return n_seqs == 0 ? 0 : -1;
    if (heads <= 0 || heads > kMaxHeads || group <= 0 || heads % group || heads / group > 4096 || q_rows < 0 ||
        kv_rows < 0 || !(scale > 0.f))
        return -1;
    if (max_q < 0 || max_keys < 0) return -1;
    if (q_rows == 0) return 0;
    if (!Q || !O || !seqs || (kv_rows > 0 && (!K || !V))) return -1;
    if (ldq < heads * 64 || ldo < heads * 64 || (kv_rows > 0 && ldkv < heads / group * 64)) return -1;
    if ((((uintptr_t)Q | (uintptr_t)K | (uintptr_t)V | (uintptr_t)O) & 15) || (ldq | ldkv | ldo) % 8) return -1;
    if (lse && lse_ld < q_rows) return -1;
    if (((uintptr_t)lse & 3) || ((uintptr_t)seqs & 7)) return -1;
    Kv4Args a = {};
    a.Q = Q;
    a.K = K;
    a.V = V;
    a.O = O;
    a.lse = lse;
    a.seqs = seqs;
    a.err = kv4_err_addr();
    a.ldq = ldq;
    a.ldkv = ldkv;
    a.ldo = ldo;
    a.lse_ld = lse_ld;
    a.n_seqs = n_seqs;
    a.heads = heads;
    a.group = group;
    a.q_rows = q_rows;
    a.kv_rows = kv_rows;
    a.scale_log2 = scale * kLog2e;
    if (!a.err) return -1;
    const int kv_heads = heads / group;
    // the tcgen05 form above 64 packed rows. 16 sequences over 1200 keys: 66 rows 20 us and 39 on mma.sync, 64 rows 20 and
    // 21, 32 rows 20 and 17; over 8000 keys: 77 and 198, 75 and 103, 75 and 55
    if ((long long)max_q * group > 64) return launch_tc(a, max_q, max_keys, st);
    const long long rows = (long long)max_q * group;
    return rows <= 8 ? launch_rows<1>(a, max_q, max_keys, kv_heads, st)
                     : rows <= 16 ? launch_rows<2>(a, max_q, max_keys, kv_heads, st)
                                  : launch_rows<4>(a, max_q, max_keys, kv_heads, st);
}

extern "C" int d1_kv4_mass(const d1_half* Q, int ldq, const float* lse, int lse_ld, const D1Kv4Seq* seqs, int n_seqs,
                           int max_q, int max_len, int heads, int group, float scale, int accumulate, int q_rows,
                           cudaStream_t st) {
    if (n_seqs <= 0) return n_seqs == 0 ? 0 : -1;
    if (heads <= 0 || heads > kMaxHeads || group <= 0 || heads % group || heads / group > 4096 || q_rows < 0 ||
        !(scale > 0.f))
        return -1;
    if (max_q < 0 || max_len < 0) return -1;
    if (!seqs || (q_rows > 0 && (!Q || !lse)) || ldq < heads * 64 || lse_ld < q_rows) return -1;
    if (((uintptr_t)Q & 15) || ldq % 8 || ((uintptr_t)lse & 3) || ((uintptr_t)seqs & 7)) return -1;
    Kv4Args a = {};
    a.Q = Q;
    a.lse = const_cast<float*>(lse);
    a.seqs = seqs;
    a.err = kv4_err_addr();
    a.ldq = ldq;
    a.lse_ld = lse_ld;
    a.n_seqs = n_seqs;
    a.heads = heads;
    a.group = group;
    a.q_rows = q_rows;
    a.accumulate = accumulate;
    a.scale_log2 = scale * kLog2e;
    if (!a.err) return -1;
    // the tcgen05 form above 64 packed rows a sequence, where its table holds the sequences. 16 sequences, 1200 keys: 66 rows
    // 20 us and 17 on mma.sync, 17 and 19 where they share 4 caches; 96 rows 19 and 19, 16 and 22; 192 rows 21 and 32, 21
    // and 38
    if ((long long)max_q * group > 64 && group <= MQ && q_rows > 0 && n_seqs <= M_SEQS) return launch_mass_tc(a, max_q, max_len, st);
    const int z = n_seqs < 65535 ? n_seqs : 65535, kv_heads = heads / group, sms = sm_count();
    if (!sms) return -1;
    auto blocks = [&](int keys) {
        const long long x = ((long long)max_len + keys - 1) / keys;
        return (unsigned)(x < 1 ? 1 : x > 65536 ? 65536 : x);
    };
    // 32 keys to a warp up to about two waves of CTAs, then 64, whose expansion the rows share out better (8 rows, one cache
    // of 8000 keys: 4.3 us and 5.0 with 64; 16 caches of 1200: 9.7 and 10.2; 16 of 8000: 43 and 33; 24 rows, 16 sequences
    // on 4 caches of 1200: 14 and 22)
    if ((long long)blocks(256) * kv_heads * z <= 5 * sms)
        launch_pdl(k_kv4_mass_rows<2>, dim3(blocks(256), kv_heads, z), 256, 0, st, a);
    else
        launch_pdl(k_kv4_mass_rows<4>, dim3(blocks(512), kv_heads, z), 256, 0, st, a);
    return (int)cudaGetLastError();
}
