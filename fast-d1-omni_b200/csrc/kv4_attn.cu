// Attention over key/value caches held in 4 bits (format: include/d1kernels.h, D1Kv4Seq), and the attention weight that
// every cached key received. Head dim 64, packed variable-length sequences, bidirectional.
#include "kv4.cuh"
#include "warp_mma.cuh"

using namespace d1;

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Kv4Args {
    const __half* Q;
    const __half* K;
    const __half* V;
    __half* O;
    float* lse;
    const D1Kv4Seq* seqs;
    int* err;
    int ldq, ldkv, ldo, lse_ld, n_seqs, group, q_rows, kv_rows, accumulate;
    float scale_log2;
};

__device__ __forceinline__ float ex2f(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ------------------------------------------------------------------------------------------------ attention, few rows
// The query rows of a kv head's group are packed: packed row p is row p / group of the sequence, head p % group of the
// group. A CTA takes 16 * MT packed rows of one (sequence, kv head); its warps take tiles of 64 keys in turn, each with
// its own running maximum, sum and output, which they join at the end through shared memory.
//
// The codes go from global memory to the registers of the MMAs (m16n8k16) directly. An MMA's k index may run over the
// dimensions in any order as long as both operands use the same: for S = Q K^T lane (r, t) = (lane / 4, lane % 4) holds
// dimensions 16t .. 16t+15 of key r of each 8 keys: 8 bytes of codes, and 32 bytes of a query row. The MMA sees the whole
// numbers code - zero; a key's step multiplies its column of S afterwards, in fp32, with the softmax scale. For O = P V
// lane (r, t) holds word r (dimensions 8r .. 8r+7) of keys 2t, 2t+1, 2t+8, 2t+9 of each 16 keys; byte permutes bring two
// keys' codes of one dimension together, and the values are (code - zero) * step, exact in fp16. n index r of the j-th MMA
// is dimension 8r + j, so that a lane ends with dimensions 16t .. 16t+15 of its rows.
constexpr int R_KEYS = 64, R_WARPS = 8, R_OLD = 68;  // padded row of the joining buffer (floats)

template <int MT>
constexpr int rows_smem() {
    return R_WARPS * 16 * MT * (R_OLD + 2) * 4;
}

template <int MT>
__global__ void __launch_bounds__(R_WARPS * 32) k_kv4_attn_rows(const Kv4Args a) {
    extern __shared__ __align__(16) float r_smem[];
    constexpr int NR = 16 * MT;
    float* sO = r_smem;                           // [warp][NR][R_OLD]
    float* sM = sO + R_WARPS * NR * R_OLD;        // [warp][NR]
    float* sL = sM + R_WARPS * NR;                // [warp][NR]
    pdl_entry();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = lane >> 2, t = lane & 3, g = blockIdx.y;
    for (int sq = blockIdx.z; sq < a.n_seqs; sq += gridDim.z) {
        const D1Kv4Seq s = a.seqs[sq];
        if (!kv4_seq_ok(s) || !rows_ok(s.q_start, s.q_len, a.q_rows) || !rows_ok(s.kv_start, s.kv_len, a.kv_rows)) {
            if (tid == 0) atomicExch(a.err, kErrTable);
            continue;
        }
        const long long n_rows = (long long)s.q_len * a.group;
        const int ext_tiles = (s.ext_len + R_KEYS - 1) / R_KEYS, tiles = ext_tiles + (s.kv_len + R_KEYS - 1) / R_KEYS;
        const uint8_t* k4 = s.k4 + (size_t)g * s.ext_cap * 32;
        const uint8_t* v4 = s.v4 + (size_t)g * s.ext_cap * 32;
        const uint16_t* kp = reinterpret_cast<const uint16_t*>(s.kp) + (size_t)g * s.ext_cap;
        const uint16_t* vp = reinterpret_cast<const uint16_t*>(s.vp) + (size_t)g * s.ext_cap;
        for (long long base = (long long)blockIdx.x * NR; base < n_rows; base += (long long)gridDim.x * NR) {
            // ---- the query rows, as A operands
            uint32_t qa[MT][4][4];
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const long long p = base + mt * 16 + hf * 8 + r;
                    uint4 x0 = make_uint4(0, 0, 0, 0), x1 = x0;
                    if (p < n_rows) {
                        const int row = (int)(p / a.group), h = g * a.group + (int)(p % a.group);
                        const uint4* src =
                            reinterpret_cast<const uint4*>(a.Q + (size_t)(s.q_start + row) * a.ldq + h * 64 + 16 * t);
                        x0 = __ldg(src);
                        x1 = __ldg(src + 1);
                    }
                    const uint32_t w[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
#pragma unroll
                    for (int ks = 0; ks < 4; ks++) {
                        qa[mt][ks][hf] = w[2 * ks];
                        qa[mt][ks][2 + hf] = w[2 * ks + 1];
                    }
                }
            }
            float o[MT][8][4], m[MT][2], l[MT][2];
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int c = 0; c < 4; c++) o[mt][j][c] = 0.f;
                m[mt][0] = m[mt][1] = -INFINITY;
                l[mt][0] = l[mt][1] = 0.f;
            }
            for (int tile = warp; tile < tiles; tile += R_WARPS) {
                const bool ext = tile < ext_tiles;
                const int key0 = (ext ? tile : tile - ext_tiles) * R_KEYS;
                const int left = (ext ? s.ext_len : s.kv_len) - key0;  // keys of this tile: min(left, 64), at least 1
                const int last = min(left, R_KEYS) - 1;
                float sc[MT][8][4];
                uint32_t vw[4][4];   // cached: the words of V
                uint32_t pv = 0;     // cached: V parameters of keys 2 lane, 2 lane + 1
                if (ext) {
                    uint2 kw[8];
#pragma unroll
                    for (int n = 0; n < 8; n++)
                        kw[n] = __ldg(reinterpret_cast<const uint2*>(k4 + (size_t)(key0 + min(8 * n + r, last)) * 32) + t);
#pragma unroll
                    for (int ks = 0; ks < 4; ks++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            vw[ks][i] = __ldg(reinterpret_cast<const uint32_t*>(
                                                  v4 + (size_t)(key0 + min(16 * ks + 2 * t + (i & 1) + (i >> 1) * 8, last)) * 32) +
                                              r);
                    // whole pairs are inside the cache's arrays: ext_cap is a multiple of 8
                    const int pk = key0 + (min(2 * lane, last) & ~1);
                    const uint32_t pkw = __ldg(reinterpret_cast<const uint32_t*>(kp + pk));
                    pv = __ldg(reinterpret_cast<const uint32_t*>(vp + pk));
                    // rows behind the cached ones hold anything: step 0 there, so that 0 * V is 0
                    if (2 * lane + 1 > last) pv = 2 * lane > last ? 0 : pv & 0xffffu;
#pragma unroll
                    for (int n = 0; n < 8; n++) {
                        const uint32_t both = __shfl_sync(D1_FULL_MASK, pkw, 4 * n + (r >> 1));
                        const uint32_t par = __byte_perm(both, 0, r & 1 ? 0x3232 : 0x1010);
                        uint32_t z0, z1, b0[4], b1[4];
                        kv4_zero(par, z0, z1);
                        kv4_expand(kw[n].x, z0, z1, b0);
                        kv4_expand(kw[n].y, z0, z1, b1);
                        const uint32_t pc = __shfl_sync(D1_FULL_MASK, pkw, 4 * n + t);
                        const float st0 = kv4_step(pc & 0xffffu) * a.scale_log2, st1 = kv4_step(pc >> 16) * a.scale_log2;
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) {
                            float c[4] = {0.f, 0.f, 0.f, 0.f};
                            mma16816(c, qa[mt][0], b0[0], b0[1]);
                            mma16816(c, qa[mt][1], b0[2], b0[3]);
                            mma16816(c, qa[mt][2], b1[0], b1[1]);
                            mma16816(c, qa[mt][3], b1[2], b1[3]);
                            sc[mt][n][0] = c[0] * st0;
                            sc[mt][n][1] = c[1] * st1;
                            sc[mt][n][2] = c[2] * st0;
                            sc[mt][n][3] = c[3] * st1;
                        }
                    }
                } else {
                    const __half* kr = a.K + (size_t)(s.kv_start + key0) * a.ldkv + g * 64 + 16 * t;
#pragma unroll
                    for (int n = 0; n < 8; n++) {
                        const uint4* src = reinterpret_cast<const uint4*>(kr + (size_t)min(8 * n + r, last) * a.ldkv);
                        const uint4 x0 = __ldg(src), x1 = __ldg(src + 1);
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) {
                            float c[4] = {0.f, 0.f, 0.f, 0.f};
                            mma16816(c, qa[mt][0], x0.x, x0.y);
                            mma16816(c, qa[mt][1], x0.z, x0.w);
                            mma16816(c, qa[mt][2], x1.x, x1.y);
                            mma16816(c, qa[mt][3], x1.z, x1.w);
#pragma unroll
                            for (int i = 0; i < 4; i++) sc[mt][n][i] = c[i] * a.scale_log2;
                        }
                    }
                }
                if (left < R_KEYS) {
#pragma unroll
                    for (int mt = 0; mt < MT; mt++)
#pragma unroll
                        for (int n = 0; n < 8; n++)
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                if (8 * n + 2 * t + (i & 1) >= left) sc[mt][n][i] = -INFINITY;
                }
                // ---- running softmax, in the exp2 domain
                uint32_t pa[MT][8][2];
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                    for (int hf = 0; hf < 2; hf++) {
                        float mx = -INFINITY;
#pragma unroll
                        for (int n = 0; n < 8; n++) mx = fmaxf(mx, fmaxf(sc[mt][n][2 * hf], sc[mt][n][2 * hf + 1]));
                        mx = fmaxf(mx, __shfl_xor_sync(D1_FULL_MASK, mx, 1));
                        mx = fmaxf(mx, __shfl_xor_sync(D1_FULL_MASK, mx, 2));
                        const float mn = fmaxf(m[mt][hf], mx);
                        const float alpha = m[mt][hf] == mn ? 1.f : ex2f(m[mt][hf] - mn);
                        m[mt][hf] = mn;
                        float sum = 0.f;
#pragma unroll
                        for (int n = 0; n < 8; n++) {
                            const float p0 = ex2f(sc[mt][n][2 * hf] - mn), p1 = ex2f(sc[mt][n][2 * hf + 1] - mn);
                            sum += p0 + p1;
                            pa[mt][n][hf] = pack_h2(p0, p1);
                        }
                        l[mt][hf] = l[mt][hf] * alpha + sum;
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            o[mt][j][2 * hf] *= alpha;
                            o[mt][j][2 * hf + 1] *= alpha;
                        }
                    }
                // ---- O += P V
#pragma unroll
                for (int ks = 0; ks < 4; ks++) {
                    uint32_t b[2][8];  // [keys 2t, 2t+1 | 2t+8, 2t+9][j]
                    if (ext) {
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const uint32_t par = __shfl_sync(D1_FULL_MASK, pv, 8 * ks + 4 * i + t);
                            const uint32_t st = kv4_step2(par);
                            uint32_t z0, z1, ev[4], od[4];
                            kv4_zero(par, z0, z1);
                            kv4_expand(__byte_perm(vw[ks][2 * i], vw[ks][2 * i + 1], 0x5410), z0, z1, ev);
                            kv4_expand(__byte_perm(vw[ks][2 * i], vw[ks][2 * i + 1], 0x7632), z0, z1, od);
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                b[i][2 * j] = h2_mul(ev[j], st);
                                b[i][2 * j + 1] = h2_mul(od[j], st);
                            }
                        }
                    } else {
                        const __half* vr = a.V + (size_t)(s.kv_start + key0) * a.ldkv + g * 64 + 8 * r;
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const int k = 16 * ks + 8 * i + 2 * t;
                            const uint4 x = __ldg(reinterpret_cast<const uint4*>(vr + (size_t)min(k, last) * a.ldkv));
                            const uint4 y = __ldg(reinterpret_cast<const uint4*>(vr + (size_t)min(k + 1, last) * a.ldkv));
                            const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                b[i][2 * j] = __byte_perm(xs[j], ys[j], 0x5410);
                                b[i][2 * j + 1] = __byte_perm(xs[j], ys[j], 0x7632);
                            }
                        }
                    }
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        const uint32_t pr[4] = {pa[mt][2 * ks][0], pa[mt][2 * ks][1], pa[mt][2 * ks + 1][0],
                                                pa[mt][2 * ks + 1][1]};
#pragma unroll
                        for (int j = 0; j < 8; j++) mma16816(o[mt][j], pr, b[0][j], b[1][j]);
                    }
                }
            }
            // ---- join the warps: weights 2^(m - M), in the warps' order
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    float sum = l[mt][hf];
                    sum += __shfl_xor_sync(D1_FULL_MASK, sum, 1);
                    sum += __shfl_xor_sync(D1_FULL_MASK, sum, 2);
                    const int row = mt * 16 + hf * 8 + r;
                    if (t == 0) {
                        sM[warp * NR + row] = m[mt][hf];
                        sL[warp * NR + row] = sum;
                    }
                    float4* dst = reinterpret_cast<float4*>(sO + (warp * NR + row) * R_OLD + 16 * t);
#pragma unroll
                    for (int q = 0; q < 4; q++)  // dimensions 16t + 4q .. : j = 4 (q & 1) .., column 2t + q / 2
                        dst[q] = make_float4(o[mt][4 * (q & 1)][2 * hf + (q >> 1)], o[mt][4 * (q & 1) + 1][2 * hf + (q >> 1)],
                                             o[mt][4 * (q & 1) + 2][2 * hf + (q >> 1)],
                                             o[mt][4 * (q & 1) + 3][2 * hf + (q >> 1)]);
                }
            __syncthreads();
            for (int i = tid; i < NR * 16; i += R_WARPS * 32) {
                const int row = i >> 4, d = (i & 15) * 4;
                const long long p = base + row;
                if (p >= n_rows) continue;
                float M = -INFINITY;
#pragma unroll
                for (int w = 0; w < R_WARPS; w++) M = fmaxf(M, sM[w * NR + row]);
                float L = 0.f, x0 = 0.f, x1 = 0.f, x2 = 0.f, x3 = 0.f;
                for (int w = 0; w < R_WARPS && w < tiles; w++) {  // warps beyond the tiles hold nothing
                    const float f = ex2f(sM[w * NR + row] - M);
                    const float4 v = *reinterpret_cast<const float4*>(sO + (w * NR + row) * R_OLD + d);
                    L += f * sL[w * NR + row];
                    x0 += f * v.x;
                    x1 += f * v.y;
                    x2 += f * v.z;
                    x3 += f * v.w;
                }
                const float il = tiles ? 1.f / L : 0.f;
                const int q = s.q_start + (int)(p / a.group), h = g * a.group + (int)(p % a.group);
                *reinterpret_cast<uint2*>(a.O + (size_t)q * a.ldo + h * 64 + d) =
                    make_uint2(pack_h2(x0 * il, x1 * il), pack_h2(x2 * il, x3 * il));
                if (a.lse && d == 0) a.lse[(size_t)h * a.lse_ld + q] = tiles ? (M + log2f(L)) * kLn2 : -INFINITY;
            }
            __syncthreads();
        }
    }
}

// ------------------------------------------------------------------------------------------------ mass, few rows
// S^T = K Q^T on m16n8k16: a warp holds 64 keys as A operands (whole numbers code - zero, as above) and goes over the
// packed query rows 8 at a time, adding exp(s - lse) into 8 sums of its keys; four lanes share a key at the end. The
// sequences that share a mass array are taken by the first of them, in the table's order.
constexpr int M_KEYS = 64 * 8;  // keys of a CTA of 8 warps

__global__ void __launch_bounds__(256) k_kv4_mass_rows(const Kv4Args a) {
    __shared__ int peers[256];
    __shared__ int n_peers;
    pdl_entry();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = lane >> 2, t = lane & 3, g = blockIdx.y;
    for (int sq = blockIdx.z; sq < a.n_seqs; sq += gridDim.z) {
        const D1Kv4Seq s = a.seqs[sq];
        if (!s.mass) continue;
        if (!kv4_seq_ok(s)) {
            if (tid == 0) atomicExch(a.err, kErrTable);
            continue;
        }
        int before = 0;
        for (int i = tid; i < sq; i += 256) before |= a.seqs[i].mass == s.mass;
        if (__syncthreads_or(before)) continue;
        const uint16_t* kp = reinterpret_cast<const uint16_t*>(s.kp) + (size_t)g * s.ext_cap;
        const uint8_t* k4 = s.k4 + (size_t)g * s.ext_cap * 32;
        for (int k0 = blockIdx.x * M_KEYS; k0 < s.ext_len; k0 += gridDim.x * M_KEYS) {
            const int key0 = k0 + warp * 64;
            uint32_t ka[4][4][4];
            float st[4][2], sum[4][2];
#pragma unroll
            for (int mt = 0; mt < 4; mt++)
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const int key = min(key0 + mt * 16 + hf * 8 + r, s.ext_len - 1);
                    const uint2 w = __ldg(reinterpret_cast<const uint2*>(k4 + (size_t)key * 32) + t);
                    const uint32_t par = __ldg(kp + key);
                    uint32_t z0, z1, x[4], y[4];
                    kv4_zero(par * 0x00010001u, z0, z1);
                    kv4_expand(w.x, z0, z1, x);
                    kv4_expand(w.y, z0, z1, y);
                    ka[mt][0][hf] = x[0];
                    ka[mt][0][2 + hf] = x[1];
                    ka[mt][1][hf] = x[2];
                    ka[mt][1][2 + hf] = x[3];
                    ka[mt][2][hf] = y[0];
                    ka[mt][2][2 + hf] = y[1];
                    ka[mt][3][hf] = y[2];
                    ka[mt][3][2 + hf] = y[3];
                    st[mt][hf] = kv4_step(par) * a.scale_log2;
                    sum[mt][hf] = 0.f;
                }
            bool any = false;
            for (int b0 = sq; b0 < a.n_seqs; b0 += 256) {  // the sequences of this mass array, in order
                __syncthreads();
                if (warp == 0) {
                    int n = 0;
                    for (int i = 0; i < 256; i += 32) {
                        const int j = b0 + i + lane;
                        const bool same = j < a.n_seqs && a.seqs[j].mass == s.mass;
                        const uint32_t v = __ballot_sync(D1_FULL_MASK, same);
                        if (same) peers[n + __popc(v & ((1u << lane) - 1))] = j;
                        n += __popc(v);
                    }
                    if (lane == 0) n_peers = n;
                }
                __syncthreads();
                for (int e = 0; e < n_peers; e++) {
                    const D1Kv4Seq& p = a.seqs[peers[e]];
                    const int q_start = p.q_start, q_len = p.q_len;
                    if (p.k4 != s.k4 || p.ext_len != s.ext_len || p.ext_cap != s.ext_cap ||
                        !rows_ok(q_start, q_len, a.q_rows)) {
                        if (tid == 0) atomicExch(a.err, kErrTable);
                        continue;
                    }
                    any = true;
                    const long long n_rows = (long long)q_len * a.group;
                    for (long long base = 0; base < n_rows; base += 8) {
                        uint4 x0 = make_uint4(0, 0, 0, 0), x1 = x0;
                        float lse = INFINITY;  // of packed row base + r, in log2; +inf: adds nothing
                        if (base + r < n_rows) {
                            const int q = q_start + (int)((base + r) / a.group), h = g * a.group + (int)((base + r) % a.group);
                            const uint4* src = reinterpret_cast<const uint4*>(a.Q + (size_t)q * a.ldq + h * 64 + 16 * t);
                            x0 = __ldg(src);
                            x1 = __ldg(src + 1);
                            const float v = __ldg(a.lse + (size_t)h * a.lse_ld + q) * kLog2e;
                            lse = v == -INFINITY ? INFINITY : v;
                        }
                        const float l0 = __shfl_sync(D1_FULL_MASK, lse, 8 * t), l1 = __shfl_sync(D1_FULL_MASK, lse, 8 * t + 4);
#pragma unroll
                        for (int mt = 0; mt < 4; mt++) {
                            float c[4] = {0.f, 0.f, 0.f, 0.f};
                            mma16816(c, ka[mt][0], x0.x, x0.y);
                            mma16816(c, ka[mt][1], x0.z, x0.w);
                            mma16816(c, ka[mt][2], x1.x, x1.y);
                            mma16816(c, ka[mt][3], x1.z, x1.w);
                            sum[mt][0] += ex2f(c[0] * st[mt][0] - l0) + ex2f(c[1] * st[mt][0] - l1);
                            sum[mt][1] += ex2f(c[2] * st[mt][1] - l0) + ex2f(c[3] * st[mt][1] - l1);
                        }
                    }
                }
            }
            float* mass = s.mass + (size_t)g * s.ext_cap;
#pragma unroll
            for (int mt = 0; mt < 4; mt++)
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    float v = sum[mt][hf];
                    v += __shfl_xor_sync(D1_FULL_MASK, v, 1);
                    v += __shfl_xor_sync(D1_FULL_MASK, v, 2);
                    const int key = key0 + mt * 16 + hf * 8 + r;
                    if (any && t == 0 && key < s.ext_len) mass[key] = a.accumulate ? mass[key] + v : v;
                }
        }
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

template <int MT>
int launch_rows(const Kv4Args& a, int max_q, int kv_heads, cudaStream_t st) {
    static unsigned long long done = 0;
    if (!smem_opt_in(k_kv4_attn_rows<MT>, rows_smem<MT>(), &done)) return -1;
    long long x = ((long long)max_q * a.group + 16 * MT - 1) / (16 * MT);
    x = x < 1 ? 1 : x > 65536 ? 65536 : x;
    const int z = a.n_seqs < 65535 ? a.n_seqs : 65535;
    launch_pdl(k_kv4_attn_rows<MT>, dim3((unsigned)x, kv_heads, z), R_WARPS * 32, rows_smem<MT>(), st, a);
    return (int)cudaGetLastError();
}

}  // namespace

extern "C" int d1_flash_attn_kv4(const d1_half* Q, int ldq, const d1_half* K, const d1_half* V, int ldkv, d1_half* O,
                                 int ldo, float* lse, int lse_ld, const D1Kv4Seq* seqs, int n_seqs, int max_q,
                                 int max_keys, int heads, int group, float scale, int q_rows, int kv_rows,
                                 cudaStream_t st) {
    if (n_seqs <= 0) return n_seqs == 0 ? 0 : -1;
    if (heads <= 0 || group <= 0 || heads % group || heads / group > 4096 || q_rows < 0 || kv_rows < 0 || !(scale > 0.f))
        return -1;
    if (max_q < 0 || max_keys < 0) return -1;
    if (q_rows == 0) return 0;
    if (!Q || !O || !seqs || (kv_rows > 0 && (!K || !V))) return -1;
    if (ldq < heads * 64 || ldo < heads * 64 || (kv_rows > 0 && ldkv < heads / group * 64)) return -1;
    if ((((uintptr_t)Q | (uintptr_t)K | (uintptr_t)V | (uintptr_t)O) & 15) || (ldq | ldkv | ldo) % 8) return -1;
    if (lse && lse_ld < q_rows) return -1;
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
    a.group = group;
    a.q_rows = q_rows;
    a.kv_rows = kv_rows;
    a.scale_log2 = scale * kLog2e;
    if (!a.err) return -1;
    const int kv_heads = heads / group;
    return (long long)max_q * group <= 16 ? launch_rows<1>(a, max_q, kv_heads, st) : launch_rows<2>(a, max_q, kv_heads, st);
}

extern "C" int d1_kv4_mass(const d1_half* Q, int ldq, const float* lse, int lse_ld, const D1Kv4Seq* seqs, int n_seqs,
                           int max_q, int max_len, int heads, int group, float scale, int accumulate, int q_rows,
                           cudaStream_t st) {
    if (n_seqs <= 0) return n_seqs == 0 ? 0 : -1;
    if (heads <= 0 || group <= 0 || heads % group || heads / group > 4096 || q_rows < 0 || !(scale > 0.f)) return -1;
    if (max_q < 0 || max_len < 0) return -1;
    if (!seqs || (q_rows > 0 && (!Q || !lse)) || ldq < heads * 64 || lse_ld < q_rows) return -1;
    if (((uintptr_t)Q & 15) || ldq % 8) return -1;
    Kv4Args a = {};
    a.Q = Q;
    a.lse = const_cast<float*>(lse);
    a.seqs = seqs;
    a.err = kv4_err_addr();
    a.ldq = ldq;
    a.lse_ld = lse_ld;
    a.n_seqs = n_seqs;
    a.group = group;
    a.q_rows = q_rows;
    a.accumulate = accumulate;
    a.scale_log2 = scale * kLog2e;
    if (!a.err) return -1;
    int x = (max_len + M_KEYS - 1) / M_KEYS;
    x = x < 1 ? 1 : x > 65536 ? 65536 : x;
    launch_pdl(k_kv4_mass_rows, dim3(x, heads / group, n_seqs < 65535 ? n_seqs : 65535), 256, 0, st, a);
    return (int)cudaGetLastError();
}
