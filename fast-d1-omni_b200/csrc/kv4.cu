// Key/value caches held in 4 bits (format: include/d1kernels.h, D1Kv4Seq): rows into a cache and back, and eviction by
// accumulated attention weight. The attention over such caches is in kv4_attn.cu.
#include "kv4.cuh"

using namespace d1;

namespace d1 {
__device__ int g_kv4_err = 0;  // read and cleared by d1_kv4_error()

int* kv4_err_addr() {
    void* a = nullptr;
    return cudaGetSymbolAddress(&a, g_kv4_err) == cudaSuccess ? static_cast<int*>(a) : nullptr;
}
}  // namespace d1

namespace {

constexpr int kMaxGridZ = 65535;

__device__ __forceinline__ void table_error() { atomicExch(&g_kv4_err, kErrTable); }

// ------------------------------------------------------------------------------------------------ append, load
// 8 lanes per vector of 64 dimensions (8 elements, one word of codes a lane), 4 consecutive rows of one kv head per
// warp, so that a warp's codes are one 128-byte run of the cache. CTA: 32 rows of (K or V, kv head).
constexpr int A_ROWS = 32;

__global__ void __launch_bounds__(256) k_kv4_append(const __half* __restrict__ K, const __half* __restrict__ V,
                                                    int ldkv, const D1Kv4Seq* __restrict__ seqs, int n_seqs) {
    pdl_entry();
    const int lane = threadIdx.x & 31, sub = lane & 7;
    const int g = blockIdx.y >> 1;
    const bool is_v = blockIdx.y & 1;
    for (int sq = blockIdx.z; sq < n_seqs; sq += gridDim.z) {
        const D1Kv4Seq s = seqs[sq];
        if (s.kv_start < 0 || s.kv_len < 0 || !kv4_seq_ok(s) || (long long)s.ext_len + s.kv_len > s.ext_cap) {
            if (threadIdx.x == 0) table_error();
            continue;
        }
        const __half* src = (is_v ? V : K) + (size_t)s.kv_start * ldkv + g * 64 + sub * 8;
        const size_t at = (size_t)g * s.ext_cap + s.ext_len;
        uint32_t* codes = reinterpret_cast<uint32_t*>(is_v ? s.v4 : s.k4) + at * 8 + sub;
        uint16_t* pars = reinterpret_cast<uint16_t*>(is_v ? s.vp : s.kp) + at;
        for (int r0 = blockIdx.x * A_ROWS; r0 < s.kv_len; r0 += gridDim.x * A_ROWS) {
            const int r = r0 + (threadIdx.x >> 3);
            const bool there = r < s.kv_len;
            const uint4 raw = there ? __ldg(reinterpret_cast<const uint4*>(src + (size_t)r * ldkv)) : make_uint4(0, 0, 0, 0);
            const __half2* x2 = reinterpret_cast<const __half2*>(&raw);
            // the range, with zero in it; x * 0 is NaN for a NaN or an infinity
            __half2 mn = __float2half2_rn(0.f), mx = mn, bad = mn;
            float x[8];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                mn = __hmin2(mn, x2[i]);
                mx = __hmax2(mx, x2[i]);
                bad = __hfma2(x2[i], __float2half2_rn(0.f), bad);
                const float2 f = __half22float2(x2[i]);
                x[2 * i] = f.x;
                x[2 * i + 1] = f.y;
            }
            float lo = __half2float(__hmin(__low2half(mn), __high2half(mn)));
            float hi = __half2float(__hmax(__low2half(mx), __high2half(mx)));
            bool nan = __hisnan(__low2half(bad)) || __hisnan(__high2half(bad));
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) {
                lo = fminf(lo, __shfl_xor_sync(D1_FULL_MASK, lo, o));
                hi = fmaxf(hi, __shfl_xor_sync(D1_FULL_MASK, hi, o));
                nan |= __shfl_xor_sync(D1_FULL_MASK, (int)nan, o) != 0;
            }
            // 7 significant bits upwards: carry into the mantissa's upper 6 bits; below 2^-14 a multiple of 2^-20
            const float want = __fdiv_rn(hi - lo, 15.f);
            const float step = want >= 6.103515625e-5f
                                   ? __uint_as_float((__float_as_uint(want) + 0x1ffffu) & ~0x1ffffu)
                                   : ceilf(want * 1048576.f) * 9.5367431640625e-7f;
            const float div = step > 0.f ? step : 1.f;
            const float zero = fminf(rintf(__fdiv_rn(-lo, div)), 15.f), top = floorf(__fdiv_rn(65504.f, div));
            uint32_t word = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float q = fmaxf(fminf(rintf(__fdiv_rn(x[i], div)), top), -top) + zero;
                const uint32_t c = (uint32_t)fmaxf(fminf(q, 15.f), 0.f);
                word |= c << ((i & 1) * 16 + (i >> 1) * 4);
            }
            uint32_t par = (uint32_t)__half_as_ushort(__float2half_rn(step)) | (uint32_t)zero;
            if (nan) {
                word = 0;
                par = 0x7e00u;  // a NaN step
            }
            if (there) {
                codes[(size_t)r * 8] = word;
                if (sub == 0) pars[r] = (uint16_t)par;
            }
        }
    }
}

__global__ void __launch_bounds__(256) k_kv4_load(const D1Kv4Seq* __restrict__ seqs, int n_seqs, __half* __restrict__ K,
                                                  __half* __restrict__ V, int ldkv) {
    pdl_entry();
    const int lane = threadIdx.x & 31, sub = lane & 7;
    const int g = blockIdx.y >> 1;
    const bool is_v = blockIdx.y & 1;
    for (int sq = blockIdx.z; sq < n_seqs; sq += gridDim.z) {
        const D1Kv4Seq s = seqs[sq];
        if (s.kv_start < 0 || s.kv_len < 0 || !kv4_seq_ok(s) || (long long)s.ext_len + s.kv_len > s.ext_cap) {
            if (threadIdx.x == 0) table_error();
            continue;
        }
        __half* dst = (is_v ? V : K) + (size_t)s.kv_start * ldkv + g * 64 + sub * 8;
        const size_t at = (size_t)g * s.ext_cap + s.ext_len;
        const uint32_t* codes = reinterpret_cast<const uint32_t*>(is_v ? s.v4 : s.k4) + at * 8 + sub;
        const uint16_t* pars = reinterpret_cast<const uint16_t*>(is_v ? s.vp : s.kp) + at;
        for (int r = blockIdx.x * A_ROWS + (threadIdx.x >> 3); r < s.kv_len; r += gridDim.x * A_ROWS) {
            const uint32_t word = codes[(size_t)r * 8], par = (uint32_t)pars[r] * 0x00010001u;
            uint32_t z0, z1, v[4];
            kv4_zero(par, z0, z1);
            kv4_expand(word, z0, z1, v);
            const uint32_t st = kv4_step2(par);
            *reinterpret_cast<uint4*>(dst + (size_t)r * ldkv) =
                make_uint4(h2_mul(v[0], st), h2_mul(v[1], st), h2_mul(v[2], st), h2_mul(v[3], st));
        }
    }
}

// ------------------------------------------------------------------------------------------------ evict
// One CTA per (part of the destination, kv head, item). Every part finds the head's threshold for itself (the masses
// are small beside the rows that move), so that the parts need not wait for each other; then each copies its slice of
// the destination's rows.
constexpr int E_THREADS = 1024, E_LIST = 4096;

// A mass as an unsigned number of the same order: NaN as -inf, -0 as +0.
__device__ __forceinline__ uint32_t mass_key(float m) {
    const uint32_t b = m != m ? 0xff800000u : __float_as_uint(m + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Sum over the CTA of v, in all threads. buf: 2 x 32 words, used in turn, so that one barrier a call is enough.
__device__ __forceinline__ uint32_t cta_sum(uint32_t v, uint32_t* buf, int turn) {
    uint32_t* b = buf + (turn & 1) * 32;
    v = __reduce_add_sync(D1_FULL_MASK, v);
    if ((threadIdx.x & 31) == 0) b[threadIdx.x >> 5] = v;
    __syncthreads();
    return __reduce_add_sync(D1_FULL_MASK, b[threadIdx.x & 31]);
}

__global__ void __launch_bounds__(E_THREADS) k_kv4_evict(const D1Kv4Evict* __restrict__ items, int n_items) {
    __shared__ uint32_t buf[64];
    __shared__ uint32_t wsum[32][2];
    __shared__ int list[E_LIST];
    pdl_entry();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = blockIdx.y;
    for (int item = blockIdx.z; item < n_items; item += gridDim.z) {
        const D1Kv4Evict it = items[item];
        const int keep = min(it.keep, it.len), recent = min(it.recent, keep);
        if (it.keep < 0 || it.recent < 0 || !kv4_cache_ok(it.len, it.cap, it.k4, it.v4, it.kp, it.vp) ||
            (it.len > 0 && !it.mass) ||
            !kv4_cache_ok(keep, it.dst_cap, it.dst_k4, it.dst_v4, it.dst_kp, it.dst_vp)) {
            if (tid == 0) table_error();
            continue;
        }
        const int per = (keep + gridDim.x - 1) / gridDim.x;
        const int p0 = min(keep, (int)blockIdx.x * per), p1 = min(keep, p0 + per);
        if (p0 >= p1) continue;
        const int nc = it.len - recent, want = keep - recent;  // keys to choose from, and how many
        const float* m = it.mass + (size_t)g * it.cap;
        // the want-th largest key: the largest t with at least `want` keys >= t, a bit at a time
        uint32_t t = 0;
        int turn = 0;
        if (want > 0) {
#pragma unroll 1
            for (int b = 31; b >= 0; b--) {
                const uint32_t c = t | (1u << b);
                uint32_t n = 0;
                for (int i = tid; i < nc; i += E_THREADS) n += mass_key(m[i]) >= c;
                if (cta_sum(n, buf, turn++) >= (uint32_t)want) t = c;
            }
        }
        // every thread's run of keys: how many above t, how many equal; their sums over the threads before it
        const int run = (nc + E_THREADS - 1) / E_THREADS, i0 = min(nc, tid * run), i1 = min(nc, i0 + run);
        uint32_t above = 0, equal = 0;
        if (want > 0)
            for (int i = i0; i < i1; i++) {
                const uint32_t k = mass_key(m[i]);
                above += k > t;
                equal += k == t;
            }
        const uint32_t n_above = cta_sum(above, buf, turn++);
        uint32_t a = above, e = equal;  // inclusive sums
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t pa = __shfl_up_sync(D1_FULL_MASK, a, o), pe = __shfl_up_sync(D1_FULL_MASK, e, o);
            if (lane >= o) {
                a += pa;
                e += pe;
            }
        }
        if (lane == 31) {
            wsum[warp][0] = a;
            wsum[warp][1] = e;
        }
        __syncthreads();
        uint32_t ba = 0, be = 0;
        for (int w = 0; w < warp; w++) {
            ba += wsum[w][0];
            be += wsum[w][1];
        }
        const uint32_t ties = want - n_above;  // of the equal ones, the first `ties` are kept
        const uint32_t a0 = ba + a - above, e0 = be + e - equal;
        const size_t src0 = (size_t)g * it.cap, dst0 = (size_t)g * it.dst_cap;
        for (int s0 = p0; s0 < p1; s0 += E_LIST) {
            const int s1 = min(p1, s0 + E_LIST);
            if (want > 0) {
                uint32_t na = a0, ne = e0;
                for (int i = i0; i < i1; i++) {
                    const uint32_t k = mass_key(m[i]);
                    if (k > t || (k == t && ne < ties)) {
                        const int pos = (int)(na + min(ne, ties));
                        if (pos >= s0 && pos < s1) list[pos - s0] = i;
                    }
                    na += k > t;
                    ne += k == t;
                }
            }
            __syncthreads();
            const uint4 *k4 = reinterpret_cast<const uint4*>(it.k4), *v4 = reinterpret_cast<const uint4*>(it.v4);
            uint4 *dk4 = reinterpret_cast<uint4*>(it.dst_k4), *dv4 = reinterpret_cast<uint4*>(it.dst_v4);
            for (int c = tid; c < (s1 - s0) * 4; c += E_THREADS) {
                const int pos = s0 + (c >> 2), h = c & 1;
                const int i = pos < want ? list[pos - s0] : nc + pos - want;
                if (c & 2)
                    dv4[(dst0 + pos) * 2 + h] = __ldg(v4 + (src0 + i) * 2 + h);
                else
                    dk4[(dst0 + pos) * 2 + h] = __ldg(k4 + (src0 + i) * 2 + h);
            }
            for (int pos = s0 + tid; pos < s1; pos += E_THREADS) {
                const int i = pos < want ? list[pos - s0] : nc + pos - want;
                it.dst_kp[dst0 + pos] = it.kp[src0 + i];
                it.dst_vp[dst0 + pos] = it.vp[src0 + i];
                if (it.dst_mass) it.dst_mass[dst0 + pos] = m[i];
                if (it.kept) it.kept[dst0 + pos] = i;
            }
            __syncthreads();
        }
    }
}

bool bad_rows(const void* K, const void* V, int ldkv, int kv_heads) {
    return !K || !V || (((uintptr_t)K | (uintptr_t)V) & 15) || ldkv % 8 || ldkv < kv_heads * 64;
}

dim3 row_grid(int max_rows, int kv_heads, int n_seqs) {
    int x = (max_rows + A_ROWS - 1) / A_ROWS;
    x = x < 1 ? 1 : x > 4096 ? 4096 : x;
    return dim3(x, kv_heads * 2, n_seqs < kMaxGridZ ? n_seqs : kMaxGridZ);
}

}  // namespace

extern "C" int d1_kv4_append(const d1_half* K, const d1_half* V, int ldkv, const D1Kv4Seq* seqs, int n_seqs,
                             int max_rows, int kv_heads, cudaStream_t st) {
    if (n_seqs <= 0) return n_seqs == 0 ? 0 : -1;
    if (!seqs || max_rows < 0 || kv_heads <= 0 || kv_heads > 4096 || bad_rows(K, V, ldkv, kv_heads)) return -1;
    launch_pdl(k_kv4_append, row_grid(max_rows, kv_heads, n_seqs), 256, 0, st, K, V, ldkv, seqs, n_seqs);
    return (int)cudaGetLastError();
}

extern "C" int d1_kv4_load(const D1Kv4Seq* seqs, int n_seqs, int max_rows, int kv_heads, d1_half* K, d1_half* V,
                           int ldkv, cudaStream_t st) {
    if (n_seqs <= 0) return n_seqs == 0 ? 0 : -1;
    if (!seqs || max_rows < 0 || kv_heads <= 0 || kv_heads > 4096 || bad_rows(K, V, ldkv, kv_heads)) return -1;
    launch_pdl(k_kv4_load, row_grid(max_rows, kv_heads, n_seqs), 256, 0, st, seqs, n_seqs, K, V, ldkv);
    return (int)cudaGetLastError();
}

extern "C" int d1_kv4_evict(const D1Kv4Evict* items, int n_items, int max_len, int kv_heads, cudaStream_t st) {
    if (n_items <= 0) return n_items == 0 ? 0 : -1;
    if (!items || kv_heads <= 0 || kv_heads > 4096 || max_len < 0) return -1;
    const int z = n_items < kMaxGridZ ? n_items : kMaxGridZ;
    launch_pdl(k_kv4_evict, dim3(1, kv_heads, z), E_THREADS, 0, st, items, n_items);
    return (int)cudaGetLastError();
}

extern "C" int d1_kv4_error(void) {
    int e = 0;
    if (cudaDeviceSynchronize() != cudaSuccess) return -1;  // streams that do not wait for the default one, too
    if (cudaMemcpyFromSymbol(&e, g_kv4_err, sizeof(int)) != cudaSuccess) return -1;
    if (e) {
        const int z = 0;
        cudaMemcpyToSymbol(g_kv4_err, &z, sizeof(int));
    }
    return e;
}
