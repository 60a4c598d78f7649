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
// Bound by HBM. 8 lanes per vector of 64 dimensions (8 elements, one word of codes a lane), 4 consecutive rows of one kv
// head per warp, so that a warp's codes are one 128-byte run of the cache. CTA: 128 rows of (K or V, kv head), four to a
// thread, whose loads go out together.
constexpr int A_STEP = 32, A_PER = 4, A_ROWS = A_STEP * A_PER;

__device__ __forceinline__ bool append_ok(const D1Kv4Seq& s) {
    return s.kv_start >= 0 && s.kv_len >= 0 && kv4_seq_ok(s) && (long long)s.ext_len + s.kv_len <= s.ext_cap;
}

// One vector's word of codes (this lane's 8 elements) and parameter. round(x / step) without a division per element:
// t = x * (1 / step) is within 2^-19 of the quotient q, |q| < 15.6. As x has 11 significant bits and step 7, q either is
// k + 1/2 exactly or at least 2^-13 away from it; t rounded to a multiple of 2^-14 (by adding and taking away 768) is
// therefore k + 1/2 in the first case and on q's side of it in the second, and rounds as q does.
__device__ __forceinline__ void quantise8(const uint4& raw, uint32_t& word, uint32_t& par) {
    const __half2* x2 = reinterpret_cast<const __half2*>(&raw);
    __half2 mn = __float2half2_rn(0.f), mx = mn, bad = mn;  // the range, with zero in it
#pragma unroll
    for (int i = 0; i < 4; i++) {
        mn = __hmin2(mn, x2[i]);
        mx = __hmax2(mx, x2[i]);
        bad = __hfma2(x2[i], __float2half2_rn(0.f), bad);  // NaN after a NaN or an infinity
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        mn = __hmin2(mn, __shfl_xor_sync(D1_FULL_MASK, mn, o));
        mx = __hmax2(mx, __shfl_xor_sync(D1_FULL_MASK, mx, o));
        bad = __hadd2(bad, __shfl_xor_sync(D1_FULL_MASK, bad, o));
    }
    const float lo = __half2float(__hmin(__low2half(mn), __high2half(mn)));
    const float hi = __half2float(__hmax(__low2half(mx), __high2half(mx)));
    // 7 significant bits upwards: carry into the mantissa's upper 6 bits; below 2^-14 a multiple of 2^-20
    const float want = __fdiv_rn(hi - lo, 15.f);
    const float step = want >= 6.103515625e-5f ? __uint_as_float((__float_as_uint(want) + 0x1ffffu) & ~0x1ffffu)
                                               : ceilf(want * 1048576.f) * 9.5367431640625e-7f;
    const float div = step > 0.f ? step : 1.f, inv = __fdiv_rn(1.f, div);
    const int zero = min(__float2int_rn(__fdiv_rn(-lo, div)), 15);
    int top = 15;  // |code - zero| * step stays within fp16; only a range above 65504 comes near
    if (step > 4096.f) top = min(15, __float2int_rd(__fdiv_rn(65504.f, div)));
    constexpr int kBias = 0x4b400000;  // 1.5 * 2^23: its sum with t is round(t) in the low bits
    const int least = kBias + max(-top, -zero), most = kBias + min(top, 15 - zero);
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(x2[i]);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const float t = ((h ? f.y : f.x) * inv + 768.f) - 768.f;
            const int q = max(least, min(most, __float_as_int(t + 12582912.f)));
            w += (uint32_t)q << (16 * h + 4 * i);  // the biases go out of all eight places together
        }
    }
    word = w + (uint32_t)(zero - kBias) * 0x11111111u;
    par = (uint32_t)__half_as_ushort(__float2half_rn(step)) | (uint32_t)zero;
    if (__hisnan(__low2half(bad)) || __hisnan(__high2half(bad))) {
        word = 0;
        par = 0x7e00u;  // a NaN step
    }
}

__global__ void __launch_bounds__(256) k_kv4_append(const __half* __restrict__ K, const __half* __restrict__ V,
                                                    int ldkv, const D1Kv4Seq* __restrict__ seqs, int n_seqs) {
    pdl_entry();
    const int sub = threadIdx.x & 7, row = threadIdx.x >> 3, g = blockIdx.y >> 1;
    const bool is_v = blockIdx.y & 1;
    for (int sq = blockIdx.z; sq < n_seqs; sq += gridDim.z) {
        const D1Kv4Seq s = seqs[sq];
        if (!append_ok(s)) {
            if (threadIdx.x == 0) table_error();
            continue;
        }
        const __half* src = (is_v ? V : K) + (size_t)s.kv_start * ldkv + g * 64 + sub * 8;
        const size_t at = (size_t)g * s.ext_cap + s.ext_len;
        uint32_t* codes = reinterpret_cast<uint32_t*>(is_v ? s.v4 : s.k4) + at * 8 + sub;
        uint16_t* pars = reinterpret_cast<uint16_t*>(is_v ? s.vp : s.kp) + at;
        for (int r0 = blockIdx.x * A_ROWS; r0 < s.kv_len; r0 += gridDim.x * A_ROWS) {
            uint4 raw[A_PER];
#pragma unroll
            for (int i = 0; i < A_PER; i++) {
                const int r = r0 + i * A_STEP + row;
                raw[i] = r < s.kv_len ? __ldcs(reinterpret_cast<const uint4*>(src + (size_t)r * ldkv)) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < A_PER; i++) {
                if (r0 + i * A_STEP >= s.kv_len) break;
                const int r = r0 + i * A_STEP + row;
                uint32_t word, par;
                quantise8(raw[i], word, par);
                if (r < s.kv_len) {
                    codes[(size_t)r * 8] = word;
                    if (sub == 0) pars[r] = (uint16_t)par;
                }
            }
        }
    }
}

__global__ void __launch_bounds__(256) k_kv4_load(const D1Kv4Seq* __restrict__ seqs, int n_seqs, __half* __restrict__ K,
                                                  __half* __restrict__ V, int ldkv) {
    pdl_entry();
    const int sub = threadIdx.x & 7, row = threadIdx.x >> 3, g = blockIdx.y >> 1;
    const bool is_v = blockIdx.y & 1;
    for (int sq = blockIdx.z; sq < n_seqs; sq += gridDim.z) {
        const D1Kv4Seq s = seqs[sq];
        if (!append_ok(s)) {
            if (threadIdx.x == 0) table_error();
            continue;
        }
        __half* dst = (is_v ? V : K) + (size_t)s.kv_start * ldkv + g * 64 + sub * 8;
        const size_t at = (size_t)g * s.ext_cap + s.ext_len;
        const uint32_t* codes = reinterpret_cast<const uint32_t*>(is_v ? s.v4 : s.k4) + at * 8 + sub;
        const uint16_t* pars = reinterpret_cast<const uint16_t*>(is_v ? s.vp : s.kp) + at;
        for (int r0 = blockIdx.x * A_ROWS; r0 < s.kv_len; r0 += gridDim.x * A_ROWS) {
            uint32_t word[A_PER], par[A_PER];
#pragma unroll
            for (int i = 0; i < A_PER; i++) {
                const int r = min(r0 + i * A_STEP + row, s.kv_len - 1);
                word[i] = codes[(size_t)r * 8];
                par[i] = pars[r];
            }
#pragma unroll
            for (int i = 0; i < A_PER; i++) {
                const int r = r0 + i * A_STEP + row;
                const uint32_t p2 = par[i] * 0x00010001u, st = kv4_step2(p2);
                uint32_t z0, z1, v[4];
                kv4_zero(p2, z0, z1);
                kv4_expand(word[i], z0, z1, v);
                if (r < s.kv_len)
                    __stcs(reinterpret_cast<uint4*>(dst + (size_t)r * ldkv),
                           make_uint4(h2_mul(v[0], st), h2_mul(v[1], st), h2_mul(v[2], st), h2_mul(v[3], st)));
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ evict
// One CTA per (part of the destination, kv head, item). Every part finds the head's threshold for itself (the masses are
// small beside the rows that move), so that the parts need not wait for each other; then each copies its slice of the
// destination's rows. The threshold is found 8 bits at a time from histograms with a column per lane: no two lanes of a
// warp count in the same place, however alike the masses are.
constexpr int E_THREADS = 512, E_WARPS = E_THREADS / 32, E_KEYS = 16384, E_LIST = 4096;
constexpr int E_SMEM = (E_KEYS + 256 * 32) * 4;
static_assert(E_LIST <= 256 * 32 && E_KEYS / E_THREADS * E_WARPS == E_THREADS, "the list replaces the histogram");

// A mass as an unsigned number of the same order: NaN as -inf, -0 as +0.
__device__ __forceinline__ uint32_t mass_key(float m) {
    const uint32_t b = m != m ? 0xff800000u : __float_as_uint(m + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__global__ void __launch_bounds__(E_THREADS, 2) k_kv4_evict(const D1Kv4Evict* __restrict__ items, int n_items) {
    extern __shared__ __align__(16) uint32_t e_smem[];
    uint32_t* keys = e_smem;              // [E_KEYS]: the head's keys, or a stretch of them
    uint32_t* hist = e_smem + E_KEYS;     // [256][32]
    int* list = reinterpret_cast<int*>(hist);
    __shared__ uint32_t bins[256], cnt[E_THREADS], wsum[E_WARPS], found[2];
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
        const int p0 = (int)min((long long)keep, (long long)blockIdx.x * per), p1 = min(keep, p0 + per);
        if (p0 >= p1) continue;
        const int nc = it.len - recent, want = keep - recent;  // keys to choose from, and how many
        const bool choose = p0 < want;                         // (a slice of recent rows alone needs no threshold)
        const float* m = it.mass + (size_t)g * it.cap;
        const bool resident = nc <= E_KEYS;
        auto stretch = [&](int base) {  // keys base .. into shared memory; zeros, below every key, behind the last
            __syncthreads();
            const int n = min(nc - base, E_KEYS), up = (n + E_THREADS - 1) / E_THREADS * E_THREADS;
            for (int i = tid; i < up; i += E_THREADS) keys[i] = i < n ? mass_key(__ldg(m + base + i)) : 0;
            __syncthreads();
            return n;
        };
        uint32_t t = 0, mask = 0, need = want;  // the threshold's known bits, and how many keys of those that share them
        if (choose) {
            if (resident) stretch(0);
#pragma unroll 1
            for (int shift = 24; shift >= 0; shift -= 8) {
                for (int i = tid; i < 256 * 32; i += E_THREADS) hist[i] = 0;
                __syncthreads();
                for (int base = 0; base < nc; base += E_KEYS) {
                    const int n = resident ? nc : stretch(base);
                    for (int i = tid; i < n; i += E_THREADS) {
                        const uint32_t k = keys[i];
                        if ((k & mask) == t) atomicAdd(hist + ((k >> shift) & 255) * 32 + lane, 1u);
                    }
                }
                __syncthreads();
                for (int b = warp; b < 256; b += E_WARPS) {
                    const uint32_t v = __reduce_add_sync(D1_FULL_MASK, hist[b * 32 + lane]);
                    if (lane == 0) bins[b] = v;
                }
                __syncthreads();
                if (warp == 0) {  // the largest bin with at least `need` keys in it and above it
                    uint32_t v[8], own = 0;
#pragma unroll
                    for (int i = 0; i < 8; i++) own += v[i] = bins[255 - (lane * 8 + i)];
                    uint32_t upto = own;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const uint32_t x = __shfl_up_sync(D1_FULL_MASK, upto, o);
                        if (lane >= o) upto += x;
                    }
                    uint32_t before = upto - own;
                    if (before < need && need <= upto) {
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            if (before < need && need <= before + v[i]) {
                                found[0] = 255 - (lane * 8 + i);
                                found[1] = need - before;
                                break;
                            }
                            before += v[i];
                        }
                    }
                }
                __syncthreads();
                t |= found[0] << shift;
                need = found[1];
                mask |= 255u << shift;
            }
        }
        // of the keys equal to t, the first `need` are kept. Positions: keys above t and kept equal ones before
        const size_t src0 = (size_t)g * it.cap, dst0 = (size_t)g * it.dst_cap;
        for (int s0 = p0; s0 < p1; s0 += E_LIST) {
            const int s1 = min(p1, s0 + E_LIST);
            if (s0 < want) {
                uint32_t above0 = 0, equal0 = 0;
                for (int base = 0; base < nc; base += E_KEYS) {
                    const int n = resident ? nc : stretch(base);
                    // the counts of 32 successive keys (above t in the upper half, equal in the lower), summed up
                    const int groups = (n + 31) / 32;
                    for (int q = warp; q < groups; q += E_WARPS) {
                        const uint32_t k = q * 32 + lane < n ? keys[q * 32 + lane] : 0;
                        const uint32_t a = __ballot_sync(D1_FULL_MASK, k > t);
                        const uint32_t e = __ballot_sync(D1_FULL_MASK, k == t && q * 32 + lane < n);
                        if (lane == 0) cnt[q] = (uint32_t)__popc(a) << 16 | __popc(e);
                    }
                    __syncthreads();
                    const uint32_t own = tid < groups ? cnt[tid] : 0;
                    uint32_t upto = own;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const uint32_t x = __shfl_up_sync(D1_FULL_MASK, upto, o);
                        if (lane >= o) upto += x;
                    }
                    if (lane == 31) wsum[warp] = upto;
                    __syncthreads();
                    uint32_t add = 0, all = 0;
                    for (int w = 0; w < E_WARPS; w++) {
                        add += w < warp ? wsum[w] : 0;
                        all += wsum[w];
                    }
                    cnt[tid] = upto - own + add;
                    __syncthreads();
                    for (int q = warp; q < groups; q += E_WARPS) {
                        const int i = q * 32 + lane;
                        const uint32_t k = i < n ? keys[i] : 0;
                        const bool is_a = k > t, is_e = k == t && i < n;
                        const uint32_t a = __ballot_sync(D1_FULL_MASK, is_a), e = __ballot_sync(D1_FULL_MASK, is_e);
                        const uint32_t lower = (1u << lane) - 1, c = cnt[q];
                        const uint32_t na = above0 + (c >> 16) + __popc(a & lower);
                        const uint32_t ne = equal0 + (c & 0xffffu) + __popc(e & lower);
                        const int pos = (int)(na + min(ne, need));
                        if ((is_a || (is_e && ne < need)) && pos >= s0 && pos < s1) list[pos - s0] = base + i;
                    }
                    above0 += all >> 16;
                    equal0 += all & 0xffffu;
                    __syncthreads();
                }
            }
            auto source = [&](int pos) { return pos < want ? list[pos - s0] : nc + pos - want; };
            const uint4 *k4 = reinterpret_cast<const uint4*>(it.k4), *v4 = reinterpret_cast<const uint4*>(it.v4);
            uint4 *dk4 = reinterpret_cast<uint4*>(it.dst_k4), *dv4 = reinterpret_cast<uint4*>(it.dst_v4);
            // a row is 4 pieces of 16 bytes: K, V and their halves
            const int half = tid & 1;
            const uint4* from = (tid & 2 ? v4 : k4) + src0 * 2 + half;
            uint4* to = (tid & 2 ? dv4 : dk4) + dst0 * 2 + half;
            constexpr int UN = 4, ROWS = E_THREADS / 4;
            for (int r = s0 + (tid >> 2); r < s1; r += ROWS * UN) {
                uint4 x[UN];
#pragma unroll
                for (int i = 0; i < UN; i++)
                    if (r + i * ROWS < s1) x[i] = __ldg(from + (size_t)source(r + i * ROWS) * 2);
#pragma unroll
                for (int i = 0; i < UN; i++)
                    if (r + i * ROWS < s1) to[(size_t)(r + i * ROWS) * 2] = x[i];
            }
            for (int pos = s0 + tid; pos < s1; pos += E_THREADS) {
                const int i = source(pos);
                const d1_half a = it.kp[src0 + i], b = it.vp[src0 + i];
                const float w = m[i];
                it.dst_kp[dst0 + pos] = a;
                it.dst_vp[dst0 + pos] = b;
                if (it.dst_mass) it.dst_mass[dst0 + pos] = w;
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
    static unsigned long long done = 0;  // the shared-memory opt-in is per device
    int dev = 0;
    cudaGetDevice(&dev);
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(__atomic_load_n(&done, __ATOMIC_ACQUIRE) & bit)) {
        if (cudaFuncSetAttribute(k_kv4_evict, cudaFuncAttributeMaxDynamicSharedMemorySize, E_SMEM) != cudaSuccess) return -1;
        __atomic_fetch_or(&done, bit, __ATOMIC_RELEASE);
    }
    // two CTAs fit an SM: enough parts to occupy them all, of no less than 128 rows were every key kept
    const int z = n_items < kMaxGridZ ? n_items : kMaxGridZ;
    const long long heads = (long long)kv_heads * z;
    long long parts = (2 * 148 + heads - 1) / heads, most = (max_len + 127) / 128;
    parts = parts > most ? most : parts;
    launch_pdl(k_kv4_evict, dim3(parts < 1 ? 1 : (unsigned)parts, kv_heads, z), E_THREADS, E_SMEM, st, items, n_items);
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
