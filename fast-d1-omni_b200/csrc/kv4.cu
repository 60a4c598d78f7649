// Key/value caches held in 4 bits (format: include/d1kernels.h, D1Kv4Seq): rows into a cache and back, and eviction by
// accumulated attention weight. The attention over such caches is in kv4_attn.cu.
#include "attn_tc.cuh"
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
// Bound by HBM; append as much by the wait for its rows and by issue slots (0.66 of them while the SMs are busy, 8 ragged
// caches of up to 4096 rows: 14 us, and 10.5 at the copy rate). Append: 4 lanes per vector of 64 dimensions (twice 8
// elements, two words of codes a lane; the parameter's arithmetic, which every lane does, was a third of it with 8 lanes: 78
// us), 8 consecutive rows of one kv head per warp; a CTA takes 64 rows of (K or V, kv head) for each of PER to a thread,
// whose loads go out together: 4 where that still occupies every SM twice, otherwise 1 (32 x 4096 rows, 8 kv heads: 62 us
// with 4, 69 with 2, 83 with 8, and 53 at the copy rate; one prefix of 1025 rows: 2.5 us). Load: 8 lanes per vector, 4 rows
// to a thread (56, 57 and 66 us with 4, 8 and 2, and 53 at the copy rate).
constexpr int A_ROWS = 64, A_STEP = 32;

__device__ __forceinline__ bool append_ok(const D1Kv4Seq& s) {
    return (s.kv_len == 0 || (s.kv_start >= 0 && s.kv_len > 0)) && kv4_seq_ok(s) &&
           (long long)s.ext_len + s.kv_len <= s.ext_cap;
}

// Words of codes of one vector (this lane's twice 8 elements of it; four lanes a vector) and its parameter.
// round(x / step) without a division per element: t = x * (1 / step) is within 2^-18 of the quotient q, |q| < 15.6. As x
// has 11 significant bits and step 7, q either is k + 1/2 exactly or at least 2^-13 away from it; 768 + t, whose last place
// is 2^-14, is therefore 768 + k + 1/2 in the first case and on q's side of it in the second, and rounds as q does.
// (hi - lo) / 15 is rounded correctly, since whole multiples of 15 are common: one step of correction after the product
// with 1 / 15.
__device__ __forceinline__ void quantise16(const uint4 (&raw)[2], uint32_t (&word)[2], uint32_t& par) {
    const __half2* x2 = reinterpret_cast<const __half2*>(raw);
    __half2 mn = __float2half2_rn(0.f), mx = mn;  // the range, with zero in it; NaN stays
#pragma unroll
    for (int i = 0; i < 8; i++) {
        mn = __hmin2_nan(mn, x2[i]);
        mx = __hmax2_nan(mx, x2[i]);
    }
    __half2 ends = __halves2half2(__hneg(__hmin_nan(__low2half(mn), __high2half(mn))),
                                  __hmax_nan(__low2half(mx), __high2half(mx)));  // (-lo, hi)
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) ends = __hmax2_nan(ends, __shfl_xor_sync(D1_FULL_MASK, ends, o));
    const float nlo = __low2float(ends), hi = __high2float(ends), range = hi + nlo;
    constexpr float kFifteenth = 1.f / 15.f;
    float want = range * kFifteenth;
    want = fmaf(fmaf(-15.f, want, range), kFifteenth, want);
    // 7 significant bits upwards: carry into the mantissa's upper 6 bits; below 2^-14 a multiple of 2^-20
    const float step = want >= 6.103515625e-5f ? __uint_as_float((__float_as_uint(want) + 0x1ffffu) & ~0x1ffffu)
                                               : ceilf(want * 1048576.f) * 9.5367431640625e-7f;
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(step > 0.f ? step : 1.f));
    constexpr int kBias = 0x4b400000 + 768;  // 768 + t + 1.5 * 2^23 has round(t) + 768 in the low bits
    const int zero = min(__float_as_int(fmaf(nlo, inv, 768.f) + 12582912.f) - kBias, 15);
    int top = 15;  // |code - zero| * step stays within fp16; only a range above 65504 comes near
    if (step > 4096.f) top = min(15, __float2int_rd(__fdiv_rn(65504.f, step)));
    const int least = kBias + max(-top, -zero), most = kBias + min(top, 15 - zero);
    const uint64_t inv2 = f2_pack(inv, inv);
#pragma unroll
    for (int k = 0; k < 2; k++) {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(x2[4 * k + i]);
            float a, b;
            f2_unpack(f2_add(f2_fma(f2_pack(f.x, f.y), inv2, f2_pack(768.f, 768.f)), f2_pack(12582912.f, 12582912.f)), a, b);
            // the biases go out of all eight places together
            w += (uint32_t)max(least, min(most, __float_as_int(a))) << (4 * i);
            w += (uint32_t)max(least, min(most, __float_as_int(b))) << (16 + 4 * i);
        }
        word[k] = w + (uint32_t)(zero - kBias) * 0x11111111u;
    }
    par = (uint32_t)__half_as_ushort(__float2half_rn(step)) | (uint32_t)zero;
    if (!(range <= 131008.f)) {  // NaN or an infinity among them: a NaN step
        word[0] = word[1] = 0;
        par = 0x7e00u;
    }
}

template <int PER>
__global__ void __launch_bounds__(256) k_kv4_append(const __half* __restrict__ K, const __half* __restrict__ V,
                                                    int ldkv, const D1Kv4Seq* __restrict__ seqs, int n_seqs) {
    pdl_entry();
    const int sub = threadIdx.x & 3, row = threadIdx.x >> 2, g = blockIdx.y >> 1;
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
        for (int r0 = blockIdx.x * (A_ROWS * PER); r0 < s.kv_len; r0 += gridDim.x * (A_ROWS * PER)) {
            uint4 raw[PER][2];
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int r = r0 + i * A_ROWS + row;
                raw[i][0] = raw[i][1] = make_uint4(0, 0, 0, 0);
                if (r < s.kv_len) {
                    const uint4* x = reinterpret_cast<const uint4*>(src + (size_t)r * ldkv);
                    raw[i][0] = __ldcs(x);
                    raw[i][1] = __ldcs(x + 4);
                }
            }
#pragma unroll
            for (int i = 0; i < PER; i++) {
                if (r0 + i * A_ROWS >= s.kv_len) break;
                const int r = r0 + i * A_ROWS + row;
                uint32_t word[2], par;
                quantise16(raw[i], word, par);
                if (r < s.kv_len) {
                    codes[(size_t)r * 8] = word[0];
                    codes[(size_t)r * 8 + 4] = word[1];
                    if (sub == 0) pars[r] = (uint16_t)par;
                }
            }
        }
    }
}

template <int PER>
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
        for (int r0 = blockIdx.x * (A_STEP * PER); r0 < s.kv_len; r0 += gridDim.x * (A_STEP * PER)) {
            uint32_t word[PER], par[PER];
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int r = min(r0 + i * A_STEP + row, s.kv_len - 1);
                word[i] = codes[(size_t)r * 8];
                par[i] = pars[r];
            }
#pragma unroll
            for (int i = 0; i < PER; i++) {
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
// One CTA per (part of the destination, kv head, item). Every part finds the head's threshold (the mass of the last key to
// be kept) for itself, so that the parts need not wait for each other, and then moves its slice of the destination's rows.
// The keys are held in registers, a run of up to 32 to a thread. The threshold is found 11, 11 and 10 bits at a time from
// histograms in shared memory. What bounds it: few heads, the latency of a dozen dependent steps; many, HBM, which fetches
// about twice the bytes of a scattered choice of rows (runs of 32 and of 2 bytes).
// Tried and slower (192 heads of 8192 to 16384 keys, 4096 kept): the threshold 2 bits at a time by counting keys above
// three candidates, 109 us; 8 bits at a time, by one CTA 90 us, by a cluster that adds its histograms up through
// distributed shared memory 91 to 121 us.
constexpr int E_THREADS = 512, E_WARPS = E_THREADS / 32, E_PER = 32, E_KEYS = E_THREADS * E_PER, E_PER_SM = 2;
constexpr int E_BINS = 2048, E_SMEM = E_BINS * 4 + E_KEYS * 2;
static_assert(E_WARPS == 16 && E_BINS == 4 * E_THREADS && E_KEYS <= 65535, "scans of 16 warps, 4 bins a thread, 16-bit counts");

// A mass as an unsigned number of the same order, above 0: NaN as -inf, -0 as +0.
__device__ __forceinline__ uint32_t mass_key(float m) {
    const uint32_t b = m != m ? 0xff800000u : __float_as_uint(m + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Sum of v over the threads before this one, and over all of them; buf: a word per warp. Ends with every thread having
// read buf only after the next barrier.
__device__ __forceinline__ uint32_t cta_scan(uint32_t v, uint32_t* buf, uint32_t& all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t upto = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(D1_FULL_MASK, upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 31) buf[warp] = upto;
    __syncthreads();
    const uint32_t w = lane < E_WARPS ? buf[lane] : 0;
    all = __reduce_add_sync(D1_FULL_MASK, w);
    return upto - v + __reduce_add_sync(D1_FULL_MASK, lane < warp ? w : 0);
}

__global__ void __launch_bounds__(E_THREADS, E_PER_SM) k_kv4_evict(const D1Kv4Evict* __restrict__ items, int n_items) {
    extern __shared__ __align__(16) uint32_t e_smem[];
    uint32_t* hist = e_smem;                                       // [E_BINS]
    uint16_t* list = reinterpret_cast<uint16_t*>(hist + E_BINS);   // [E_KEYS]: kept keys of the stretch, of the part's slice
    __shared__ uint32_t buf[3][E_WARPS], found[3];
    pdl_entry();
    const int tid = threadIdx.x, g = blockIdx.y;
    for (int item = blockIdx.z; item < n_items; item += gridDim.z) {
        const D1Kv4Evict* it = items + item;
        const int len = it->len, cap = it->cap, dst_cap = it->dst_cap;
        const int keep = min(it->keep, len), recent = min(it->recent, keep);
        if (it->keep < 0 || it->recent < 0 || !kv4_cache_ok(len, cap, it->k4, it->v4, it->kp, it->vp) ||
            (len > 0 && !it->mass) || !kv4_cache_ok(keep, dst_cap, it->dst_k4, it->dst_v4, it->dst_kp, it->dst_vp) ||
            (((uintptr_t)it->mass | (uintptr_t)it->dst_mass | (uintptr_t)it->kept) & 3)) {
            if (tid == 0) table_error();
            continue;
        }
        const int slice = (keep + gridDim.x - 1) / gridDim.x;
        const int p0 = (int)min((long long)keep, (long long)blockIdx.x * slice), p1 = min(keep, p0 + slice);
        if (p0 >= p1) continue;
        const int nc = len - recent, want = keep - recent;  // keys to choose from, and how many
        const size_t src0 = (size_t)g * cap, dst0 = (size_t)g * dst_cap;
        const float* m = it->mass + src0;
        // moves n rows base + list[i] -> to + i, and the recent ones at positions q0 .. q0 + more - 1. Four threads to a
        // row, each with 16 bytes of K or V and one of the row's parameters, mass and index
        auto move = [&](int n, int base, int to, int q0, int more) {
            constexpr int UN = 4, ROWS = E_THREADS / 4;
            const int part = tid & 3;
            const uint4* from = reinterpret_cast<const uint4*>(part & 2 ? it->v4 : it->k4) + src0 * 2 + (part & 1);
            uint4* dst = reinterpret_cast<uint4*>(part & 2 ? it->dst_v4 : it->dst_k4) + dst0 * 2 + (part & 1);
            const uint16_t* par = reinterpret_cast<const uint16_t*>(part & 1 ? it->vp : it->kp) + src0;
            uint16_t* dst_par = reinterpret_cast<uint16_t*>(part & 1 ? it->dst_vp : it->dst_kp) + dst0;
            float* dst_mass = part == 2 ? it->dst_mass : nullptr;
            int* kept = part == 3 ? it->kept : nullptr;
            for (int r = tid >> 2; r < n + more; r += ROWS * UN) {
                uint4 x[UN];
                uint32_t y[UN];
#pragma unroll
                for (int i = 0; i < UN; i++) {
                    const int q = r + i * ROWS;
                    if (q >= n + more) continue;
                    const int src = q < n ? base + list[q] : nc + (q0 - want) + q - n;
                    x[i] = __ldg(from + (size_t)src * 2);
                    y[i] = part < 2 ? __ldg(par + src) : part == 2 ? __float_as_uint(__ldg(m + src)) : (uint32_t)src;
                }
#pragma unroll
                for (int i = 0; i < UN; i++) {
                    const int q = r + i * ROWS;
                    if (q >= n + more) continue;
                    const size_t at = q < n ? to + q : q0 + q - n;
                    dst[at * 2] = x[i];
                    if (part < 2) dst_par[at] = (uint16_t)y[i];
                    if (dst_mass) dst_mass[dst0 + at] = __uint_as_float(y[i]);
                    if (kept) kept[dst0 + at] = (int)y[i];
                }
            }
        };
        const int q0 = max(p0, want);  // the slice's recent rows
        int more = max(0, p1 - q0);
        if (p0 < want) {
            const bool resident = nc <= E_KEYS, wide = ((uintptr_t)m & 15) == 0;
            const int run = resident ? ((nc + E_THREADS - 1) / E_THREADS + 3) & ~3 : E_PER;  // keys of a thread
            uint32_t key[E_PER];  // keys base + tid * run + j; 0, below every key, behind the last
            auto fetch = [&](int base) {
                const int i0 = base + tid * run;
#pragma unroll
                for (int j = 0; j < E_PER; j += 4) {
                    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (j < run && wide && i0 + j + 3 < nc) {
                        x = __ldg(reinterpret_cast<const float4*>(m + i0 + j));
                    } else if (j < run) {
                        if (i0 + j < nc) x.x = __ldg(m + i0 + j);
                        if (i0 + j + 1 < nc) x.y = __ldg(m + i0 + j + 1);
                        if (i0 + j + 2 < nc) x.z = __ldg(m + i0 + j + 2);
                        if (i0 + j + 3 < nc) x.w = __ldg(m + i0 + j + 3);
                    }
                    key[j] = __float_as_uint(x.x);
                    key[j + 1] = __float_as_uint(x.y);
                    key[j + 2] = __float_as_uint(x.z);
                    key[j + 3] = __float_as_uint(x.w);
                }
#pragma unroll
                for (int j = 0; j < E_PER; j++)
                    key[j] = j < run && i0 + j < nc ? mass_key(__uint_as_float(key[j])) : 0;
            };
            if (resident) fetch(0);
            uint32_t t = 0, mask = 0, need = want;  // the threshold's known bits; how many of the keys sharing them are kept
            bool exact = false;                     // all of them are
#pragma unroll 1
            for (int d = 0; d < 3 && !exact; d++) {
                const int shift = d == 0 ? 21 : d == 1 ? 10 : 0;
                const uint32_t field = d == 2 ? 1023u : 2047u;
                reinterpret_cast<uint4*>(hist)[tid] = make_uint4(0, 0, 0, 0);
                __syncthreads();
                for (int base = 0; base < nc; base += E_KEYS) {
                    if (!resident) fetch(base);
#pragma unroll
                    for (int j = 0; j < E_PER; j++) {
                        if (j % 8 == 0 && j >= run) break;
                        if (key[j] != 0 && (key[j] & mask) == t) atomicAdd(hist + ((key[j] >> shift) & field), 1u);
                    }
                }
                __syncthreads();
                // the largest bin with `need` keys or more in it and above it: four bins a thread, from the top
                const uint4 h = reinterpret_cast<const uint4*>(hist)[E_THREADS - 1 - tid];
                const uint32_t v[4] = {h.w, h.z, h.y, h.x};
                uint32_t all, before = cta_scan((h.x + h.y) + (h.z + h.w), buf[d], all);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (before < need && need <= before + v[i]) {
                        found[0] = E_BINS - 1 - (tid * 4 + i);
                        found[1] = need - before;
                        found[2] = v[i];
                    }
                    before += v[i];
                }
                __syncthreads();
                t |= found[0] << shift;
                mask |= field << shift;
                need = found[1];
                exact = need == found[2];
            }
            if (exact) {  // every key with t's known bits is above a threshold just below them
                t = t > 0 ? t - 1 : 0;
                need = 0;
            }
            // the keys above t are kept, and the first `need` of those equal to it
            uint32_t above0 = 0, equal0 = 0;
            for (int base = 0; base < nc; base += E_KEYS) {
                if (!resident) fetch(base);
                uint32_t mine = 0;  // keys above t in the upper half, equal to it in the lower
#pragma unroll
                for (int j = 0; j < E_PER; j++) {
                    if (j % 8 == 0 && j >= run) break;
                    mine += (key[j] > t ? 0x10000u : 0u) + (key[j] == t && key[j] != 0 ? 1u : 0u);
                }
                __syncthreads();  // buf[0] and the list have been read
                uint32_t all;
                const uint32_t ahead = cta_scan(mine, buf[0], all);
                uint32_t na = above0 + (ahead >> 16), ne = equal0 + (ahead & 0xffffu);
                const int to = (int)(above0 + min(equal0, need));  // position of this stretch's first kept key
                const int first = max(to, p0);
#pragma unroll
                for (int j = 0; j < E_PER; j++) {
                    if (j % 8 == 0 && j >= run) break;
                    const bool is_a = key[j] > t, is_e = key[j] == t && key[j] != 0;
                    const int pos = (int)(na + min(ne, need));
                    if ((is_a || (is_e && ne < need)) && pos >= first && pos < p1) list[pos - first] = (uint16_t)(tid * run + j);
                    na += is_a;
                    ne += is_e;
                }
                above0 += all >> 16;
                equal0 += all & 0xffffu;
                __syncthreads();
                const bool last = base + E_KEYS >= nc;
                move(max(0, min(p1, (int)(above0 + min(equal0, need))) - first), base, first, q0, last ? more : 0);
                if (last) more = 0;
            }
            __syncthreads();  // the list and the histogram have been read
        }
        if (more > 0) move(0, 0, 0, q0, more);
    }
}

bool bad_rows(const void* K, const void* V, int ldkv, int kv_heads) {
    return !K || !V || (((uintptr_t)K | (uintptr_t)V) & 15) || ldkv % 8 || ldkv < kv_heads * 64;
}

dim3 row_grid(int max_rows, int rows, int kv_heads, int n_seqs) {
    const int x = max_rows <= rows ? 1 : max_rows > 4096 * rows ? 4096 : (max_rows - 1) / rows + 1;
    return dim3(x, kv_heads * 2, n_seqs < kMaxGridZ ? n_seqs : kMaxGridZ);
}

}  // namespace

extern "C" int d1_kv4_append(const d1_half* K, const d1_half* V, int ldkv, const D1Kv4Seq* seqs, int n_seqs,
                             int max_rows, int kv_heads, cudaStream_t st) {
    if (n_seqs <= 0) return n_seqs == 0 ? 0 : -1;
    if (!seqs || ((uintptr_t)seqs & 7) || max_rows < 0 || kv_heads <= 0 || kv_heads > 4096 || bad_rows(K, V, ldkv, kv_heads))
        return -1;
    const int sms = sm_count();
    if (!sms) return -1;
    const dim3 g4 = row_grid(max_rows, 4 * A_ROWS, kv_heads, n_seqs);
    if ((long long)g4.x * g4.y * g4.z >= 2 * sms)
        launch_pdl(k_kv4_append<4>, g4, 256, 0, st, K, V, ldkv, seqs, n_seqs);
    else
        launch_pdl(k_kv4_append<1>, row_grid(max_rows, A_ROWS, kv_heads, n_seqs), 256, 0, st, K, V, ldkv, seqs, n_seqs);
    return (int)cudaGetLastError();
}

extern "C" int d1_kv4_load(const D1Kv4Seq* seqs, int n_seqs, int max_rows, int kv_heads, d1_half* K, d1_half* V,
                           int ldkv, cudaStream_t st) {
    if (n_seqs <= 0) return n_seqs == 0 ? 0 : -1;
    if (!seqs || ((uintptr_t)seqs & 7) || max_rows < 0 || kv_heads <= 0 || kv_heads > 4096 || bad_rows(K, V, ldkv, kv_heads))
        return -1;
    launch_pdl(k_kv4_load<4>, row_grid(max_rows, 4 * A_STEP, kv_heads, n_seqs), 256, 0, st, seqs, n_seqs, K, V, ldkv);
    return (int)cudaGetLastError();
}

extern "C" int d1_kv4_evict(const D1Kv4Evict* items, int n_items, int max_len, int kv_heads, cudaStream_t st) {
    if (n_items <= 0) return n_items == 0 ? 0 : -1;
    if (!items || ((uintptr_t)items & 7) || kv_heads <= 0 || kv_heads > 4096 || max_len < 0) return -1;
    const int sms = sm_count();
    if (!sms) return -1;
    static unsigned long long done = 0;  // the shared-memory opt-in is per device
    int dev = 0;
    cudaGetDevice(&dev);
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(__atomic_load_n(&done, __ATOMIC_ACQUIRE) & bit)) {
        if (cudaFuncSetAttribute(k_kv4_evict, cudaFuncAttributeMaxDynamicSharedMemorySize, E_SMEM) != cudaSuccess) return -1;
        __atomic_fetch_or(&done, bit, __ATOMIC_RELEASE);
    }
    // parts to occupy the GPU, at most 8 (each finds the threshold again), of no less than 64 rows were every key kept
    const int z = n_items < kMaxGridZ ? n_items : kMaxGridZ;
    const long long heads = (long long)kv_heads * z, most = max_len > 448 ? 8 : (max_len + 63) / 64;
    long long parts = E_PER_SM * sms / heads;
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
