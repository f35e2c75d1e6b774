// lgx_filter.hip -- a token for each row of logits by temperature, top-k, top-p and
// min-p, with a given random number per row.
#include "lgx_device.h"

// ---------------------------------------------------------------------------
// Definition: lgx_sample_filtered in lgx.h.  The weights of a row's tokens are w =
// exp((l - M) / T), M the row's largest logit; with the tokens in order of (logit
// descending, index ascending) every filter keeps a prefix, and the draw goes over the
// kept tokens in order of index.
//
// The scan reads every logit once: the largest of each 64 (cmax), the largest of each 4096
// and the sum of their weights.  The pick, a workgroup per row, derives from them a
// logit tau below which no token can be kept, reads again only the runs of 64 whose largest
// reaches it, and selects among those tokens, in LDS.  A row without filters needs the
// sums and one run of 4096.  Rows of which top-p or min-p keep more tokens than that list
// holds (wide) are left to one more launch: bins of the weights by 4096 logits, and by the
// workgroup that brings a row's last bins the choice from them.
//
// What bounds it, at 151936 logits: many rows the scan, which reads at 4.1 to 5.2 TB/s
// (512 rows of all kinds 60 us of 138; 256 rows without sums 35), and its weights where
// top-p or no filter needs their sums (another 25 us of 256 rows: binary64 arithmetic).  One
// row its chain of memory rounds and barriers: scan 3.5 us, pick 4 to 10 us, 1 us for the
// launch that finds no wide row; 71 us for a row of which 100000 tokens are kept.
//   One pass over the row by its own workgroup in place of scan and pick: 152064 logits at
//   one compute unit's rate are 20 us or more a pass, and small batches need all of them.
//   Tokens read by the runs' maxima: a row with top-k 50 reads 60 to 100 runs of 2374.
//   Wide rows in three launches (bins, the deciding tokens listed by all slices, choice): one
//   58 against 71 us, 256 of them 237 against 245, 512 mixed rows 127 against 138; but 3 us
//   more for every call without a wide row (top-k 50 and top-p 17.9 against 14.9), and 2 to
//   3 us of the host's.
//
// Sums decide between tokens, so they must not depend on their order: the weights that a
// selection adds up are whole multiples of 2^-42 in 64-bit integers, each rounded by 2^-43
// at most (the smaller ones to nothing); the scan's are binary64.  exp is binary64
// arithmetic with a relative error of 1.5e-13 (sf_root_exp).  A sum over n tokens is
// so off by n 2^-43 at most and by 2^-41 of itself: 6e-8 for half a million tokens of
// 2^-43 each behind one of 1, some 1e-12 for a few.  A finer unit that holds 1e-12 over 2^19
// tokens would take sums of 80 bits.
// ---------------------------------------------------------------------------
#define SF_ONE 0x1p42                             // 2^19 weights stay below 2^62
#define SF_LIST LGX_SF_LIST                       // tokens kept in LDS

// e^x for x <= 0: x = (256 n + j) ln 2 / 256 + r, 2^(j/256) from a table (sf_roots), e^r by its
// Taylor polynomial of degree 3 (|r| <= 0.00136: the term after it is under 2e-13).  The
// argument comes in units of ln 2 / 256.
#define SF_ROOTS 256
__device__ __forceinline__ double sf_root_exp(double y, const double* roots, int& n) {
    const double k = rint(y), r = (y - k) * (0.69314718055994530942 / SF_ROOTS);
    double p = fma(r, 1.0 / 6.0, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    const int i = (int)k;
    n = i >> 8;                                   // floor
    return roots[i & (SF_ROOTS - 1)] * p;
}
#define SF_UNITS_PER (SF_ROOTS * 1.4426950408889634074)   // of an argument's units in 1
__device__ __forceinline__ double sf_exp(double y, const double* roots) {
    int n;
    const double p = sf_root_exp(y, roots, n);
    return y > -700.0 * SF_UNITS_PER ? __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, p) + ((uint64_t)(int64_t)n << 52)) : 0.0;
}
// In units of 2^-42, rounded, for x > -30.5: a shift of the bits (a conversion of binary64
// to a 64-bit integer takes as long as all of the above).
__device__ __forceinline__ uint64_t sf_units(double y, const double* roots) {
    int n;
    const uint64_t bits = __builtin_bit_cast(uint64_t, sf_root_exp(y, roots, n));
    const int down = 52 - 42 + 1023 - (int)(bits >> 52) - n;
    const uint64_t m = (bits & ((1ull << 52) - 1)) | 1ull << 52;
    return down > 54 ? 0 : (m + (1ull << (down - 1))) >> down;
}
// The table, by threads 0 .. 255: e^x of [0, 0.7) by its Taylor polynomial of degree 15
// (the term after it is under 2e-16).
__device__ __forceinline__ void sf_roots(double* roots) {
    if (threadIdx.x >= SF_ROOTS) return;
    constexpr struct Inverse {                    // 1 / i!
        double c[16];
        constexpr Inverse() : c() {
            double f = 1.0;
            for (int i = 0; i < 16; ++i) {
                c[i] = 1.0 / f;
                f *= i + 1;
            }
        }
    } t;
    const double x = threadIdx.x * (0.69314718055994530942 / SF_ROOTS);
    double p = t.c[15];
#pragma unroll
    for (int i = 14; i >= 0; --i) p = fma(p, x, t.c[i]);
    roots[threadIdx.x] = p;
}
// Weight of logit l by the maximum M; 0 for NaN and -inf, 1 for the maximum, whatever it is.
__device__ __forceinline__ double sf_weight(float l, float M, double inv, const double* roots) {
    const double y = ((double)l - (double)M) * inv;
    return l == M ? 1.0 : l > -__builtin_inff() && l < M ? sf_exp(y, roots) : 0.0;
}

__device__ __forceinline__ uint64_t sf_weight_units(float l, float M, double inv, const double* roots) {
    const double y = ((double)l - (double)M) * inv;
    return l == M ? 1ull << 42 : l > -__builtin_inff() && y > -30.5 * SF_UNITS_PER ? sf_units(y, roots) : 0;
}

struct SfRow {
    double inv;                                   // 1 / T in units of ln 2 / 256
    float p, mp;                                  // top_p (1: none), min_p (0: none)
    int k;                                        // top_k (0: none)
    bool greedy;
    __device__ __forceinline__ bool plain() const { return !k && p >= 1.0f && mp <= 0.0f; }
    // whether the sum of all weights is needed
    __device__ __forceinline__ bool sums() const { return !greedy && !k && (p < 1.0f || mp <= 0.0f); }
};
__device__ __forceinline__ float sf_temperature(const lgx_filter_args& a, int row) { return a.temperature ? a.temperature[row] : 1.0f; }
__device__ __forceinline__ SfRow sf_row(const lgx_filter_args& a, int row) {
    SfRow r;
    const float T = sf_temperature(a, row);
    r.greedy = !(T > 0.0f);
    r.inv = SF_UNITS_PER / (double)T;
    const int k = a.top_k ? a.top_k[row] : 0;
    r.k = k > 0 && k < a.vocab ? k : 0;
    const float p = a.top_p ? a.top_p[row] : 1.0f, mp = a.min_p ? a.min_p[row] : 0.0f;
    r.p = p < 1.0f ? fmaxf(p, 0.0f) : 1.0f;       // NaN: none
    r.mp = mp > 0.0f ? fminf(mp, 1.0f) : 0.0f;
    return r;
}

// Inclusive sums over 16 lanes, and over all lanes, as wave_scan, of 64-bit integers or
// binary64 numbers.
template <int C, int R, class V>
__device__ __forceinline__ V scan64_step(V v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, C, R, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), C, R, 0xf, false);
    return v + __builtin_bit_cast(V, (uint64_t)hi << 32 | lo);
}
template <class V>
__device__ __forceinline__ V row_scan64(V v) {
    v = scan64_step<0x111, 0xf>(v);
    v = scan64_step<0x112, 0xf>(v);
    v = scan64_step<0x114, 0xf>(v);
    return scan64_step<0x118, 0xf>(v);
}
template <class V>
__device__ __forceinline__ V wave_scan64(V v) {
    v = scan64_step<0x142, 0xa>(row_scan64(v));
    return scan64_step<0x143, 0xc>(v);
}

// Workgroup (4096 logits, row): thread t holds 4 (256 i + t) .. + 3 of them.
extern "C" __global__ __launch_bounds__(256) void lgx_k_filter_scan(const lgx_filter_args a) {
    __shared__ float mx_s[4];
    __shared__ double sum_s[4], roots[SF_ROOTS];
    const int tid = threadIdx.x, sl = blockIdx.x, row = blockIdx.y;
    if (a.slots && sl == 0 && row == 0 && tid == 0) *a.wide_n = 0;
    sf_roots(roots);
    const SfRow r = sf_row(a, row);
    const float* x = a.logits + (int64_t)row * a.ld;
    const float ninf = -__builtin_inff();
    float v[4][4], mt = ninf;
    const int base = sl * LGX_SF_SLICE + 4 * tid;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int e = base + 1024 * i;
        if (a.vec && e + 4 <= a.vocab) {
            const float4 f = *(const float4*)(x + e);
            v[i][0] = f.x, v[i][1] = f.y, v[i][2] = f.z, v[i][3] = f.w;
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) v[i][c] = e + c < a.vocab ? x[e + c] : ninf;
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // fmaxf leaves a NaN behind; a run of NaN alone has no largest
        float m = fmaxf(fmaxf(fmaxf(ninf, v[i][0]), v[i][1]), fmaxf(fmaxf(ninf, v[i][2]), v[i][3]));
        mt = fmaxf(mt, m);
        m = max8(m);
        m = fmaxf(m, dpp_f<0x140>(m));            // of 16 lanes
        if ((tid & 15) == 0) a.cmax[((int64_t)row * a.nslices + sl) * 64 + 16 * i + (tid >> 4)] = m;
    }
    mt = wave_max(mt);
    if ((tid & 63) == 0) mx_s[tid >> 6] = mt;
    __syncthreads();
    const float M = fmaxf(fmaxf(mx_s[0], mx_s[1]), fmaxf(mx_s[2], mx_s[3]));
    if (tid == 0) a.smax[(int64_t)row * a.nslices + sl] = M;
    if (!r.sums()) return;                        // uniform
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) s += sf_weight(v[i][c], M, r.inv, roots);
    s = wave_scan64(s);
    if ((tid & 63) == 63) sum_s[tid >> 6] = s;
    __syncthreads();
    if (tid == 0) a.sum[(int64_t)row * a.nslices + sl] = sum_s[0] + sum_s[1] + (sum_s[2] + sum_s[3]);
}

// Order of logits as unsigned numbers: ascending keys are descending logits, -0 is 0.
__device__ __forceinline__ uint32_t sf_key(float l) {
    const uint32_t u = __float_as_uint(l + 0.0f);
    return u & 0x80000000u ? u : ~(u | 0x80000000u);
}

__device__ __forceinline__ float sf_logit(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key : ~key & 0x7fffffffu); }

#define SF_NT 1024
#define SF_BINS 1024                              // of a selection's first step
#define SF_FEW 448                                // elements that one wave chooses among (64 more: its registers run out)
#define SF_GUESS 256                              // runs whose tokens are tried first for top-p
struct SfLds {
    union {
        uint64_t bins[SF_BINS];
        uint16_t runs[SF_LIST];                   // runs of 64 logits to read
    };
    uint64_t wi[SF_LIST];                         // weight << 20 | index
    uint32_t key[SF_LIST];
    uint64_t few[SF_FEW];                         // measures of a selection's second step
    uint32_t few_key[SF_FEW];
    uint64_t wave[SF_NT / 64];
    double dwave[SF_NT / 64];
    double roots[SF_ROOTS];                       // 2^(j / 256)
    uint64_t below;
    int found, count;
};
static_assert(sizeof(SfLds) <= 81920, "two workgroups per compute unit");
static_assert(LGX_SF_VOCAB <= 1 << 20 && LGX_SF_VOCAB / LGX_SF_CHUNK <= 65536, "an index has 20 bits, a run 16");

template <class V>
__device__ __forceinline__ V lane_of(V v, int lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(V, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane) << 32 |
                                     (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane));
}
__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) { return lane_of(wave_scan64(v), 63); }

// What the waves of the workgroup have together and those before this one, from each
// wave's uniform value.  (Sixteen lanes sum sixteen waves: sixteen waves on four SIMDs
// make every instruction cost 16 cycles, and a loop over the waves 1 us.)
template <class V>
__device__ __forceinline__ V sf_waves(V mine, V* waves, V& total) {
    static_assert(SF_NT == 1024, "a lane per wave");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (lane == 0) waves[wave] = mine;
    __syncthreads();
    const V w = row_scan64(waves[lane & 15]);
    total = lane_of(w, 15);
    const V before = wave ? lane_of(w, wave - 1) : V(0);
    __syncthreads();
    return before;
}
// Inclusive sums over the workgroup's threads.
template <class V>
__device__ __forceinline__ V sf_scan(V v, V* waves, V& total) {
    v = wave_scan64(v);
    return sf_waves(lane_of(v, 63), waves, total) + v;
}
// Their sum alone.
__device__ __forceinline__ uint64_t sf_sum(uint64_t v, uint64_t* waves) {
    uint64_t total;
    sf_waves(wave_sum64(v), waves, total);
    return total;
}

// The smallest key of one wave's E elements per lane such that those up to it measure
// `need` or more (no more than all); below: the measure of smaller keys.  Bisection
// of the keys' range; sum(k): the measure of keys <= k.
template <class F>
__device__ __forceinline__ uint32_t sf_bisect(uint32_t lo, uint32_t hi, uint64_t need, uint64_t& below, const F& sum) {
    below = 0;
    while (lo < hi) {                             // uniform
        const uint32_t mid = lo + (hi - lo) / 2;
        const uint64_t s = sum(mid);
        if (s >= need) {
            hi = mid;
        } else {
            lo = mid + 1;
            below = s;                            // the last such sum is that of keys < lo
        }
    }
    return lo;
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// The row's tokens that can be kept, in LDS or in memory: load(i) is element i, the others
// say of it whether it counts (not below tau), its key, index and weight.  Elements
// ascend by index.  U: loads in flight per thread.
struct SfInLds {
    static constexpr int U = 1;
    struct Raw {
        uint32_t key;
        uint64_t wi;
    };
    const SfLds& s;
    int n;
    __device__ __forceinline__ Raw load(int i) const { return {s.key[i], s.wi[i]}; }
    __device__ __forceinline__ bool valid(const Raw&) const { return true; }
    __device__ __forceinline__ uint32_t key(const Raw& x) const { return x.key; }
    __device__ __forceinline__ int index(const Raw& x, int) const { return (int)(x.wi & 0xfffff); }
    __device__ __forceinline__ uint64_t weight(const Raw& x) const { return x.wi >> 20; }
};
struct SfInRow {
    static constexpr int U = 8;
    typedef float Raw;
    const float* x;
    int n;
    float tau, M;
    double inv;
    const double* roots;
    __device__ __forceinline__ float load(int i) const { return x[i]; }
    __device__ __forceinline__ bool valid(float v) const { return v >= tau; }
    __device__ __forceinline__ uint32_t key(float v) const { return sf_key(v); }
    __device__ __forceinline__ int index(float, int i) const { return i; }
    __device__ __forceinline__ uint64_t weight(float v) const { return sf_weight_units(v, M, inv, roots); }
};
// f(element, i) for the elements first, first + step, .. below end
template <class S, class F>
__device__ __forceinline__ void sf_each(const S& e, int first, int end, int step, const F& f) {
    for (int i0 = first; i0 < end; i0 += step * S::U) {
        typename S::Raw x[S::U];
#pragma unroll
        for (int u = 0; u < S::U; ++u) x[u] = e.load(min(i0 + u * step, end - 1));
#pragma unroll
        for (int u = 0; u < S::U; ++u)
            if (i0 + u * step < end) f(x[u], i0 + u * step);
    }
}

// f(16 logits, their indexes by a function) for a row's logits; NaN past its end.
template <class F>
__device__ __forceinline__ void sf_row_each(const float* x, int V, int vec, const F& f) {
    const int tid = threadIdx.x, n4 = vec ? V / 4 : 0;
    const float nan = __builtin_nanf("");
    float v[16];
    for (int i0 = tid; i0 - tid < n4; i0 += 4 * SF_NT) {   // uniform
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = i0 + u * SF_NT;
            const float4 w = ((const float4*)x)[min(i, n4 - 1)];
            v[4 * u] = i < n4 ? w.x : nan;
            v[4 * u + 1] = i < n4 ? w.y : nan;
            v[4 * u + 2] = i < n4 ? w.z : nan;
            v[4 * u + 3] = i < n4 ? w.w : nan;
        }
        f(v, [&](int e) { return 4 * (i0 + (e >> 2) * SF_NT) + (e & 3); });
    }
    for (int i0 = 4 * n4 + tid; i0 - tid < V; i0 += 16 * SF_NT) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int i = i0 + e * SF_NT;
            v[e] = i < V ? x[i] : nan;
        }
        f(v, [&](int e) { return i0 + e * SF_NT; });
    }
}

// Bin of a key: linear in the logit between the row's maximum and tau, so that keys of
// one bin follow each other.  A constant for all calls of a row.
struct SfBins {
    float M, scale;
    __device__ __forceinline__ SfBins(float M, float tau) : M(M), scale((float)SF_BINS / (M - tau)) {
        if (!(scale > 0.0f && scale < 1e30f)) scale = 0.0f;   // one logit, or an infinite range: one bin
    }
    __device__ __forceinline__ int operator()(uint32_t key) const {
        const float b = (M - sf_logit(key)) * scale;
        return b < (float)(SF_BINS - 1) ? max((int)b, 0) : SF_BINS - 1;   // (NaN: the last)
    }
};

// The smallest key such that elements of it and of smaller keys measure `need` (> 0) or
// more.  Elements of one key measure the same.
struct SfCut {
    uint32_t key;
    uint64_t below;                               // the measure of smaller keys
    uint64_t equal, one;                          // elements of the key, and what each measures
};
// false if all together measure less.  each(f): f(key, measure function) for the thread's
// elements.  Sums per bin, then the elements of the bin that passes `need`: by one wave
// if they are few, else digit by digit.
template <class E>
__device__ __forceinline__ bool sf_select(SfLds& s, const SfBins& bin, uint64_t need, SfCut& c, const E& each) {
    const int tid = threadIdx.x, lane = tid & 63;
    s.bins[tid] = 0;
    if (tid == 0) s.count = 0;
    __syncthreads();
    each([&](uint32_t k, auto measure) {
        __hip_atomic_fetch_add(&s.bins[bin(k)], (uint64_t)measure(), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    });
    __syncthreads();
    const uint64_t mine = s.bins[tid];
    uint64_t total;
    const uint64_t upto = sf_scan<uint64_t>(mine, s.wave, total);
    if (total < need) return false;               // uniform
    if (upto >= need && upto - mine < need) {
        s.found = tid;
        s.below = upto - mine;
    }
    __syncthreads();
    const int at = s.found;
    const uint64_t base = s.below;
    each([&](uint32_t k, auto measure) {
        if (bin(k) != at) return;
        const int i = __hip_atomic_fetch_add(&s.count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        if (i < SF_FEW) {
            s.few_key[i] = k;
            s.few[i] = (uint64_t)measure();
        }
    });
    __syncthreads();
    const int n = s.count;
    if (n <= SF_FEW) {
        if (tid < 64) {
            uint32_t k[SF_FEW / 64], lo = 0xffffffffu, hi = 0;
            uint64_t m[SF_FEW / 64];
#pragma unroll
            for (int e = 0; e < SF_FEW / 64; ++e) {
                const int i = 64 * e + lane;
                k[e] = i < n ? s.few_key[i] : 0xffffffffu;
                m[e] = i < n ? s.few[i] : 0;
                lo = min(lo, k[e]);
                hi = max(hi, i < n ? k[e] : 0u);
            }
            lo = ~wave_max_u32(~lo);
            hi = wave_max_u32(hi);
            const int ne = (n + 63) / 64;
            uint64_t b;
            const uint32_t t = sf_bisect(lo, hi, need - base, b, [&](uint32_t mid) {
                uint64_t v = 0;
#pragma unroll
                for (int e = 0; e < SF_FEW / 64; ++e)
                    if (e < ne) v += k[e] <= mid ? m[e] : 0;
                return wave_sum64(v);
            });
            uint64_t v = 0;
            uint32_t q = 0;
#pragma unroll
            for (int e = 0; e < SF_FEW / 64; ++e) {
                const bool eq = 64 * e + lane < n && k[e] == t;
                v += eq ? m[e] : 0;
                q += __builtin_popcountll(__builtin_amdgcn_ballot_w64(eq));
            }
            v = wave_sum64(v);
            if (lane == 0) {
                s.few_key[0] = t;
                s.few[0] = base + b;
                s.few[1] = q;
                s.few[2] = v / q;
            }
        }
        __syncthreads();
        c = {s.few_key[0], s.few[0], s.few[1], s.few[2]};
        __syncthreads();
        return true;
    }
    // many in one bin: equal or nearly equal logits
    uint32_t prefix = 0;
    uint64_t below = base;
    int shift = 24;
#pragma unroll 1
    for (int round = 0; round < 4; ++round, shift -= 8) {
        __syncthreads();
        if (tid < 256) s.bins[tid] = 0;
        __syncthreads();
        each([&](uint32_t k, auto measure) {
            if (bin(k) == at && (round == 0 || k >> (shift + 8) == prefix))
                __hip_atomic_fetch_add(&s.bins[k >> shift & 255], (uint64_t)measure(), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        });
        __syncthreads();
        const uint64_t b = tid < 256 ? s.bins[tid] : 0;
        const uint64_t up = below + sf_scan<uint64_t>(b, s.wave, total);
        if (up >= need && up - b < need) {
            s.found = tid;
            s.below = up - b;
        }
        __syncthreads();
        prefix = prefix << 8 | (uint32_t)s.found;
        below = s.below;
    }
    __syncthreads();
    uint64_t equal = 0, sum = 0;
    each([&](uint32_t k, auto measure) {
        if (k != prefix) return;
        ++equal;
        sum += (uint64_t)measure();
    });
    equal = sf_sum(equal, s.wave);
    sum = sf_sum(sum, s.wave);
    c = {prefix, below, equal, sum / equal};
    return true;
}

// The first element at which the sum of measures passes t (t below the sum of all), on
// every thread: the wave's sixteenth that holds it, then that one's, down to an
// element per thread.  measure(element, i).
template <class S, class M>
__device__ __forceinline__ int sf_first(SfLds& s, const S& e, uint64_t t, const M& measure) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int lo = 0, hi = e.n;
    uint64_t total;
#pragma unroll 1
    while (hi - lo > SF_NT) {
        const int part = (hi - lo + SF_NT - 1) / SF_NT * 64, a = lo + wave * part;
        uint64_t m = 0;
        sf_each(e, a + lane, min(a + part, hi), 64, [&](const typename S::Raw& x, int i) { m += measure(x, i); });
        const uint64_t upto = sf_scan<uint64_t>(m, s.wave, total);
        const uint64_t all = lane_of(upto, 63), before = lane_of(upto - m, 0);
        if (lane == 0 && all > t && before <= t) {
            s.found = wave;
            s.below = before;
        }
        __syncthreads();
        lo += min(s.found, SF_NT / 64 - 1) * part;
        hi = min(lo + part, hi);
        t -= s.below;
        __syncthreads();
    }
    const uint64_t m = lo + tid < hi ? measure(e.load(lo + tid), lo + tid) : 0;
    const uint64_t upto = sf_scan<uint64_t>(m, s.wave, total);
    if (upto > t && upto - m <= t) s.found = lo + tid;
    __syncthreads();
    const int at = s.found;
    __syncthreads();
    return min(max(at, 0), e.n - 1);              // an element even of rows that change meanwhile
}

// What remains of u: the sum that the drawn token's has to pass.
__device__ __forceinline__ uint64_t sf_draw(float u, uint64_t total) {
    return u > 0.0f ? min((uint64_t)(fmin((double)u, 1.0) * (double)total), total - 1) : 0;
}

// Selection and draw by the workgroup; all: the weight of every token of the row in units
// of 2^-42, where no top-k cuts it.
template <class S>
__device__ __forceinline__ void sf_choose(SfLds& s, const lgx_filter_args& a, const SfRow& r, const SfBins& bin, int row, double all,
                                          const S& e) {
    typedef typename S::Raw Raw;
    // kept: key < last, or key == last and place <= most
    uint32_t last = 0xffffffffu;
    int most = 0x7fffffff;
    auto kept = [&](const Raw& x, int i) {
        const uint32_t k = e.key(x);
        return e.valid(x) && (k < last || (k == last && i <= most));
    };
    auto each = [&](auto f) {
        sf_each(e, threadIdx.x, e.n, SF_NT, [&](const Raw& x, int i) {
            if (kept(x, i)) f(x, i);
        });
    };
    auto sum = [&](auto f) {
        uint64_t n = 0;
        each([&](const Raw& x, int) { n += f(x); });
        return sf_sum(n, s.wave);
    };
    // of the kept tokens those of smaller keys and the first n (>= 1) of the cut's
    auto keep = [&](const SfCut& c, uint64_t n) {
        if (c.key != last) most = 0x7fffffff;
        last = c.key;
        if (n < c.equal)
            most = sf_first(s, e, n - 1, [&](const Raw& x, int i) { return (uint64_t)(e.valid(x) && e.key(x) == last && i <= most); });
    };
    SfCut c;
    uint64_t total = 0;                           // weight of the kept tokens, once known
    // fewer tokens than top_k that count: all of them
    if (r.k && sf_select(s, bin, r.k, c, [&](auto f) { each([&](const Raw& x, int) { f(e.key(x), [] { return 1; }); }); }))
        keep(c, r.k - c.below);
    if (r.p < 1.0f) {
        // of the kept tokens those that reach the share, the first at least
        const double whole = r.k ? (double)sum([&](const Raw& x) { return e.weight(x); }) : all;
        const uint64_t need = max((uint64_t)ceil((double)r.p * whole), (uint64_t)1);
        if (sf_select(s, bin, need, c, [&](auto f) { each([&](const Raw& x, int) { f(e.key(x), [&] { return e.weight(x); }); }); })) {
            const uint64_t n = min((need - c.below + c.one - 1) / c.one, c.equal);
            keep(c, n);
            total = c.below + n * c.one;
        }
    }
    const uint64_t low = (uint64_t)ceil((double)r.mp * SF_ONE);
    auto weight = [&](const Raw& x) {
        const uint64_t w = e.weight(x);
        return w >= low ? w : 0;
    };
    if (total == 0 || low) total = sum([&](const Raw& x) { return weight(x); });
    const int at = sf_first(s, e, sf_draw(a.u[row], total), [&](const Raw& x, int i) { return kept(x, i) ? weight(x) : 0; });
    if (threadIdx.x == 0) {
        const Raw x = e.load(at);
        a.out[row] = e.index(x, at);
        if (a.prob) a.prob[row] = (float)((double)weight(x) / (double)total);
    }
}

// The same by one wave, for n <= 64 elements of the list, one per lane: each lane sums over
// those that come before its own in the order of (key, index).
__device__ __forceinline__ void sf_choose_lanes(const SfLds& s, const lgx_filter_args& a, const SfRow& r, int row, double all, int n) {
    const int lane = threadIdx.x & 63;
    bool on = lane < n;
    const uint32_t key = on ? s.key[lane] : 0xffffffffu;
    const uint64_t wi = on ? s.wi[lane] : 0, w = wi >> 20;
    if (r.k || r.p < 1.0f) {
        uint64_t before = 0;                      // weight of the elements ahead, and their number << 52
        const uint64_t wn = w | 1ull << 52;
        for (int j = 0; j < n; ++j) {             // 64 weights of 2^42 stay below 2^49
            const uint32_t kj = (uint32_t)__builtin_amdgcn_readlane((int)key, j);
            const uint64_t wj = lane_of(wn, j);
            before += kj < key || (kj == key && j < lane) ? wj : 0;
        }
        if (r.k) on = on && (int)(before >> 52) < r.k;
        if (r.p < 1.0f) {
            const double whole = r.k ? (double)wave_sum64(on ? w : 0) : all;
            const uint64_t need = max((uint64_t)ceil((double)r.p * whole), (uint64_t)1);
            on = on && (before & ((1ull << 52) - 1)) < need;
        }
    }
    on = on && w >= (uint64_t)ceil((double)r.mp * SF_ONE);
    const uint64_t mine = on ? w : 0, upto = wave_scan64(mine), total = lane_of(upto, 63), t = sf_draw(a.u[row], total);
    if (upto > t && upto - mine <= t) {
        a.out[row] = (int)(wi & 0xfffff);
        if (a.prob) a.prob[row] = (float)((double)w / (double)total);
    }
}

// The same by the workgroup, for n <= 128 elements: the weight and the number of those ahead
// of each, an eighth of them per pair of waves, then two elements per lane of one wave.
__device__ __forceinline__ void sf_choose_pairs(SfLds& s, const lgx_filter_args& a, const SfRow& r, int row, double all, int n) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (r.k || r.p < 1.0f) {
        const int i = 64 * (wave & 1) + lane;
        const uint32_t key = i < n ? s.key[i] : 0u;
        uint64_t before = 0;                      // number << 52: 128 weights of 2^42 stay below
#pragma unroll 4
        for (int j = wave >> 1; j < n; j += SF_NT / 128) {
            const uint32_t kj = s.key[j];
            const uint64_t wj = s.wi[j] >> 20 | 1ull << 52;
            before += kj < key || (kj == key && j < i) ? wj : 0;
        }
        s.bins[128 * (wave >> 1) + i] = before;
        __syncthreads();
    }
    if (wave) return;
    uint64_t w[2], before[2] = {0, 0};
    bool on[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int i = 2 * lane + e;
        on[e] = i < n;
        w[e] = on[e] ? s.wi[i] >> 20 : 0;
        if (r.k || r.p < 1.0f) {
#pragma unroll
            for (int q = 0; q < SF_NT / 128; ++q) before[e] += s.bins[128 * q + i];
        }
    }
    if (r.k) {
#pragma unroll
        for (int e = 0; e < 2; ++e) on[e] = on[e] && (int)(before[e] >> 52) < r.k;
    }
    if (r.p < 1.0f) {
        const double whole = r.k ? (double)wave_sum64((on[0] ? w[0] : 0) + (on[1] ? w[1] : 0)) : all;
        const uint64_t need = max((uint64_t)ceil((double)r.p * whole), (uint64_t)1);
#pragma unroll
        for (int e = 0; e < 2; ++e) on[e] = on[e] && (before[e] & ((1ull << 52) - 1)) < need;
    }
    const uint64_t low = (uint64_t)ceil((double)r.mp * SF_ONE);
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (!on[e] || w[e] < low) w[e] = 0;
    const uint64_t upto = wave_scan64(w[0] + w[1]), total = lane_of(upto, 63), t = sf_draw(a.u[row], total);
    const uint64_t from = upto - w[0] - w[1];
    if (upto > t && from <= t) {
        const int e = from + w[0] > t ? 0 : 1;
        a.out[row] = (int)(s.wi[2 * lane + e] & 0xfffff);
        if (a.prob) a.prob[row] = (float)((double)(e ? w[1] : w[0]) / (double)total);
    }
}

// The same for n <= SF_FEW: lane l holds elements l ne .. , so that sums over lanes go by index.
// Where top-k leaves 64 at most, they go on as above.
__device__ __forceinline__ void sf_choose_wave(SfLds& s, const lgx_filter_args& a, SfRow r, int row, double all, int n) {
    constexpr int E = SF_FEW / 64;
    const int lane = threadIdx.x & 63, ne = (n + 63) / 64;
    uint32_t k[E], lo = 0xffffffffu, hi = 0;
    uint64_t wi[E];
    bool on[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int i = lane * ne + e;
        on[e] = e < ne && i < n;
        k[e] = on[e] ? s.key[i] : 0xffffffffu;
        wi[e] = on[e] ? s.wi[i] : 0;
        lo = min(lo, k[e]);
        hi = max(hi, on[e] ? k[e] : 0u);
    }
    lo = ~wave_max_u32(~lo);
    hi = wave_max_u32(hi);
    // of the kept elements those of keys below t, and the first m of key t
    auto cut = [&](uint32_t t, uint64_t m) {
        uint32_t c = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) c += on[e] && k[e] == t;
        uint32_t before = (uint32_t)wave_scan((int)c) - c;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const bool eq = on[e] && k[e] == t;
            on[e] = on[e] && (k[e] < t || (eq && before < m));
            before += eq;
        }
        hi = t;
    };
    uint64_t below;
    if (r.k && r.k < n) {
        const uint32_t t = sf_bisect(lo, hi, r.k, below, [&](uint32_t mid) {
            uint32_t c = 0;
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (e < ne) c += __builtin_popcountll(__builtin_amdgcn_ballot_w64(on[e] && k[e] <= mid));
            return (uint64_t)c;
        });
        cut(t, r.k - below);
        if (r.k <= 64) {
            uint32_t c = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) c += on[e];
            uint32_t to = (uint32_t)wave_scan((int)c) - c;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (on[e]) {
                    s.key[to] = k[e];
                    s.wi[to] = wi[e];
                }
                to += on[e];
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the wave reads what its lanes wrote
            sf_choose_lanes(s, a, r, row, all, r.k);
            return;
        }
    }
    auto sum = [&](auto f) {
        uint64_t v = 0;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (e < ne) v += on[e] && f(e) ? wi[e] >> 20 : 0;
        return wave_sum64(v);
    };
    if (r.p < 1.0f) {
        const uint64_t have = sum([](int) { return true; });
        const uint64_t need = max((uint64_t)ceil((double)r.p * (r.k ? (double)have : all)), (uint64_t)1);
        if (need <= have) {
            const uint32_t t = sf_bisect(lo, hi, need, below, [&](uint32_t mid) { return sum([&](int e) { return k[e] <= mid; }); });
            uint32_t c = 0;
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (e < ne) c += __builtin_popcountll(__builtin_amdgcn_ballot_w64(on[e] && k[e] == t));
            const uint64_t w = sum([&](int e) { return k[e] == t; }) / c;   // one weight for one logit
            cut(t, (need - below + w - 1) / w);
        }
    }
    const uint64_t low = (uint64_t)ceil((double)r.mp * SF_ONE);
    uint64_t mine = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        on[e] = on[e] && wi[e] >> 20 >= low;
        mine += on[e] ? wi[e] >> 20 : 0;
    }
    const uint64_t upto = wave_scan64(mine), total = lane_of(upto, 63), t = sf_draw(a.u[row], total);
    if (upto > t && upto - mine <= t) {
        uint64_t c = upto - mine;
        bool done = false;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            c += on[e] ? wi[e] >> 20 : 0;
            if (!done && c > t) {
                done = true;
                a.out[row] = (int)(wi[e] & 0xfffff);
                if (a.prob) a.prob[row] = (float)((double)(wi[e] >> 20) / (double)total);
            }
        }
    }
}

extern "C" __global__ __launch_bounds__(SF_NT) void lgx_k_filter_pick(const lgx_filter_args a) {
    __shared__ SfLds s;
    const int tid = threadIdx.x, lane = tid & 63, row = blockIdx.x, V = a.vocab;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const SfRow r = sf_row(a, row);
    const float* x = a.logits + (int64_t)row * a.ld;
    const float* smax = a.smax + (int64_t)row * a.nslices;
    const float* cmax = a.cmax + (int64_t)row * a.nslices * 64;
    const int nruns = (V + LGX_SF_CHUNK - 1) / LGX_SF_CHUNK;
    const float ninf = -__builtin_inff();
    // the runs' maxima, a sixteenth of them per wave
    constexpr int CM = LGX_SF_VOCAB / LGX_SF_CHUNK / SF_NT;
    const int rw = (nruns + SF_NT - 1) / SF_NT;   // per lane
    const int c0 = wave * 64 * rw + lane;
    float cm[CM];
#pragma unroll
    for (int j = 0; j < CM; ++j) cm[j] = j < rw && c0 + 64 * j < nruns ? cmax[c0 + 64 * j] : __builtin_nanf("");
    // (the sums are there only where they are needed)
    const double part = tid < a.nslices ? a.sum[(int64_t)row * a.nslices + tid] : 0.0;
    const float part_max = tid < a.nslices ? smax[tid] : ninf;
    // the row's maximum: at most 128 slices
    float M = ninf;
    for (int i = lane; i < a.nslices; i += 64) M = fmaxf(M, smax[i]);
    M = wave_max(M);
    sf_roots(s.roots);
    if (M == ninf) {                              // uniform: no token at all
        if (tid == 0) {
            a.out[row] = 0;
            if (a.prob) a.prob[row] = 0.0f;
        }
        return;
    }
    if (r.greedy) {
        if (tid == 0) s.found = 0x7fffffff;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < CM; ++j)
            if (cm[j] == M) __hip_atomic_fetch_min(&s.found, c0 + 64 * j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        __syncthreads();
        if (wave) return;
        const int i = s.found * LGX_SF_CHUNK + lane;
        const uint64_t hit = __builtin_amdgcn_ballot_w64(i < V && x[min(i, V - 1)] == M);
        if (lane == 0) {
            a.out[row] = s.found * LGX_SF_CHUNK + __builtin_ctzll(hit);
            if (a.prob) a.prob[row] = 1.0f;
        }
        return;
    }
    __syncthreads();                              // the table
    double S = 0.0;                               // of all weights, by M
    if (r.sums()) {
        const double mine = tid < a.nslices ? part * sf_weight(part_max, M, r.inv, s.roots) : 0.0;
        const double upto = sf_scan<double>(mine, s.dwave, S);
        if (r.plain()) {
            // the slice that the draw falls into: the last with a weight that starts at
            // or before it; then the token in the slice
            const double t = fmin(fmax((double)a.u[row], 0.0), 1.0) * S;
            if (tid == 0) s.found = 0;
            __syncthreads();
            if (mine > 0.0 && upto - mine <= t) __hip_atomic_fetch_max(&s.found, tid, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            __syncthreads();
            const int sl = s.found;
            if (tid == sl) s.dwave[0] = t - (upto - mine);
            __syncthreads();
            const double in = s.dwave[0];
            __syncthreads();
            const int e0 = sl * LGX_SF_SLICE + 4 * tid;
            double w[4], c = 0.0, all;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[i] = e0 + i < V ? sf_weight(x[min(e0 + i, V - 1)], M, r.inv, s.roots) : 0.0;
                c += w[i];
            }
            double at = sf_scan<double>(c, s.dwave, all) - c;
            if (tid == 0) s.found = 0;
            __syncthreads();
            int best = -1;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (w[i] > 0.0 && at <= in) best = 4 * tid + i;
                at += w[i];
            }
            if (best >= 0) __hip_atomic_fetch_max(&s.found, best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            __syncthreads();
            if (best >= 0 && s.found == best) {
                const double wb = (best & 3) == 0 ? w[0] : (best & 3) == 1 ? w[1] : (best & 3) == 2 ? w[2] : w[3];
                a.out[row] = sl * LGX_SF_SLICE + best;
                if (a.prob) a.prob[row] = (float)(wb / S);
            }
            return;
        }
    }
    // tau: tokens below it are not kept.  A weight under 2^-43 counts as nothing (e^-29.9);
    // the tokens under (1 - p) / V of the whole are less than 1 - p of it together; the k-th
    // largest of the runs' maxima is no larger than the k-th largest token.  The margins
    // are far above the rounding of the logarithms.  (Top-p of the top k weighs all k.)
    const float T = sf_temperature(a, row);
    float tau = M - 30.0f * T;
    if (r.mp > 0.0f && !(r.k && r.p < 1.0f)) tau = fmaxf(tau, M + T * (logf(r.mp) - 0.001f));
    if (r.p < 1.0f && !r.k) tau = fmaxf(tau, M + T * (logf((1.0f - r.p) / (float)V) + logf((float)S) - 0.001f));
    tau -= fmaxf(fabsf(M), fabsf(tau)) * 1e-6f;
    if (!(tau == tau)) tau = M == __builtin_inff() ? M : ninf;
    // Top-p alone: that bound is loose where a few tokens weigh nearly all.  The tokens from
    // the 256th largest run's maximum on are tried first: if they reach the share, they
    // are enough.
    const bool guess = !r.k && r.p < 1.0f && nruns > 2 * SF_GUESS;
    const int most = r.k ? r.k : SF_GUESS;
    float high = tau;
    if (guess || (r.k && r.k <= nruns)) {
        // a bin of the runs' maxima by which so many of them are reached
        s.bins[tid] = 0;
        __syncthreads();
        const SfBins bin(M, fmaxf(tau, -3e38f));
#pragma unroll
        for (int j = 0; j < CM; ++j)
            if (cm[j] >= tau)
                __hip_atomic_fetch_add((uint32_t*)&s.bins[bin(sf_key(cm[j]))], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        __syncthreads();
        const uint64_t mine = (uint32_t)s.bins[tid];
        uint64_t total;
        const uint64_t upto = sf_scan<uint64_t>(mine, s.wave, total);
        if (total >= (uint64_t)most) {            // uniform
            if (upto >= (uint64_t)most && upto - mine < (uint64_t)most) s.found = tid;
            __syncthreads();
            // no run of that bin or an earlier one is below the bin's end (with its roundings)
            const float end = M - (float)(s.found + 1) / bin.scale * 1.000001f;
            if (bin.scale > 0.0f) high = fmaxf(tau, end - fmaxf(fabsf(M), fabsf(end)) * 1e-6f);
        }
    }
    const double all = S * SF_ONE;
#pragma unroll 1
    for (bool first = guess && high > tau;; first = false) {   // uniform
        if (r.k || first) {
            const float t = tau;
            tau = high;
            high = t;
        }
        // the runs that reach tau, in order
        int mine = 0;
#pragma unroll
        for (int j = 0; j < CM; ++j) mine += __builtin_popcountll(__builtin_amdgcn_ballot_w64(cm[j] >= tau));
        __syncthreads();                          // bins and counts are read
        uint64_t runs;
        int to = (int)sf_waves<uint64_t>(mine, s.wave, runs);
        const int nr = (int)runs;
#pragma unroll
        for (int j = 0; j < CM; ++j) {
            const uint64_t hit = __builtin_amdgcn_ballot_w64(cm[j] >= tau);
            const int q = to + __builtin_popcountll(hit & ((1ull << lane) - 1));
            if (cm[j] >= tau && q < SF_LIST) s.runs[q] = (uint16_t)(c0 + 64 * j);
            to += __builtin_popcountll(hit);
        }
        __syncthreads();
        int n = SF_LIST + 1;
        uint64_t weighs = 0;
        // (runs have a token each at least; one workgroup takes 1 us for 64 of them)
        if (nr <= (a.slots && !r.k ? SF_LIST / 4 : SF_LIST)) {
            // their tokens that reach it, in order: a sixteenth of the runs per wave
            const int per = (nr + SF_NT / 64 - 1) / (SF_NT / 64), q0 = min(wave * per, nr), q1 = min(q0 + per, nr);
            float v[4];
            int t[4];
            auto load = [&](int q) {              // four runs in flight
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    t[u] = s.runs[min(q + u, q1 - 1)] * LGX_SF_CHUNK + lane;
                    v[u] = t[u] < V && q + u < q1 ? x[t[u]] : __builtin_nanf("");
                }
            };
            int c = 0;
            for (int q = q0; q < q1; q += 4) {
                load(q);
#pragma unroll
                for (int u = 0; u < 4; ++u) c += __builtin_popcountll(__builtin_amdgcn_ballot_w64(v[u] >= tau));
            }
            uint64_t tokens;
            int at = (int)sf_waves<uint64_t>(c, s.wave, tokens);
            n = (int)tokens;
            if (n <= SF_LIST) {                   // uniform
                for (int q = q0; q < q1; q += 4) {
                    if (q1 - q0 > 4) load(q);     // else still there
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const uint64_t hit = __builtin_amdgcn_ballot_w64(v[u] >= tau);
                        const int i = at + __builtin_popcountll(hit & ((1ull << lane) - 1));
                        if (v[u] >= tau) {
                            s.key[i] = sf_key(v[u]);
                            s.wi[i] = (uint64_t)t[u];
                        }
                        at += __builtin_popcountll(hit);
                    }
                }
                __syncthreads();
                // their weights, by as many lanes as there are tokens (a run has few)
                for (int i = tid; i < n; i += SF_NT) {
                    const uint64_t w = sf_weight_units(sf_logit(s.key[i]), M, r.inv, s.roots);
                    weighs += w;
                    s.wi[i] |= w << 20;
                }
                __syncthreads();
            }
        }
        if (first) {                              // uniform
            if (n > SF_LIST || (double)sf_sum(weighs, s.wave) < ceil((double)r.p * all)) {
                tau = high;
                continue;
            }
        }
        const SfBins bin(M, fmaxf(tau, -3e38f));
        if (n <= 128) {
            sf_choose_pairs(s, a, r, row, all, n);
        } else if (n <= SF_FEW) {
            if (wave == 0) sf_choose_wave(s, a, r, row, all, n);
        } else if (n <= SF_LIST) {
            sf_choose(s, a, r, bin, row, all, SfInLds{s, n});
        } else if (a.slots && !r.k && tau > -3e38f && M < __builtin_inff()) {
            // more than LDS holds: the row for lgx_k_filter_wide
            if (tid == 0) {
                const int i = atomicAdd(a.wide_n, 1);
                a.wide_row[i] = row;
                a.wide_tau[i] = tau;
                a.wide_all[i] = all;
                if (i < a.slots) a.wide_done[i] = 0;
            }
        } else {
            // the row itself
            sf_choose(s, a, r, bin, row, all, SfInRow{x, V, tau, M, r.inv, s.roots});
        }
        return;
    }
}

// Bins of the wide rows' weights, slice by slice: workgroup (slice, rows y, y + gridDim.y ..
// of the list).
struct SfSliceBins {
    float M, scale;
    __device__ __forceinline__ SfSliceBins(float M, float tau) : M(M), scale((float)LGX_SF_BINS / (M - tau)) {
        if (!(scale > 0.0f && scale < 1e30f)) scale = 0.0f;
    }
    __device__ __forceinline__ int operator()(float l) const {
        const float b = (M - l) * scale;
        return b < (float)(LGX_SF_BINS - 1) ? (int)b : LGX_SF_BINS - 1;
    }
};
__device__ __forceinline__ float sf_row_max(const lgx_filter_args& a, int row) {
    float M = -__builtin_inff();
    for (int i = threadIdx.x & 63; i < a.nslices; i += 64) M = fmaxf(M, a.smax[(int64_t)row * a.nslices + i]);
    return wave_max(M);
}
// What other workgroups of this launch have written, past the caches that are not theirs
// too: loads and stores of the whole device's scope.  (Fences of that scope in their place
// would write back and drop whole caches.)
__device__ __forceinline__ uint64_t sf_shared(const uint64_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// The choice in wide row w, from the bins of its slices: the bin in which top-p ends, the
// tokens in it, then what is kept of each slice, the slice that the draw falls into and
// the token in it.
__device__ __forceinline__ void sf_choose_wide(SfLds& s, const lgx_filter_args& a, const SfRow& r, const SfSliceBins& bin, int w, int row,
                                               float tau, float M) {
    const int tid = threadIdx.x, lane = tid & 63, V = a.vocab;
    const double all = a.wide_all[w];
    const float* x = a.logits + (int64_t)row * a.ld;
    const uint64_t* hist = a.hist + (int64_t)w * a.nslices * LGX_SF_BINS;
    // weight per bin: four threads a bin, each a quarter of the slices
    uint64_t mine = 0, total;
    for (int i0 = tid >> 8; i0 < a.nslices; i0 += 12 * (SF_NT / LGX_SF_BINS)) {
        uint64_t u[12];                       // in flight together
#pragma unroll
        for (int q = 0; q < 12; ++q) u[q] = sf_shared(hist + min(i0 + q * (SF_NT / LGX_SF_BINS), a.nslices - 1) * LGX_SF_BINS + (tid & 255));
#pragma unroll
        for (int q = 0; q < 12; ++q) mine += i0 + q * (SF_NT / LGX_SF_BINS) < a.nslices ? u[q] : 0;
    }
    s.bins[tid] = mine;
    if (tid == 0) s.count = 0;
    __syncthreads();
    mine = tid < LGX_SF_BINS ? s.bins[tid] + s.bins[tid + 256] + s.bins[tid + 512] + s.bins[tid + 768] : 0;
    const uint64_t upto = sf_scan<uint64_t>(mine, s.wave, total);
    const uint64_t need = max((uint64_t)ceil((double)r.p * all), (uint64_t)1), low = (uint64_t)ceil((double)r.mp * SF_ONE);
    // of bins first .. end not all tokens are known to be kept or not: those are listed
    int first = LGX_SF_BINS, end = LGX_SF_BINS - 1;
    if (r.mp > 0.0f) first = bin(fminf(M + sf_temperature(a, row) * (logf(r.mp) + 0.001f), M));
    uint64_t base = 0;                        // weight of the bins below `end`
    bool few = true;
    const bool cut = r.p < 1.0f && need <= total;
    if (cut) {                                // uniform
        if (upto >= need && upto - mine < need) {
            s.found = tid;
            s.below = upto - mine;
        }
        __syncthreads();
        end = s.found;
        base = s.below;
        first = min(first, end);
    }
    int n = 0;
    if (first < LGX_SF_BINS) {                // uniform
        // counted, then written from one place per wave; weights afterwards, by as many lanes
        // as there are tokens
        sf_row_each(x, V, a.vec, [&](float (&v)[16], auto index) __attribute__((always_inline)) {
            int c = 0;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int b = bin(v[e]);
                const bool on = v[e] >= tau && b >= first && b <= end;
                v[e] = on ? v[e] : __builtin_nanf("");
                c += on;
            }
            int to = wave_scan(c);
            const int all_lanes = __builtin_amdgcn_readlane(to, 63);
            if (all_lanes == 0) return;           // uniform
            int from = 0;
            if (lane == 0) from = __hip_atomic_fetch_add(&s.count, all_lanes, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            to += __builtin_amdgcn_readlane(from, 0) - c;
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (v[e] == v[e]) {
                    if (to < SF_LIST) {
                        s.key[to] = sf_key(v[e]);
                        s.wi[to] = (uint64_t)index(e);
                    }
                    ++to;
                }
        });
        __syncthreads();
        n = s.count;
        for (int i = tid; i < min(n, SF_LIST); i += SF_NT)
            s.wi[i] |= sf_weight_units(sf_logit(s.key[i]), M, r.inv, s.roots) << 20;
        __syncthreads();
        few = n <= SF_LIST;
    }
    if (!few) {                               // equal or nearly equal logits
        sf_choose(s, a, r, SfBins(M, tau), row, all, SfInRow{x, V, tau, M, r.inv, s.roots});
        return;
    }
    uint32_t last = 0xffffffffu;              // kept: key < last, or key == last and index <= most
    int most = 0x7fffffff;
    if (cut) {
        auto ends = [&](int i) { return bin(sf_logit(s.key[i])) == end; };
        SfCut c;
        const float wide = bin.scale > 0.0f ? 1.0f / bin.scale : 0.0f;
        const SfBins sub(fminf(M, M - (float)end * wide + 1e-6f * fabsf(M)), fmaxf(tau, M - (float)(end + 1) * wide));
        sf_select(s, sub, need - base, c, [&](auto f) {
            for (int i = tid; i < n; i += SF_NT)
                if (ends(i)) f(s.key[i], [&] { return s.wi[i] >> 20; });
        });
        last = c.key;
        const uint64_t m = (need - base - c.below + c.one - 1) / c.one;
        if (m < c.equal) {                    // the m-th lowest index among the equal ones
            int lo = 0, hi = V - 1;
            while (lo < hi) {                 // uniform
                const int mid = (lo + hi) / 2;
                uint64_t q = 0;
                for (int i = tid; i < n; i += SF_NT) q += s.key[i] == last && (int)(s.wi[i] & 0xfffff) <= mid;
                if (sf_sum(q, s.wave) >= m) hi = mid;
                else lo = mid + 1;
            }
            most = lo;
        }
    }
    // what is kept of each slice: its bins below `first`, and tokens of the list
    auto keeps = [&](uint32_t k, int i, uint64_t u) { return (k < last || (k == last && i <= most)) && u >= low ? u : 0; };
    __syncthreads();
    if (tid < LGX_SF_VOCAB / LGX_SF_SLICE) s.few[tid] = 0;
    __syncthreads();
    for (int i0 = tid >> 6; i0 < a.nslices; i0 += 3 * (SF_NT / 64)) {
        uint64_t u[3][LGX_SF_BINS / 64];
#pragma unroll
        for (int q = 0; q < 3; ++q)
#pragma unroll
            for (int b = 0; b < LGX_SF_BINS / 64; ++b)
                u[q][b] = sf_shared(hist + min(i0 + q * (SF_NT / 64), a.nslices - 1) * LGX_SF_BINS + 64 * b + lane);
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            const int i = i0 + q * (SF_NT / 64);
            if (i >= a.nslices) break;        // uniform
            uint64_t m = 0;
#pragma unroll
            for (int b = 0; b < LGX_SF_BINS / 64; ++b) m += 64 * b + lane < first ? u[q][b] : 0;
            m = wave_sum64(m);
            if (lane == 0) __hip_atomic_fetch_add(&s.few[i], m, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        }
    }
    for (int i = tid; i < n; i += SF_NT) {
        const uint64_t wi = s.wi[i];
        const int at = (int)(wi & 0xfffff);
        __hip_atomic_fetch_add(&s.few[at / LGX_SF_SLICE], keeps(s.key[i], at, wi >> 20), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
    auto kept = [&](float v, int i) { return v >= tau ? keeps(sf_key(v), i, sf_weight_units(v, M, r.inv, s.roots)) : 0; };
    __syncthreads();
    mine = tid < a.nslices ? s.few[tid] : 0;
    const uint64_t to = sf_scan<uint64_t>(mine, s.wave, total), t = sf_draw(a.u[row], total);
    if (to > t && to - mine <= t) {
        s.found = tid;
        s.below = to - mine;
    }
    __syncthreads();
    const int sl = s.found;
    const uint64_t in = t - s.below;
    const int i0 = sl * LGX_SF_SLICE + 4 * tid;
    uint64_t u[4], c = 0, sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        u[i] = i0 + i < V ? kept(x[min(i0 + i, V - 1)], i0 + i) : 0;
        c += u[i];
    }
    uint64_t at = sf_scan<uint64_t>(c, s.wave, sum) - c;
    bool done = at > in || at + c <= in;      // not this thread's
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        at += u[i];
        if (!done && at > in) {
            done = true;
            a.out[row] = i0 + i;
            if (a.prob) a.prob[row] = (float)((double)u[i] / (double)total);
        }
    }
}

// The wide rows.  Each workgroup takes a run of their (row, slice)s: bins of the slice's
// weights, stored; the one that brings a row's last bins goes on with the row.  None waits
// for another.  Rows without room for bins come after, one per workgroup.
extern "C" __global__ __launch_bounds__(SF_NT) void lgx_k_filter_wide(const lgx_filter_args a) {
    __shared__ SfLds s;
    __shared__ int last;
    const int tid = threadIdx.x, n_all = *a.wide_n, n = min(n_all, a.slots), items = n * a.nslices;
    const int per = (int)((unsigned)(items + gridDim.x - 1) / gridDim.x), at1 = min((int)blockIdx.x * per + per, items);
    if (n_all == 0) return;
    sf_roots(s.roots);
    for (int at = blockIdx.x * per; at < at1;) {  // uniform
        const int w = at / a.nslices, sl0 = at - w * a.nslices, sl1 = min(a.nslices, sl0 + at1 - at);
        const int row = a.wide_row[w];
        const float tau = a.wide_tau[w], M = sf_row_max(a, row);
        const SfRow r = sf_row(a, row);
        const float* x = a.logits + (int64_t)row * a.ld;
        const SfSliceBins bin(M, tau);
        for (int sl = sl0; sl < sl1; ++sl) {
            float v[LGX_SF_SLICE / SF_NT];
#pragma unroll
            for (int i = 0; i < LGX_SF_SLICE / SF_NT; ++i) {
                const int e = sl * LGX_SF_SLICE + SF_NT * i + tid;
                v[i] = e < a.vocab ? x[e] : __builtin_nanf("");
            }
            __syncthreads();                      // what was in LDS is read
            if (tid < LGX_SF_BINS) s.bins[tid] = 0;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < LGX_SF_SLICE / SF_NT; ++i)
                if (v[i] >= tau)
                    __hip_atomic_fetch_add(&s.bins[bin(v[i])], sf_weight_units(v[i], M, r.inv, s.roots), __ATOMIC_RELAXED,
                                           __HIP_MEMORY_SCOPE_WORKGROUP);
            __syncthreads();
            if (tid < LGX_SF_BINS)
                __hip_atomic_store(a.hist + ((int64_t)w * a.nslices + sl) * LGX_SF_BINS + tid, s.bins[tid], __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_AGENT);
        }
        at += sl1 - sl0;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // each wave's bins have reached memory
        __syncthreads();
        if (tid == 0)
            last = __hip_atomic_fetch_add(a.wide_done + w, sl1 - sl0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + sl1 - sl0 == a.nslices;
        __syncthreads();
        if (last) sf_choose_wide(s, a, r, bin, w, row, tau, M);   // uniform
    }
    for (int w = n + blockIdx.x; w < n_all; w += gridDim.x) {   // uniform
        const int row = a.wide_row[w];
        const float tau = a.wide_tau[w], M = sf_row_max(a, row);
        const SfRow r = sf_row(a, row);
        __syncthreads();
        sf_choose(s, a, r, SfBins(M, tau), row, a.wide_all[w], SfInRow{a.logits + (int64_t)row * a.ld, a.vocab, tau, M, r.inv, s.roots});
    }
}
