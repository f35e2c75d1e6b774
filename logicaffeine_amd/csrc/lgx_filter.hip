// lgx_filter.hip -- a token for each row of logits by temperature, top-k, top-p and
// min-p, with a given random number per row.
#include "lgx_device.h"

// ---------------------------------------------------------------------------
// Definition: lgx_sample_filtered in lgx.h.  The weights of a row's tokens are w =
// exp((l - M) / T), M the row's largest logit; with the tokens in order of (logit
// descending, index ascending) every filter keeps a prefix, and the draw goes over the
// kept tokens in order of index.
//
// Two launches.  The scan reads every logit once: the largest of each 64 (cmax), the
// largest of each 4096 and the sum of their weights.  The pick, a workgroup per row,
// derives from them a logit tau below which no token can be kept, reads again only the
// runs of 64 whose largest reaches it, and selects among those tokens, in LDS; a row
// with more of them than fit there is gone over in memory.  A row without filters needs
// the sums and one run of 4096.
//
// Sums decide between tokens, so they are exact or nearly: the weights that a
// selection adds up are whole multiples of 2^-42 in 64-bit integers, whose sums
// do not depend on any order; the scan's are binary64.  exp is computed in binary64.
// ---------------------------------------------------------------------------
#define SF_ONE 0x1p42                             // 2^20 weights stay below 2^63
#define SF_LIST 4096                              // tokens kept in LDS

// e^x for x <= 0: Cody-Waite reduction by ln 2 in two parts, then the Taylor polynomial
// of degree 11 on |r| <= 0.347 (the term after it is under 7e-15).
__device__ __forceinline__ double sf_exp(double x) {
    const double n = rint(x * 1.4426950408889634074);
    double r = fma(-n, 0x1.62e42fefap-1, x);
    r = fma(-n, 0x1.cf79abc9e3b39p-40, r);
    double p = 1.0 / 39916800.0;
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return x > -700.0 ? ldexp(p, (int)n) : 0.0;
}
// Weight of logit l by the maximum M; 0 for NaN and -inf, 1 for the maximum, whatever it is.
__device__ __forceinline__ double sf_weight(float l, float M, double inv) {
    const double x = ((double)l - (double)M) * inv;
    return l == M ? 1.0 : l > -__builtin_inff() && l < M ? sf_exp(x) : 0.0;
}

struct SfRow {
    double inv;                                   // 1 / T
    float p, mp;                                  // top_p (1: none), min_p (0: none)
    int k;                                        // top_k (0: none)
    bool greedy;
    __device__ __forceinline__ bool plain() const { return !k && p >= 1.0f && mp <= 0.0f; }
    // whether the sum of all weights is needed
    __device__ __forceinline__ bool sums() const { return !greedy && !k && (p < 1.0f || mp <= 0.0f); }
};
__device__ __forceinline__ SfRow sf_row(const lgx_filter_args& a, int row) {
    SfRow r;
    const float T = a.temperature ? a.temperature[row] : 1.0f;
    r.greedy = !(T > 0.0f);
    r.inv = 1.0 / (double)T;
    const int k = a.top_k ? a.top_k[row] : 0;
    r.k = k > 0 && k < a.vocab ? k : 0;
    const float p = a.top_p ? a.top_p[row] : 1.0f, mp = a.min_p ? a.min_p[row] : 0.0f;
    r.p = p < 1.0f ? fmaxf(p, 0.0f) : 1.0f;       // NaN: none
    r.mp = mp > 0.0f ? fminf(mp, 1.0f) : 0.0f;
    return r;
}

// Workgroup (4096 logits, row): thread t holds 4 (256 i + t) .. + 3 of them.
extern "C" __global__ __launch_bounds__(256) void lgx_k_filter_scan(const lgx_filter_args a) {
    __shared__ float mx_s[4];
    __shared__ double sum_s[4];
    const int tid = threadIdx.x, sl = blockIdx.x, row = blockIdx.y;
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
        for (int c = 0; c < 4; ++c) s += sf_weight(v[i][c], M, r.inv);
#pragma unroll
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d, 64);
    if ((tid & 63) == 0) sum_s[tid >> 6] = s;
    __syncthreads();
    if (tid == 0) a.sum[(int64_t)row * a.nslices + sl] = sum_s[0] + sum_s[1] + (sum_s[2] + sum_s[3]);
}

// Order of logits as unsigned numbers: ascending keys are descending logits, -0 is 0.
__device__ __forceinline__ uint32_t sf_key(float l) {
    const uint32_t u = __float_as_uint(l + 0.0f);
    return u & 0x80000000u ? u : ~(u | 0x80000000u);
}

#define SF_NT 1024
struct SfLds {
    uint64_t bins[2048];                          // of a selection; before it, runs of 64 and the places of their tokens
    uint64_t wi[SF_LIST];                         // weight << 20 | index
    uint32_t key[SF_LIST];
    uint64_t wave[SF_NT / 64];
    double dwave[SF_NT / 64];
    uint64_t below;
    int found;
};
static_assert(sizeof(SfLds) <= 81920, "two workgroups per compute unit");
static_assert(LGX_SF_VOCAB <= 1 << 20, "an index has 20 bits beside its weight");

// Inclusive sums over the workgroup's threads.
template <class V>
__device__ __forceinline__ V sf_scan(V v, V* waves, V& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const V o = __shfl_up(v, d, 64);
        v += lane >= d ? o : V(0);
    }
    if (lane == 63) waves[wave] = v;
    __syncthreads();
    V before = 0;
    total = 0;
    for (int w = 0; w < SF_NT / 64; ++w) {
        before += w < wave ? waves[w] : V(0);
        total += waves[w];
    }
    __syncthreads();
    return before + v;
}

// The smallest key whose elements and those of smaller keys measure `need` (> 0) or more,
// found digit by digit with sums per digit; below: the measure of smaller keys; false
// if all together measure less.  each(f): f(key, measure function) for the thread's
// elements.
template <class E>
__device__ __forceinline__ bool sf_select(SfLds& s, uint64_t need, uint32_t& key, uint64_t& below, const E& each) {
    const int tid = threadIdx.x;
    uint32_t prefix = 0;
    below = 0;
    int shift = 21;
#pragma unroll 1
    for (int round = 0; round < 3; ++round) {
        const int bits = round < 2 ? 11 : 10;
        s.bins[tid] = 0;
        s.bins[tid + SF_NT] = 0;
        __syncthreads();
        each([&](uint32_t k, auto measure) {
            if (round == 0 || k >> (shift + bits) == prefix)
                __hip_atomic_fetch_add(&s.bins[(k >> shift) & ((1u << bits) - 1)], (uint64_t)measure(), __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_WORKGROUP);
        });
        __syncthreads();
        const uint64_t b0 = s.bins[2 * tid], b1 = s.bins[2 * tid + 1];
        uint64_t total;
        const uint64_t upto = below + sf_scan<uint64_t>(b0 + b1, s.wave, total);
        if (total + below < need) return false;   // uniform; in the first round if ever
        if (upto >= need && upto - b0 - b1 < need) {
            const bool first = upto - b1 >= need;
            s.found = 2 * tid + !first;
            s.below = upto - b1 - (first ? b0 : 0);
        }
        __syncthreads();
        prefix = prefix << bits | (uint32_t)s.found;
        below = s.below;
        __syncthreads();
        shift -= round == 1 ? 10 : 11;
    }
    key = prefix;
    return true;
}

// The first of n elements at which the sum of measures passes t (t below the sum of
// all), on every thread: the wave's sixteenth that holds it, then that one's, down to
// an element per thread.
template <class M>
__device__ __forceinline__ int sf_first(SfLds& s, int n, uint64_t t, const M& measure) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int lo = 0, hi = n;
    uint64_t total;
#pragma unroll 1
    while (hi - lo > SF_NT) {
        const int part = (hi - lo + SF_NT - 1) / SF_NT * 64, a = lo + wave * part, e = min(a + part, hi);
        uint64_t m = 0;
        for (int i = a + lane; i < e; i += 64) m += measure(i);
        const uint64_t upto = sf_scan<uint64_t>(m, s.wave, total);
        const uint64_t all = __shfl(upto, 63, 64), before = __shfl(upto - m, 0, 64);
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
    const uint64_t m = lo + tid < hi ? measure(lo + tid) : 0;
    const uint64_t upto = sf_scan<uint64_t>(m, s.wave, total);
    if (upto > t && upto - m <= t) s.found = lo + tid;
    __syncthreads();
    const int at = s.found;
    __syncthreads();
    return min(max(at, 0), n - 1);                // an element even of rows that change meanwhile
}

// The row's tokens that can be kept: in LDS, or in memory.  key(i, k): element i's key,
// false if it is none; index and weight of element i.
struct SfInLds {
    const SfLds& s;
    int n;
    __device__ __forceinline__ bool key(int i, uint32_t& k) const {
        k = s.key[i];
        return true;
    }
    __device__ __forceinline__ int index(int i) const { return (int)(s.wi[i] & 0xfffff); }
    __device__ __forceinline__ uint64_t weight(int i) const { return s.wi[i] >> 20; }
};
struct SfInRow {
    const float* x;
    int n;
    float tau, M;
    double inv;
    __device__ __forceinline__ bool key(int i, uint32_t& k) const {
        k = sf_key(x[i]);
        return x[i] >= tau;
    }
    __device__ __forceinline__ int index(int i) const { return i; }
    __device__ __forceinline__ uint64_t weight(int i) const { return (uint64_t)rint(sf_weight(x[i], M, inv) * SF_ONE); }
};

// Selection and draw; all: the weight of every token of the row in units of 2^-42, where
// no top-k cuts it.  Elements ascend by index.
template <class S>
__device__ __forceinline__ void sf_choose(SfLds& s, const lgx_filter_args& a, const SfRow& r, int row, double all, const S& e) {
    // kept: key < last, or key == last and place <= most
    uint32_t last = 0xffffffffu;
    int most = 0x7fffffff;
    auto kept = [&](uint32_t key, int i) { return key < last || (key == last && i <= most); };
    auto each = [&](auto f) {
        uint32_t k;
        for (int i = threadIdx.x; i < e.n; i += SF_NT)
            if (e.key(i, k) && kept(k, i)) f(k, i);
    };
    auto sum = [&](auto f) {
        uint64_t n = 0, total;
        each([&](uint32_t k, int i) { n += f(k, i); });
        sf_scan<uint64_t>(n, s.wave, total);
        return total;
    };
    // of the kept tokens with key `last` only the first n (>= 1)
    auto cut = [&](uint64_t n) {
        if (sum([&](uint32_t k, int) { return k == last; }) <= n) return;
        const int at = sf_first(s, e.n, n - 1, [&](int i) {
            uint32_t k;
            return (uint64_t)(e.key(i, k) && k == last && i <= most);
        });
        most = at;
    };
    uint32_t key;
    uint64_t below;
    // fewer tokens than top_k that count: all of them
    if (r.k && sf_select(s, r.k, key, below, [&](auto f) { each([&](uint32_t k, int) { f(k, [] { return 1; }); }); })) {
        last = key;
        cut(r.k - below);
    }
    if (r.p < 1.0f) {
        // of the kept tokens those that reach the share, the first at least
        const double whole = r.k ? (double)sum([&](uint32_t, int i) { return e.weight(i); }) : all;
        const uint64_t need = max((uint64_t)ceil((double)r.p * whole), (uint64_t)1);
        if (sf_select(s, need, key, below, [&](auto f) { each([&](uint32_t k, int i) { f(k, [&] { return e.weight(i); }); }); })) {
            if (key != last) most = 0x7fffffff;
            last = key;
            // tokens of one logit weigh the same: what they weigh together, by their number
            const uint64_t w = sum([&](uint32_t k, int i) { return k == last ? e.weight(i) : 0; }) /
                               sum([&](uint32_t k, int) { return k == last; });
            cut((need - below + w - 1) / w);
        }
    }
    const uint64_t low = (uint64_t)ceil((double)r.mp * SF_ONE);
    auto weight = [&](int i) {
        const uint64_t w = e.weight(i);
        return w >= low ? w : 0;
    };
    const uint64_t total = sum([&](uint32_t, int i) { return weight(i); });
    const double u = (double)a.u[row];
    const uint64_t t = u > 0.0 ? min((uint64_t)(fmin(u, 1.0) * (double)total), total - 1) : 0;
    const int at = sf_first(s, e.n, t, [&](int i) {
        uint32_t k;
        return e.key(i, k) && kept(k, i) ? weight(i) : 0;
    });
    if (threadIdx.x == 0) {
        a.out[row] = e.index(at);
        if (a.prob) a.prob[row] = (float)((double)weight(at) / (double)total);
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
    // the row's maximum: at most 256 slices
    float M = ninf;
    for (int i = lane; i < a.nslices; i += 64) M = fmaxf(M, smax[i]);
    M = wave_max(M);
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
        for (int c = tid; c < nruns; c += SF_NT)
            if (cmax[c] == M) __hip_atomic_fetch_min(&s.found, c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
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
    double S = 0.0;                               // of all weights, by M
    if (r.sums()) {
        const double* sums = a.sum + (int64_t)row * a.nslices;
        const double mine = tid < a.nslices ? sums[tid] * sf_weight(smax[tid], M, r.inv) : 0.0;
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
                w[i] = e0 + i < V ? sf_weight(x[min(e0 + i, V - 1)], M, r.inv) : 0.0;
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
    const float T = (float)(1.0 / r.inv);
    float tau = M - 30.0f * T;
    if (r.mp > 0.0f && !(r.k && r.p < 1.0f)) tau = fmaxf(tau, M + T * (logf(r.mp) - 0.001f));
    if (r.p < 1.0f && !r.k) tau = fmaxf(tau, M + T * (logf((1.0f - r.p) / (float)V) + logf((float)S) - 0.001f));
    tau -= fmaxf(fabsf(M), fabsf(tau)) * 1e-6f;
    if (!(tau == tau)) tau = M == __builtin_inff() ? M : ninf;
    if (r.k && r.k <= nruns) {
        uint64_t below;
        uint32_t key;
        sf_select(s, r.k, key, below, [&](auto f) {
            for (int c = tid; c < nruns; c += SF_NT) f(sf_key(cmax[c]), [] { return 1; });
        });
        tau = fmaxf(tau, __uint_as_float(key & 0x80000000u ? key : ~key & 0x7fffffffu));
    }
    // the runs that reach it, in order
    uint16_t* runs = (uint16_t*)s.bins;
    uint16_t* place = runs + SF_LIST;
    static_assert(2 * SF_LIST * sizeof(uint16_t) <= sizeof(s.bins) && LGX_SF_VOCAB / LGX_SF_CHUNK <= 65536, "runs and places in the bins");
    int nr = 0;
    for (int c0 = 0; c0 < nruns; c0 += SF_NT) {
        const int c = c0 + tid;
        const bool on = c < nruns && cmax[min(c, nruns - 1)] >= tau;
        uint64_t more;
        const int at = nr + (int)sf_scan<uint64_t>(on, s.wave, more) - 1;
        if (on && at < SF_LIST) runs[at] = (uint16_t)c;
        nr += (int)more;
    }
    __syncthreads();
    int n = 0;
    bool fits = nr <= SF_LIST;
    // f(q, the lane's token of run q, its logit): waves take the runs in turn, four in flight
    auto tokens = [&](auto f) {
        for (int q0 = wave; q0 < nr; q0 += SF_NT / 16) {
            float v[4];
            int t[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                t[u] = runs[min(q0 + u * (SF_NT / 64), nr - 1)] * LGX_SF_CHUNK + lane;
                v[u] = t[u] < V ? x[t[u]] : __builtin_nanf("");
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (q0 + u * (SF_NT / 64) < nr) f(q0 + u * (SF_NT / 64), t[u], v[u]);
        }
    };
    if (fits) {
        tokens([&](int q, int, float v) {
            const int c = __builtin_popcountll(__builtin_amdgcn_ballot_w64(v >= tau));
            if (lane == 0) place[q] = (uint16_t)c;
        });
        __syncthreads();
        for (int q0 = 0; q0 < nr; q0 += SF_NT) {
            const int q = q0 + tid, c = q < nr ? place[q] : 0;
            uint64_t more;
            const int at = n + (int)sf_scan<uint64_t>((uint64_t)c, s.wave, more) - c;
            if (q < nr) place[q] = (uint16_t)min(at, SF_LIST);
            n += (int)more;
        }
        fits = n <= SF_LIST;
        __syncthreads();
    }
    const double all = S * SF_ONE;
    if (fits) {                                   // uniform
        tokens([&](int q, int t, float v) {
            const uint64_t hit = __builtin_amdgcn_ballot_w64(v >= tau);
            const int to = place[q] + __builtin_popcountll(hit & ((1ull << lane) - 1));
            if (v >= tau) {
                s.key[to] = sf_key(v);
                s.wi[to] = (uint64_t)rint(sf_weight(v, M, r.inv) * SF_ONE) << 20 | (uint64_t)t;
            }
        });
        __syncthreads();
        sf_choose(s, a, r, row, all, SfInLds{s, n});
    } else {
        // more than LDS holds: the row itself
        sf_choose(s, a, r, row, all, SfInRow{x, V, tau, M, r.inv});
    }
}
