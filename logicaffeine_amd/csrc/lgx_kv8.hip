// lgx_kv8.hip -- the 8-bit KV cache: append with rotation, read-back, and the
// attention of decode and prefill rows over it.  Part of lgx_kernels.hip (one
// code object).
//
// Format.  A block is the 16 tokens of a page for one KV head; K and V blocks
// hold int8 quants and one binary32 scale each, value = scale * quant.  K lies
// token by token ([16][d]); V dimension by dimension ([d][16]), the order in
// which the PV product takes it: 16 tokens of a dimension are one 16-byte load.

// ---------------------------------------------------------------------------
// Append.  All arithmetic between the binary32 input and the rounded result is
// binary64, so a quant next to a rounding border does not depend on how the
// products were formed.
// A block that already holds tokens keeps its scale unless a new value exceeds
// 127 of it; then the scale doubles until it does not and the old quants are
// halved as often, rounded once: an old value is off by less than one step of
// the final scale however often its block grew (1/2 + 1/4 + ...).
//
// A head is D / 2 pairs: pair p < rot / 2 is (p, p + rot / 2), or (2p, 2p + 1)
// when interleaved, and turns; the others are (2p, 2p + 1) and do not.  A thread
// holds E / 2 consecutive pairs as two runs of E / 2 dimensions (Pairs): the two
// members of its turning pairs, or E neighbours.
// ---------------------------------------------------------------------------
template <int H>
struct Pairs {
    int ia, ib;        // first dimension of each run
    int p;             // first pair
    bool apart, turn;  // members half a rotation apart; any of the pairs turns
};
// Runs of H pairs from pair p on of a head with `rot` turning dimensions; `vec`:
// rot / 2 is a multiple of H, so that the pairs of a run are all of one kind.
template <int H>
__device__ __forceinline__ Pairs<H> pairs_of(int p, int rot, bool inter, bool vec) {
    Pairs<H> r;
    r.p = p;
    r.turn = p < rot / 2;
    r.apart = vec && r.turn && !inter;
    r.ia = r.apart ? p : 2 * p;
    r.ib = r.apart ? p + rot / 2 : 2 * p + H;
    return r;
}
// Dimensions of pair p + k, one by one (rot / 2 not a multiple of H).
__device__ __forceinline__ void pair_dims(int p, int rot, bool inter, int& i0, int& i1) {
    const bool apart = p < rot / 2 && !inter;
    i0 = apart ? p : 2 * p;
    i1 = apart ? p + rot / 2 : 2 * p + 1;
}
template <int H>
struct RunT;
template <>
struct RunT<1> { typedef float type __attribute__((ext_vector_type(1))); };
template <>
struct RunT<2> { typedef float type __attribute__((ext_vector_type(2))); };
template <>
struct RunT<4> { typedef float type __attribute__((ext_vector_type(4))); };

// The head row's values at the thread's pairs: x[k], z[k] the members of pair k
// (runs that are neighbours come out as (2k, 2k + 1) too), bias added.
template <int H>
__device__ __forceinline__ void load_pairs(const float* xr, const float* br, const Pairs<H>& w, int rot, bool inter, bool vec,
                                           double (&x)[H], double (&z)[H]) {
    typedef typename RunT<H>::type V;
    if (vec) {                                    // uniform
        float v[2 * H], o[2 * H];
        *(V*)v = *(const V*)(xr + w.ia);
        *(V*)(v + H) = *(const V*)(xr + w.ib);
        if (br) {
            *(V*)o = *(const V*)(br + w.ia);
            *(V*)(o + H) = *(const V*)(br + w.ib);
        }
#pragma unroll
        for (int k = 0; k < H; ++k) {
            x[k] = w.apart ? v[k] : v[2 * k];
            z[k] = w.apart ? v[H + k] : v[2 * k + 1];
            if (br) {
                x[k] += w.apart ? o[k] : o[2 * k];
                z[k] += w.apart ? o[H + k] : o[2 * k + 1];
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < H; ++k) {
            int i0, i1;
            pair_dims(w.p + k, rot, inter, i0, i1);
            x[k] = xr[i0];
            z[k] = xr[i1];
            if (br) {
                x[k] += br[i0];
                z[k] += br[i1];
            }
        }
    }
}
// The tables' values of the thread's pairs at a position; (1, 0) where a pair
// does not turn.
template <int H>
__device__ __forceinline__ void load_turns(const lgx_kv8_append_args& a, const Pairs<H>& w, int64_t pos, bool vec, float (&c)[H],
                                           float (&s)[H]) {
    typedef typename RunT<H>::type V;
    const int64_t at = pos * (a.rot / 2) + w.p;
    if (vec) {
        if (w.turn) {
            *(V*)c = *(const V*)(a.cos_t + at);
            *(V*)s = *(const V*)(a.sin_t + at);
        } else {
#pragma unroll
            for (int k = 0; k < H; ++k) c[k] = 1.0f, s[k] = 0.0f;
        }
    } else {
#pragma unroll
        for (int k = 0; k < H; ++k) {
            const bool on = w.p + k < a.rot / 2;
            c[k] = on ? a.cos_t[at + k] : 1.0f;
            s[k] = on ? a.sin_t[at + k] : 0.0f;
        }
    }
}
// The pair's rotation; one that does not turn keeps its bits (an infinite member
// would meet the other's 0).
template <int H>
__device__ __forceinline__ void turn_pairs(const float (&c)[H], const float (&s)[H], const Pairs<H>& w, int rot, double (&x)[H],
                                           double (&z)[H]) {
#pragma unroll
    for (int k = 0; k < H; ++k) {
        const double y0 = x[k] * (double)c[k] - z[k] * (double)s[k], y1 = z[k] * (double)c[k] + x[k] * (double)s[k];
        const bool on = w.p + k < rot / 2;
        x[k] = on ? y0 : x[k];
        z[k] = on ? y1 : z[k];
    }
}
template <int H>
__device__ __forceinline__ void store_q(float* q, const Pairs<H>& w, int rot, bool inter, bool vec, const double (&x)[H],
                                        const double (&z)[H]) {
    typedef typename RunT<H>::type V;
    if (vec) {
        float v[2 * H];
#pragma unroll
        for (int k = 0; k < H; ++k) {
            // runs of one member, or neighbours in turn
            v[k] = (float)(w.apart ? x[k] : k & 1 ? z[k / 2] : x[k / 2]);
            v[H + k] = (float)(w.apart ? z[k] : k & 1 ? z[(H + k) / 2] : x[(H + k) / 2]);
        }
        *(V*)(q + w.ia) = *(const V*)v;
        *(V*)(q + w.ib) = *(const V*)(v + H);
    } else {
#pragma unroll
        for (int k = 0; k < H; ++k) {
            int i0, i1;
            pair_dims(w.p + k, rot, inter, i0, i1);
            q[i0] = (float)x[k];
            q[i1] = (float)z[k];
        }
    }
}
// The scale of a block: `need` of its new values (NaN where one is not finite),
// `old` the scale of the tokens it holds (0 for a new block); grow: doublings.
__device__ __forceinline__ float block_scale(double am, bool bad, float old, int& grow) {
    // a block whose values are all below 2^-119 is zero: scales are normal numbers
    const float need = am < 0x1p-119 ? 0.0f : (float)(am / 127.0);
    grow = 0;
    if (bad || !(old >= 0.0f && old < __builtin_inff())) return __builtin_nanf("");
    if (!(old > 0.0f)) return need;
    float scale = old;
    while (scale < need) {
        scale *= 2.0f;
        ++grow;
    }
    return scale;
}
// The integer nearest to y / scale, halves away from zero; inv: 1 / scale rounded (0
// for a scale of 0 or NaN, whose quants are 0).  |y| inv, rounded too, may say one
// integer less or more than the quotient's whole part; what is left of |y| after
// that many scales is a multiple of the smaller of their units and no larger than |y|,
// so a binary64 number, and its comparison with half a scale is exact.
__device__ __forceinline__ int quant8(double y, double scale, double inv) {
    const double a = fabs(y), m = floor(a * inv);
    const int q = min((int)m + (inv > 0.0 && fma(-m, scale, a) >= 0.5 * scale), 127);
    return y < 0.0 ? -q : q;
}
__device__ __forceinline__ int halve8(int v, int grow) {
    const int m = grow > 8 ? 0 : ((v < 0 ? -v : v) + (1 << (grow - 1))) >> grow;
    return v < 0 ? -m : m;
}

// Workgroup (block of 16 token slots of sequence b; QH query heads, or a K or V
// head): thread (slot, c) holds D / 32 pairs of the slot's row.  Query heads share
// the thread's cosines and sines.  Bound by memory: 8 x 2047 rows of 28/4 heads of
// 128, 575 MB, in 130 us (4.4 TB/s; a copy reaches 5.2); 643 us with every element's
// row, partner and tables loaded number by number.
#define KV8_QH LGX_KV8_QH
template <int D>
__device__ __forceinline__ void kv8_append_body(const lgx_kv8_append_args& a) {
    constexpr int H = D / 32;
    __shared__ double am_s[4];
    __shared__ int bad_s[4];
    __shared__ __align__(16) int8_t v_s[D * LGX_PAGE];
    const int tid = threadIdx.x, slot = tid >> 4;
    const int b = blockIdx.x / a.nblk, nqg = (a.hq + KV8_QH - 1) / KV8_QH;
    const bool isq = (int)blockIdx.y < nqg, isv = (int)blockIdx.y >= nqg + a.hkv;
    const int sl = min(max(a.seq_len[b], 0), a.maxp * LGX_PAGE);
    const int nn = a.n_new ? min(max(a.n_new[b], 0), a.P) : a.P;
    const int pb = sl / LGX_PAGE + (blockIdx.x - b * a.nblk), t0 = pb * LGX_PAGE;
    if (nn == 0 || t0 >= sl + nn) return;         // uniform: no new row in this block
    const int j = t0 + slot - sl;                 // row of this slot
    const bool is_new = j >= 0 && j < nn;
    const int rot = isv ? 0 : a.rot;
    const bool inter = a.interleaved != 0, vec = a.vec != 0;
    const Pairs<H> w = pairs_of<H>((tid & 15) * H, rot, inter, vec);
    const int64_t row = (int64_t)b * a.P + j;
    const float* xr = a.x + row * ((int64_t)(a.hq + 2 * a.hkv) * D);
    float c[H], s[H];
    if (is_new && !isv) load_turns<H>(a, w, min(t0 + slot, a.max_pos - 1), vec, c, s);
    if (isq) {
        if (!is_new) return;
        const int h0 = blockIdx.y * KV8_QH;
        double x[KV8_QH][H], z[KV8_QH][H];
#pragma unroll
        for (int i = 0; i < KV8_QH; ++i) {
            const int h = min(h0 + i, a.hq - 1);
            load_pairs<H>(xr + h * D, a.bias ? a.bias + h * D : nullptr, w, rot, inter, vec, x[i], z[i]);
        }
#pragma unroll
        for (int i = 0; i < KV8_QH; ++i) {
            if (h0 + i >= a.hq) break;            // uniform
            turn_pairs<H>(c, s, w, rot, x[i], z[i]);
            store_q<H>(a.q_out + (row * a.hq + h0 + i) * D, w, rot, inter, vec, x[i], z[i]);
        }
        return;
    }
    if (pb >= a.maxp) return;                     // uniform: past the sequence's pages
    const int page = a.page_table[(int64_t)b * a.maxp + pb];
    if (page < 0 || page >= a.num_pages) return;  // uniform
    const int g = blockIdx.y - nqg - (isv ? a.hkv : 0), hh = a.hq + (isv ? a.hkv : 0) + g;
    double y[2 * H];
    {
        double x[H], z[H];
#pragma unroll
        for (int k = 0; k < H; ++k) x[k] = z[k] = 0.0;
        if (is_new) {
            load_pairs<H>(xr + hh * D, a.bias ? a.bias + hh * D : nullptr, w, rot, inter, vec, x, z);
            if (!isv) turn_pairs<H>(c, s, w, rot, x, z);
        }
#pragma unroll
        for (int k = 0; k < H; ++k) {
            y[k] = x[k];
            y[H + k] = z[k];
        }
    }
    // dimension of y[e]
    auto dim = [&](int e) {
        if (vec) return w.apart ? (e < H ? w.ia + e : w.ib + e - H) : 2 * (w.p + e % H) + e / H;
        int i0, i1;
        pair_dims(w.p + e % H, rot, inter, i0, i1);
        return e < H ? i0 : i1;
    };
    double am = 0.0;
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 2 * H; ++e) {
        am = fmax(am, fabs(y[e]));
        bad = bad || !(fabs(y[e]) < __builtin_inf());
    }
#pragma unroll
    for (int m = 32; m; m >>= 1) am = fmax(am, __shfl_xor(am, m, 64));
    const bool wave_bad = __builtin_amdgcn_ballot_w64(bad) != 0;
    if ((tid & 63) == 0) {
        am_s[tid >> 6] = am;
        bad_s[tid >> 6] = wave_bad;
    }
    const int64_t blk = (int64_t)page * a.hkv + g;
    float* sp = (isv ? a.vs : a.ks) + blk;
    const int s0 = max(sl - t0, 0);               // the first new slot
    const float old = s0 ? *sp : 0.0f;
    __syncthreads();
    am = fmax(fmax(am_s[0], am_s[1]), fmax(am_s[2], am_s[3]));
    bad = bad_s[0] || bad_s[1] || bad_s[2] || bad_s[3];
    int grow;
    const float scale = block_scale(am, bad, old, grow);
    __syncthreads();                              // every wave has read the old scale
    if (tid == 0) *sp = scale;
    const double inv = scale > 0.0f ? 1.0 / (double)scale : 0.0;
    int q[2 * H];
#pragma unroll
    for (int e = 0; e < 2 * H; ++e) q[e] = bad ? 0 : quant8(y[e], scale, inv);
    const bool again = slot < s0 && grow > 0;     // an old token whose quants shrink
    if (!isv) {
        int8_t* kr = a.k + (blk * LGX_PAGE + slot) * D;
        if (again) {
#pragma unroll
            for (int e = 0; e < 2 * H; ++e) q[e] = halve8(kr[dim(e)], grow);
        }
        if (is_new || again) {
            if (vec) {
                // the runs' bytes in one store each
                uint32_t ra = 0, rb = 0;
#pragma unroll
                for (int k = 0; k < H; ++k) {
                    const int ea = w.apart ? q[k] : q[(k & 1) * H + k / 2];
                    const int eb = w.apart ? q[H + k] : q[(k & 1) * H + (H + k) / 2];
                    ra |= (uint32_t)(ea & 255) << (8 * k);
                    rb |= (uint32_t)(eb & 255) << (8 * k);
                }
                if (H == 4) {
                    *(uint32_t*)(kr + w.ia) = ra;
                    *(uint32_t*)(kr + w.ib) = rb;
                } else {
                    *(uint16_t*)(kr + w.ia) = (uint16_t)ra;
                    *(uint16_t*)(kr + w.ib) = (uint16_t)rb;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 2 * H; ++e) kr[dim(e)] = (int8_t)q[e];
            }
        }
        return;
    }
    int8_t* vb = a.v + blk * LGX_PAGE * D;
    if (s0 == 0 && t0 + LGX_PAGE <= sl + nn) {    // uniform: a whole block
#pragma unroll
        for (int e = 0; e < 2 * H; ++e) v_s[dim(e) * LGX_PAGE + slot] = (int8_t)q[e];
        __syncthreads();
        if (tid < D) *(uint4*)(vb + tid * LGX_PAGE) = *(const uint4*)(v_s + tid * LGX_PAGE);
        return;
    }
    if (again) {
#pragma unroll
        for (int e = 0; e < 2 * H; ++e) q[e] = halve8(vb[dim(e) * LGX_PAGE + slot], grow);
    }
    if (is_new || again) {
#pragma unroll
        for (int e = 0; e < 2 * H; ++e) vb[dim(e) * LGX_PAGE + slot] = (int8_t)q[e];
    }
}
extern "C" __global__ __launch_bounds__(256) void lgx_k_kv8_append_d64(const lgx_kv8_append_args a) { kv8_append_body<64>(a); }
extern "C" __global__ __launch_bounds__(256) void lgx_k_kv8_append_d128(const lgx_kv8_append_args a) { kv8_append_body<128>(a); }

// One new row per sequence (a decode step): a wave per head, a pair per lane (with
// D = 64 the upper half of the wave idles).  The row does not depend on the
// length, so its loads are in flight together with the length's, and the cosines
// with the page's.  Bound by those two memory rounds and the launch: 64 sequences of
// 28/4 heads of 128 in 4.1 us (8.7 with the form above, 16 of its 256 threads at
// work).
template <int D>
__device__ __forceinline__ void kv8_append1_body(const lgx_kv8_append_args& a) {
    const int p = threadIdx.x & 63, b = blockIdx.x;
    const int hh = __builtin_amdgcn_readfirstlane(blockIdx.y * 4 + (threadIdx.x >> 6));
    const bool on = p < D / 2, isv = hh >= a.hq + a.hkv, inter = a.interleaved != 0;
    if (hh >= a.hq + 2 * a.hkv || (a.n_new && a.n_new[b] < 1)) return;   // uniform per wave
    const int rot = isv ? 0 : a.rot;
    int i0, i1;
    pair_dims(on ? p : 0, rot, inter, i0, i1);
    const int64_t at = (int64_t)b * (a.hq + 2 * a.hkv) * D + hh * D;
    double x[1] = {a.x[at + i0]}, z[1] = {a.x[at + i1]};
    const int sl = min(max(a.seq_len[b], 0), a.maxp * LGX_PAGE);
    const int pb = sl / LGX_PAGE;
    if (a.bias) {
        x[0] += a.bias[hh * D + i0];
        z[0] += a.bias[hh * D + i1];
    }
    const int page = pb < a.maxp ? a.page_table[(int64_t)b * a.maxp + pb] : -1;
    const Pairs<1> w = {i0, i1, p, false, p < rot / 2};
    if (!isv) {
        float c[1], s[1];
        load_turns<1>(a, w, min(sl, a.max_pos - 1), false, c, s);
        turn_pairs<1>(c, s, w, rot, x, z);
    }
    if (hh < a.hq) {
        if (on) store_q<1>(a.q_out + ((int64_t)b * a.hq + hh) * D, w, rot, inter, false, x, z);
        return;
    }
    if (page < 0 || page >= a.num_pages) return;
    const int g = hh - a.hq - (isv ? a.hkv : 0), s0 = sl % LGX_PAGE;
    const int64_t blk = (int64_t)page * a.hkv + g;
    float* sp = (isv ? a.vs : a.ks) + blk;
    const float old = s0 ? *sp : 0.0f;
    double am = on ? fmax(fabs(x[0]), fabs(z[0])) : 0.0;
    const bool bad = __builtin_amdgcn_ballot_w64(on && !(fabs(x[0]) < __builtin_inf() && fabs(z[0]) < __builtin_inf())) != 0;
#pragma unroll
    for (int m = 32; m; m >>= 1) am = fmax(am, __shfl_xor(am, m, 64));
    int grow;
    const float scale = block_scale(am, bad, old, grow);
    if (p == 0) *sp = scale;
    if (!on) return;
    const double inv = scale > 0.0f ? 1.0 / (double)scale : 0.0;
    const int q0 = bad ? 0 : quant8(x[0], scale, inv), q1 = bad ? 0 : quant8(z[0], scale, inv);
    // K: slot s0 of 16 rows; V: column s0
    int8_t* base = (isv ? a.v : a.k) + blk * LGX_PAGE * D;
    const int ds = isv ? LGX_PAGE : 1, ts = isv ? 1 : D;
    if (grow > 0)
        for (int t = 0; t < s0; ++t) {
            int8_t *e0 = base + i0 * ds + t * ts, *e1 = base + i1 * ds + t * ts;
            *e0 = (int8_t)halve8(*e0, grow);
            *e1 = (int8_t)halve8(*e1, grow);
        }
    base[i0 * ds + s0 * ts] = (int8_t)q0;
    base[i1 * ds + s0 * ts] = (int8_t)q1;
}
extern "C" __global__ __launch_bounds__(256) void lgx_k_kv8_append1_d64(const lgx_kv8_append_args a) { kv8_append1_body<64>(a); }
extern "C" __global__ __launch_bounds__(256) void lgx_k_kv8_append1_d128(const lgx_kv8_append_args a) { kv8_append1_body<128>(a); }

// ---------------------------------------------------------------------------
// Read-back: tokens start[b] .. + n of every sequence as binary32.  Workgroup
// (block of 16 token slots of sequence b, KV head).  K: thread (slot, c) has d / 16
// neighbouring values.  V: a thread has a run of tokens of one dimension, so that
// neighbouring threads write neighbouring dimensions of a row.  Bound by memory: 8 x
// 2064 rows of 4 heads of 128, 85 MB, in 17.5 us (4.8 TB/s; V through LDS, written by
// the row's threads: 38 us, the byte reads of 16 dimensions met in one bank).
// ---------------------------------------------------------------------------
template <int D>
__device__ __forceinline__ void kv8_read_body(const lgx_kv8_read_args& a) {
    constexpr int E = D / 16, NT = LGX_PAGE * D / 256;   // tokens of a thread's V run: 8 or 4
    const int tid = threadIdx.x, slot = tid >> 4, e0 = (tid & 15) * E;
    const int b = blockIdx.x / a.nblk, g = blockIdx.y;
    const int st = min(max(a.start[b], 0), a.maxp * LGX_PAGE);
    const int pb = st / LGX_PAGE + (blockIdx.x - b * a.nblk);
    const int64_t row0 = (int64_t)pb * LGX_PAGE - st;    // row of slot 0, possibly before the first
    const bool has = pb < a.maxp;                        // uniform
    const int page = has ? min(max(a.page_table[(int64_t)b * a.maxp + pb], 0), a.num_pages - 1) : 0;
    const int64_t blk = (int64_t)page * a.hkv + g;
    const float ks = has ? a.ks[blk] : 0.0f, vs = has ? a.vs[blk] : 0.0f;
    int8_t kq[E], vq[NT];
    const int dim = tid % D, t0 = tid / D * NT;
    if (E == 8) {
        *(uint2*)kq = *(const uint2*)(a.k + (blk * LGX_PAGE + slot) * D + e0);
        *(uint2*)vq = *(const uint2*)(a.v + (blk * D + dim) * LGX_PAGE + t0);
    } else {
        *(uint32_t*)kq = *(const uint32_t*)(a.k + (blk * LGX_PAGE + slot) * D + e0);
        *(uint32_t*)vq = *(const uint32_t*)(a.v + (blk * D + dim) * LGX_PAGE + t0);
    }
    auto at = [&](int64_t row) { return (((int64_t)b * a.n + row) * a.hkv + g) * D; };
    auto on = [&](int64_t row) { return row >= 0 && row < a.n; };
    if (on(row0 + slot)) {
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            float f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = has ? ks * (float)kq[e + i] : 0.0f;
            *(float4*)(a.k_out + at(row0 + slot) + e0 + e) = make_float4(f[0], f[1], f[2], f[3]);
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
        if (on(row0 + t0 + t)) a.v_out[at(row0 + t0 + t) + dim] = has ? vs * (float)vq[t] : 0.0f;
}
extern "C" __global__ __launch_bounds__(256) void lgx_k_kv8_read_d64(const lgx_kv8_read_args a) { kv8_read_body<64>(a); }
extern "C" __global__ __launch_bounds__(256) void lgx_k_kv8_read_d128(const lgx_kv8_read_args a) { kv8_read_body<128>(a); }

// ---------------------------------------------------------------------------
// Attention.  The (row, query head) pairs of one KV head are the columns of the
// products, 16 to a matrix instruction; a tile is 64 tokens, four pages.
//   scores   S^T[token][column] = K . Q^T on v_mfma_i32_16x16x64_i8, K quants as
//            they lie in memory.  q is an integer of 24 bits (its row scaled by a
//            power of two) in three signed base-256 digits: three exact int32
//            products, joined in binary32.  (128 columns: K and two parts of q in
//            binary16.)
//   softmax  running maximum and sum per column, in base 2.
//   PV       O^T[dim][column] += V^T . P^T on v_mfma_f32_16x16x32_f16: V quants are
//            binary16 numbers, a weight (times its page's V scale) is the sum of
//            two binary16 numbers, 22 bits.  The matrix unit sums a tile, the VALU
//            the tiles, both in binary32.
// Row 4 p + v of score sub-tile u is token 4 u + v of page p, so that lane (column,
// kg) ends up with all 16 scores of page kg: its scales are one value per lane,
// and its weights are the PV operand as they stand (V's 16-byte loads give lane
// (dim, kg) the 16 tokens of page kg).  Scores and weights pass neither through LDS
// nor across lanes, but for the column's maxima; through LDS go, with 32 columns, the
// query's digits, and with 128 the tiles of K and V.
// ---------------------------------------------------------------------------

// Four int8 quants as binary16: the byte of v + 128 under the exponent of 1024
// is 1152 + v.
__device__ __forceinline__ void i8_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    typedef _Float16 v2h __attribute__((ext_vector_type(2)));
    const uint32_t x = w ^ 0x80808080u;
    const v2h off = {(_Float16)1152.0f, (_Float16)1152.0f};
    const v2h l = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) - off;
    const v2h h = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) - off;
    lo = __builtin_bit_cast(uint32_t, l);
    hi = __builtin_bit_cast(uint32_t, h);
}

// What a workgroup of NC columns works on: a sequence, a KV head, a block of
// columns, and a run of tiles.
struct A8Block {
    int b, g, G, c0, ncols, sl;
    int tb0, tb1;      // tiles
    int unit;          // b * ncb + column block
    int pos, ns;       // place among all splits, and splits of the unit
};
template <int NC, bool X>
struct A8 {
    const lgx_attn8_args& a;
    A8Block k;
    // tokens that the row of column c of a sequence of sl tokens sees: [first, last)
    __device__ __forceinline__ int last(int sl, int c) const {
        const int j = a.P == 1 ? 0 : c / k.G;
        return (int)min((int64_t)sl + j + a.len_add, (int64_t)a.maxlen);
    }
    __device__ __forceinline__ int first(int sl, int c) const { return X && a.window ? max(last(sl, c) - a.window, 0) : 0; }
    __device__ __forceinline__ int last(int c) const { return last(k.sl, c); }
    __device__ __forceinline__ int first(int c) const { return first(k.sl, c); }
    __device__ __forceinline__ int rows(int b) const { return a.n_new ? min(max(a.n_new[b], 0), a.P) : a.P; }
    __device__ __forceinline__ int2 tiles(int sl, int c0, int ncols) const {
        return make_int2(first(sl, c0) / LGX_A8_TILE,
                         (last(sl, min(c0 + NC, ncols) - 1) + LGX_A8_TILE - 1) / LGX_A8_TILE);
    }
    // false: nothing to do.  With a.per alone, all units' tiles go in about equal runs
    // to the workgroups: every wave computes the run length from all lengths (four
    // units per lane), nearly the least with which all runs fit into a.per per KV
    // head, then finds the unit and the run of this workgroup in the sums over the
    // units.  Against runs that would do if all sequences had the longest length:
    // 32 sequences of 1024 to 16384 tokens, 12/2 heads of 128, 38.1 against 45.8 us, 16
    // of 512 to 8192, 28/4 heads, 22.5 against 24.7; equal lengths, where the
    // computation buys nothing, 34.4 against 33.6.
    __device__ __forceinline__ bool place() {
        k.G = a.hq / a.hkv;
        int s = 0, cps = a.cps;
        if (a.cps) {
            // one unit without a window: runs of a fixed length, which nothing has
            // to be read for
            s = k.pos = __builtin_amdgcn_readfirstlane(blockIdx.x / a.hkv);
            k.g = blockIdx.x - s * a.hkv;
            k.unit = 0;
            k.ns = a.per;
            if (blockIdx.x == 0 && threadIdx.x == 0) {
                a.plan[0] = 0;
                a.plan[1] = a.per;
            }
        } else if (a.per) {
            const int lane = threadIdx.x & 63;
            k.pos = __builtin_amdgcn_readfirstlane(blockIdx.x / a.hkv);
            k.g = blockIdx.x - k.pos * a.hkv;
            int n[4], len[4], cnt[4], all = 0;    // tiles of the lane's units; -1: no such columns
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int u = 4 * lane + i, uc = min(u, a.units - 1), b = a.ncb == 1 ? uc : uc / a.ncb;
                const int c0 = (uc - b * a.ncb) * NC;
                cnt[i] = rows(b) * k.G;
                len[i] = max(a.seq_len[b], 0);
                const int2 t = tiles(len[i], c0, cnt[i]);
                n[i] = u < a.units && c0 < cnt[i] ? t.y - t.x : -1;
                all += max(n[i], 0);
            }
            const int total = __builtin_amdgcn_readlane(wave_scan(all), 63);
            cps = max(LGX_A8_MIN, (int)((unsigned)(total + a.per - 1) / (unsigned)a.per));
            int m[4], upto;
            for (;;) {
                int c = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    m[i] = n[i] < 0 ? 0 : max((int)((unsigned)(n[i] + cps - 1) / (unsigned)cps), 1);
                    c += m[i];
                }
                upto = wave_scan(c);
                if (__builtin_amdgcn_readlane(upto, 63) <= a.per) break;
                cps += max(1, cps >> 4);          // ends: a.per >= a.units
            }
            const uint64_t past = __builtin_amdgcn_ballot_w64(upto > k.pos);
            if (!past) return false;
            const int at = __builtin_ctzll(past);
            s = k.pos - __builtin_amdgcn_readlane(upto - (m[0] + m[1] + m[2] + m[3]), at);
            int i = 0;
#pragma unroll
            for (int q = 0; q < 3; ++q) {
                const int mq = __builtin_amdgcn_readlane(m[q], at);
                const bool next = i == q && s >= mq;
                s -= next ? mq : 0;
                i += next ? 1 : 0;
            }
            auto pick = [&](const int (&v)[4]) {
                const int v0 = __builtin_amdgcn_readlane(v[0], at), v1 = __builtin_amdgcn_readlane(v[1], at);
                const int v2 = __builtin_amdgcn_readlane(v[2], at), v3 = __builtin_amdgcn_readlane(v[3], at);
                return i == 0 ? v0 : i == 1 ? v1 : i == 2 ? v2 : v3;
            };
            k.ns = pick(m);
            k.sl = pick(len);
            k.ncols = pick(cnt);
            k.unit = 4 * at + i;
            if (s == 0 && k.g == 0 && threadIdx.x == 0) {
                a.plan[2 * k.unit] = k.pos;
                a.plan[2 * k.unit + 1] = k.ns;
            }
        } else {
            // column blocks side by side: they share K and V
            const int bg = blockIdx.x / a.ncb, cb = blockIdx.x - bg * a.ncb;
            const int b = bg / a.hkv;
            k.g = __builtin_amdgcn_readfirstlane(bg - b * a.hkv);
            k.unit = __builtin_amdgcn_readfirstlane(b * a.ncb + cb);
            k.ns = 1;
        }
        k.b = __builtin_amdgcn_readfirstlane(k.unit / a.ncb);
        k.c0 = (k.unit - k.b * a.ncb) * NC;
        if (!a.per || a.cps) {
            k.ncols = rows(k.b) * k.G;
            k.sl = max(a.seq_len[k.b], 0);
        }
        if (k.c0 >= k.ncols) return false;
        const int2 t = tiles(k.sl, k.c0, k.ncols);
        k.tb0 = t.x + s * cps;
        k.tb1 = a.per ? min(t.y, k.tb0 + cps) : t.y;
        return true;
    }
};

// The query of a lane's column: its digits as B operands, the factor that turns
// an integer score (times the page's K scale) into a score (in base 2 unless X).
template <int NS>
__device__ __forceinline__ void a8_query_load(const float* qr, float (&x)[NS][16]) {
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const float4 v = *(const float4*)(qr + 64 * s + e);
            x[s][e] = v.x;
            x[s][e + 1] = v.y;
            x[s][e + 2] = v.z;
            x[s][e + 3] = v.w;
        }
}
template <int NS, bool X>
__device__ __forceinline__ float a8_query(const lgx_attn8_args& a, const float (&x)[NS][16], v4i (&qd)[3][NS]) {
    float am = 0.0f;
    bool bad = false;
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            am = fmaxf(am, fabsf(x[s][e]));
            bad = bad || !(fabsf(x[s][e]) < __builtin_inff());
        }
    am = col_max(am);
    const bool isbad = col_max(bad ? 1.0f : 0.0f) != 0.0f;
    // the largest power of two that keeps every |q| within 127 * 65536, the range of
    // three balanced digits; up to 2^122, where scale / up is still a normal number (rows
    // below 2^-99 in magnitude have fewer bits)
    const float up = __uint_as_float(__float_as_uint(fminf(127.0f * 65536.0f / am, 0x1p122f)) & 0x7f800000u);
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            uint32_t v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float y = isbad ? 0.0f : x[s][4 * w + e] * up;
                v[e] = ((uint32_t)(int)rintf(y) + 0x808080u) ^ 0x808080u;
            }
            // byte i of the four numbers is digit i
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                const uint32_t sel = 0x0c0c0000u | (uint32_t)(4 + i) << 8 | (uint32_t)i;
                const uint32_t p01 = __builtin_amdgcn_perm(v[1], v[0], sel);
                const uint32_t p23 = __builtin_amdgcn_perm(v[3], v[2], sel);
                qd[i][s][w] = (int)(p01 | p23 << 16);
            }
        }
    return isbad ? __builtin_nanf("") : a.scale / up * (X ? 1.0f : 1.44269504088896341f);
}

// Integer scores of a tile for one column tile: S[4 u + v] is token 4 u + v of
// page kg.  kf(u, s): K fragment of sub-tile u, dimensions 64 s ..
template <int NS, class KF>
__device__ __forceinline__ void a8_scores(const KF& kf, const v4i (&qd)[3][NS], float (&S)[16]) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        v4i c2 = {0, 0, 0, 0}, c1 = {0, 0, 0, 0}, c0 = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const v4i kv = __builtin_bit_cast(v4i, kf(u, s));
            c2 = __builtin_amdgcn_mfma_i32_16x16x64_i8(kv, qd[2][s], c2, 0, 0, 0);
            c1 = __builtin_amdgcn_mfma_i32_16x16x64_i8(kv, qd[1][s], c1, 0, 0, 0);
            c0 = __builtin_amdgcn_mfma_i32_16x16x64_i8(kv, qd[0][s], c0, 0, 0, 0);
        }
        // |c1| 256 + |c0| < 2^30
#pragma unroll
        for (int v = 0; v < 4; ++v) S[4 * u + v] = fmaf((float)c2[v], 65536.0f, (float)(c1[v] * 256 + c0[v]));
    }
}

// One column's running softmax.  L, lo: the tokens it sees; m: its reference, within
// 4 below the largest score (base 2) so far; l: the sum of 2^(score - m).  e: the PV
// operand of a token is 2^(score - m) vs 2^(A8_UP - e), vs its page's V scale, e a whole
// number that keeps the largest such operand between 2^10 and 2^15, at binary16's upper
// end.  What a page contributes decides, not its V scale alone: a large scale that meets
// no weight, or a heavy page of small values, takes no bits from the others.
#define A8_UP 137              // 10, and the 127 by which a8_exponent is biased
struct A8Col {
    float f, slope, m, l, e;
    int L, lo;
};
__device__ __forceinline__ void a8_reset(A8Col& c) {
    c.m = -__builtin_inff();
    c.l = 0.0f;
    c.e = -400.0f;
}
__device__ __forceinline__ int a8_exponent(float x) { return (int)(__float_as_uint(x) >> 23 & 255); }

// From the scores of N column tiles (integers, times k.f and the K scale) to their
// weights, each times its page's V scale, as two binary16 parts; o, what was summed
// before, is brought to the new references where they move.  EDGE: some column does not
// see the whole tile, or the scores are capped, biased or windowed (X).  ks, vs: the
// scales of the lane's page; pt: its first token.
template <bool X, bool EDGE, int N, int ND>
__device__ __forceinline__ void a8_weights(const lgx_attn8_args& a, float (*S)[16], A8Col* k, float ks, float vs, int pt, v8h (*ph)[2],
                                           v8h (*pl)[2], v4f (*o)[ND]) {
    static_assert(EDGE || !X, "other scores are formed ahead of the maximum");
    constexpr float kLog2e = 1.44269504088896341f;
    const float inf = __builtin_inff();
    const int ve = a8_exponent(vs);
    float fk[N], mt[N], top[N];
    bool page[N], moves = false;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        fk[n] = k[n].f * ks;
        page[n] = true;
        if (EDGE) {
            const int hi = k[n].L - pt, lo = k[n].lo - pt;   // what the column sees of the page
#pragma unroll
            for (int e = 0; e < 16; ++e) S[n][e] *= fk[n];
            if constexpr (X) {
                if (a.softcap > 0.0f) {
                    const float inv = 1.0f / a.softcap;
#pragma unroll
                    for (int e = 0; e < 16; ++e) S[n][e] = a.softcap * a8_tanh(S[n][e] * inv);
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) S[n][e] = (S[n][e] - k[n].slope * (float)(hi - 1 - e)) * kLog2e;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (e >= hi || e < lo) S[n][e] = -inf;
            // a page that the column does not see may hold anything
            page[n] = hi > 0 && lo < LGX_PAGE;
        }
        float m = fmaxf(fmaxf(S[n][0], S[n][1]), S[n][2]);
#pragma unroll
        for (int e = 3; e < 15; e += 2) m = fmaxf(fmaxf(m, S[n][e]), S[n][e + 1]);
        m = fmaxf(m, S[n][15]);
        if (!EDGE) m *= fk[n];                    // scales are not negative
        // the page's largest contribution, -inf where the column sees nothing of it
        top[n] = col_max(m + (float)ve);
        mt[n] = col_max(m);
        // the references move when a maximum passes theirs by more than 2^4: most
        // tiles leave what was summed as it is
        moves = moves || mt[n] > k[n].m + 4.0f || top[n] > k[n].m + k[n].e + 4.0f;
    }
    if (__builtin_amdgcn_ballot_w64(moves)) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const float mn = mt[n] > k[n].m + 4.0f ? mt[n] : k[n].m;
            const bool none = mn == -inf;         // nothing seen yet
            const float d = none ? 0.0f : k[n].m - mn;
            const float rel = fmaxf(none ? -inf : top[n] - mn, -400.0f);   // a NaN falls away
            const float en = mn != k[n].m || rel > k[n].e + 4.0f ? floorf(fmaxf(rel, k[n].e + d)) : k[n].e;
            const float down = __builtin_amdgcn_exp2f(d + (k[n].e - en));
#pragma unroll
            for (int i = 0; i < ND; ++i) o[n][i] *= down;
            k[n].l *= __builtin_amdgcn_exp2f(d);
            k[n].m = mn;
            k[n].e = en;
        }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const float off = k[n].m == -inf ? 0.0f : -k[n].m;
        // below 2^128: a larger factor's weights are under 2^-113 of the row's largest
        const float r = page[n] ? ldexpf(vs, min(A8_UP - (int)k[n].e, 2 * 127 - ve)) : 0.0f;
        float ps = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            S[n][e] = __builtin_amdgcn_exp2f(EDGE ? S[n][e] + off : fmaf(S[n][e], fk[n], off));
            ps += S[n][e];
            S[n][e] *= r;
        }
        k[n].l += ps;
        uint32_t hw[8], lw[8];
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
            // both parts rounded to nearest: the sum of the weights and that of their
            // roundings then differ to either side, also where the second part is
            // subnormal (cut, the results were 7.5e-8 low, and by 2^-17 of the weights
            // of 131072 tokens behind one that weighs as much as they together)
            const uint32_t h = f16_pair(S[n][e], S[n][e + 1]);
            hw[e >> 1] = h;
            lw[e >> 1] = f16_pair(minus_half<0>(S[n][e], h), minus_half<1>(S[n][e + 1], h));
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            ph[n][i] = as_v8h(make_uint4(hw[4 * i], hw[4 * i + 1], hw[4 * i + 2], hw[4 * i + 3]));
            pl[n][i] = as_v8h(make_uint4(lw[4 * i], lw[4 * i + 1], lw[4 * i + 2], lw[4 * i + 3]));
        }
    }
}
struct A8Edge { static constexpr bool value = true; };
struct A8Whole { static constexpr bool value = false; };

// Sixteen quants (16 dimensions of a K row, 16 tokens of a V dimension) as two
// binary16 operands.
__device__ __forceinline__ void i8_to_v8h(const uint4& v, uint4& h0, uint4& h1) {
    i8_to_f16(v.x, h0.x, h0.y);
    i8_to_f16(v.y, h0.z, h0.w);
    i8_to_f16(v.z, h1.x, h1.y);
    i8_to_f16(v.w, h1.z, h1.w);
}
// o += V^T . P^T for N column tiles; vf(i, h0, h1): V operands of dimensions 16 i ..
// A tile's products are summed from zero and joined to o on the VALU.  The matrix unit
// adds them in groups of eight and rounds its sum after each: added to o itself, the
// second parts of the weights fall below half a step of it as o grows (equal weights of
// 65536 tokens: 3.2e-5 off; a sink among 131072: 2.5e-5, now 1.2e-5 of repeated pages'
// own roundings).  It costs 3 % of prompts (8 x 512 rows at 4000 tokens 445 against 434
// us) and nothing where memory bounds.
template <int ND, int N, class VF>
__device__ __forceinline__ void a8_pv(const VF& vf, const v8h (&ph)[N][2], const v8h (&pl)[N][2], v4f (&o)[N][ND]) {
#pragma unroll
    for (int i = 0; i < ND; ++i) {
        uint4 h0, h1;
        vf(i, h0, h1);
        v4f t[N];
#pragma unroll
        for (int n = 0; n < N; ++n) t[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_v8h(h0), pl[n][0], (v4f){0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
        for (int n = 0; n < N; ++n) t[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_v8h(h0), ph[n][0], t[n], 0, 0, 0);
#pragma unroll
        for (int n = 0; n < N; ++n) t[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_v8h(h1), pl[n][1], t[n], 0, 0, 0);
#pragma unroll
        for (int n = 0; n < N; ++n) t[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_v8h(h1), ph[n][1], t[n], 0, 0, 0);
#pragma unroll
        for (int n = 0; n < N; ++n) o[n][i] += t[n];
    }
}

// A column's result, or its split's (divided by the split's own sum of weights, so that
// it is no larger than V's values); c: the column, NC columns per block.
template <int NC, int ND>
__device__ __forceinline__ void a8_store(const lgx_attn8_args& a, const A8Block& k, int64_t orow, int c, const A8Col& x, int kg,
                                         const v4f (&o)[ND]) {
    constexpr int D = 16 * ND;
    const bool part = k.ns > 1;
    const int64_t at = part ? ((int64_t)k.pos * a.hkv + k.g) * NC + c - k.c0 : orow;
    const int unit = (int)x.e - A8_UP;
    // NaN sums stay NaN; nothing seen gives zeros
    const float s = x.l == 0.0f ? 0.0f : 1.0f / x.l;
    float* dst = (part ? a.part : a.out) + at * D;
#pragma unroll
    for (int i = 0; i < ND; ++i)
        *(float4*)(dst + 16 * i + 4 * kg) =
            make_float4(ldexpf(o[i][0] * s, unit), ldexpf(o[i][1] * s, unit), ldexpf(o[i][2] * s, unit), ldexpf(o[i][3] * s, unit));
    if (part && kg == 0) *(float2*)(a.ml + 2 * at) = make_float2(x.m, x.l);
}

// 16 NT columns per workgroup (a decode row's heads): its four waves take the tiles
// in turn, K and V straight into registers: the next tile's K is in flight
// from the end of the scores on, its V from the end of the PV product; at the end
// the waves' results are joined in LDS.  One column tile is bound by memory: 16
// sequences of 32768 tokens, 12/2 heads of 128, 268 MB, in 51 us (5.2 TB/s), 51 with
// the loads alone; 64 of 256 to 4096 tokens, 28/4 heads, 145 MB, in 39, as with the
// loads alone (the longest one's workgroup takes what one compute unit can load), and 53
// with capped scores.  Eight waves per workgroup load no faster there and wait a fifth
// longer for one sequence of 8191.  Two column tiles are bound by the VALU and the matrix
// units in turn: 8 x 64 rows at 2000 tokens 43 us, the operations alone 13.
template <int D, int NT, bool X>
__device__ __forceinline__ void attn8_narrow_body(const lgx_attn8_args& a) {
    constexpr int WT = 4, NS = D / 64, ND = D / 16;
    __shared__ v4f o_s[WT / 2 * NT * ND * 64];
    __shared__ float ml_s[WT / 2 * NT * 3 * 64];
    const int lane = threadIdx.x & 63, col = lane & 15, kg = lane >> 4;
    const int wt = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    A8<16 * NT, X> w{a, {}};
    if (!w.place()) return;                       // uniform
    const int b = w.k.b, g = w.k.g, G = w.k.G;
    auto orow = [&](int c) { return ((int64_t)b * a.P + c / G) * a.hq + g * G + c % G; };
    const int32_t* ptab = a.page_table + (int64_t)b * a.maxp;
    struct Pages {
        int k, v;
    };
    auto pages = [&](int t) {
        Pages p;
        p.k = ptab[min(4 * t + (col >> 2), a.maxp - 1)];
        p.v = ptab[min(4 * t + kg, a.maxp - 1)];
        return p;
    };
    auto block = [&](int p) { return (int64_t)min(max(p, 0), a.num_pages - 1) * a.hkv + g; };
    uint4 kw[4][NS], vw[ND];
    auto load_k = [&](const Pages& p) __attribute__((always_inline)) {
        const int8_t* kp = a.k + (block(p.k) * LGX_PAGE + (col & 3)) * D + 16 * kg;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int s = 0; s < NS; ++s) kw[u][s] = *(const uint4*)(kp + 4 * u * D + 64 * s);
    };
    auto load_v = [&](const Pages& p) __attribute__((always_inline)) {
        const int8_t* vp = a.v + (block(p.v) * D + col) * LGX_PAGE;
#pragma unroll
        for (int i = 0; i < ND; ++i) vw[i] = *(const uint4*)(vp + 16 * i * LGX_PAGE);
    };
    int t = w.k.tb0 + wt;
    const int end = w.k.tb1;
    // Loads are issued whether or not there is such a tile (the wave's last one's
    // again, from the cache): a conditional load's registers would be copied, and so
    // waited for, where the branches meet.
    const int mine = end - 1 - t >= 0 ? t + (end - 1 - t) / WT * WT : t;   // the wave's last tile
    // the query and the first pages in one memory round; its digits while K and V
    // are on their way
    float x[NT][NS][16];
    Pages p = pages(t);
#pragma unroll
    for (int n = 0; n < NT; ++n) a8_query_load<NS>(a.q + orow(min(w.k.c0 + 16 * n + col, w.k.ncols - 1)) * D + 16 * kg, x[n]);
    __builtin_amdgcn_sched_barrier(0);
    load_k(p);
    float ks = a.ks[block(p.v)], vs = a.vs[block(p.v)];
    load_v(p);
    p = pages(min(t + WT, mine));
    __builtin_amdgcn_sched_barrier(0);
    v4f o[NT][ND];
    A8Col k[NT];
    // two column tiles' digits do not fit beside the rest: they stay in LDS, the
    // same for all waves, and pass through registers one column tile at a time
    v4i qd[3][NS];
    __shared__ v4i q_s[NT > 1 ? NT * 3 * NS * 64 : 1];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < ND; ++i) o[n][i] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
        const int cc = min(w.k.c0 + 16 * n + col, w.k.ncols - 1);   // columns past the last repeat it
        a8_reset(k[n]);
        k[n].L = w.last(cc);
        k[n].lo = w.first(cc);
        k[n].slope = X && a.slopes ? a.slopes[g * G + cc % G] : 0.0f;
        k[n].f = a8_query<NS, X>(a, x[n], qd);
        if (NT > 1 && wt == n) {
#pragma unroll
            for (int i = 0; i < 3 * NS; ++i) q_s[(n * 3 * NS + i) * 64 + lane] = qd[i / NS][i % NS];
        }
    }
    if (NT > 1) __syncthreads();
    auto tile = [&](auto form) __attribute__((always_inline)) {
        constexpr bool edge = decltype(form)::value;
        const int pt = t * LGX_A8_TILE + 16 * kg;
        const float ksn = ks, vsn = vs;
        const Pages pn = p;
        v8h ph[NT][2], pl[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float S[1][16];
            if (NT > 1) {
                int at = lane;
                asm volatile("" : "+v"(at));      // read here, not once ahead of the loop
#pragma unroll
                for (int i = 0; i < 3 * NS; ++i) qd[i / NS][i % NS] = q_s[(n * 3 * NS + i) * 64 + at];
            }
            a8_scores<NS>([&](int u, int s) { return kw[u][s]; }, qd, S[0]);
            if (n == NT - 1) {
                load_k(pn);
                ks = a.ks[block(pn.v)];
                vs = a.vs[block(pn.v)];
                p = pages(min(t + 2 * WT, mine));
            }
            a8_weights<X, edge, 1, ND>(a, S, k + n, ksn, vsn, pt, ph + n, pl + n, o + n);
        }
        a8_pv<ND, NT>([&](int i, uint4& h0, uint4& h1) { i8_to_v8h(vw[i], h0, h1); }, ph, pl, o);
        load_v(pn);
    };
    // the tiles that every column sees whole, then the others
    if constexpr (!X) {
#pragma unroll 1
        for (const int whole = min(end, w.last(w.k.c0) / LGX_A8_TILE); t < whole; t += WT) tile(A8Whole());
    }
#pragma unroll 1
    for (; t < end; t += WT) tile(A8Edge());
#pragma unroll
    for (int n = 0; n < NT; ++n) k[n].l = col_sum(k[n].l);
    // join the waves, halving their number
#pragma unroll
    for (int h = WT / 2; h; h >>= 1) {
        const int at = wt % h * NT;
        if (wt >= h && wt < 2 * h) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                ml_s[((at + n) * 3 + 0) * 64 + lane] = k[n].m;
                ml_s[((at + n) * 3 + 1) * 64 + lane] = k[n].l;
                ml_s[((at + n) * 3 + 2) * 64 + lane] = k[n].e;
#pragma unroll
                for (int i = 0; i < ND; ++i) o_s[((at + n) * ND + i) * 64 + lane] = o[n][i];
            }
        }
        __syncthreads();
        if (wt < h) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float mo = ml_s[((at + n) * 3 + 0) * 64 + lane], lo = ml_s[((at + n) * 3 + 1) * 64 + lane];
                const float eo = ml_s[((at + n) * 3 + 2) * 64 + lane];
                const float mn = fmaxf(k[n].m, mo);
                // a wave that has seen nothing: -inf, so weights of 0
                const float d0 = k[n].m == -__builtin_inff() ? k[n].m : k[n].m - mn, d1 = mo == -__builtin_inff() ? mo : mo - mn;
                const float en = fmaxf(floorf(fmaxf(k[n].e + d0, eo + d1)), -400.0f);
                const float w0 = __builtin_amdgcn_exp2f(d0), w1 = __builtin_amdgcn_exp2f(d1);
                const float u0 = __builtin_amdgcn_exp2f(d0 + (k[n].e - en)), u1 = __builtin_amdgcn_exp2f(d1 + (eo - en));
                k[n].l = k[n].l * w0 + lo * w1;
                k[n].m = mn;
                k[n].e = en;
#pragma unroll
                for (int i = 0; i < ND; ++i) o[n][i] = o[n][i] * u0 + o_s[((at + n) * ND + i) * 64 + lane] * u1;
            }
        }
        __syncthreads();
    }
    if (wt) return;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int c = w.k.c0 + 16 * n + col;
        if (c < w.k.ncols) a8_store<16 * NT, ND>(a, w.k, orow(c), c, k[n], kg, o[n]);
    }
}

// The query of a lane's column as two binary16 parts per operand (22 bits under the
// row's largest magnitude, which a power of two brings to 2^14 .. 2^15), dimensions
// 64 s + 16 kg + 8 h .. in step 2 s + h.
template <int D, bool X>
__device__ __forceinline__ float a8_query16(const lgx_attn8_args& a, const float* qr, v8h (&qh)[2][D / 32]) {
    constexpr int NH = D / 32;
    float x[NH][8], am = 0.0f;
    bool bad = false;
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
            const float4 v = *(const float4*)(qr + 64 * (h >> 1) + 8 * (h & 1) + e);
            x[h][e] = v.x;
            x[h][e + 1] = v.y;
            x[h][e + 2] = v.z;
            x[h][e + 3] = v.w;
        }
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            am = fmaxf(am, fabsf(x[h][e]));
            bad = bad || !(fabsf(x[h][e]) < __builtin_inff());
        }
    am = col_max(am);
    const bool isbad = col_max(bad ? 1.0f : 0.0f) != 0.0f;
    const float up = __uint_as_float(__float_as_uint(fminf(32768.0f / am, 0x1p122f)) & 0x7f800000u);
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float y = isbad ? 0.0f : x[h][e] * up;
            qh[0][h][e] = (_Float16)y;
            qh[1][h][e] = (_Float16)(y - (float)qh[0][h][e]);
        }
    return isbad ? __builtin_nanf("") : a.scale / up * (X ? 1.0f : 1.44269504088896341f);
}

// Many columns (prefill): 64 NT per workgroup, 16 NT per wave.  Every tile is converted to
// binary16 once for all of them: each wave brings a quarter of its quants into LDS
// (two waves K, two V; a direct load brings one 1 KiB fragment in the order of the
// lanes), a tile ahead, and then turns them into operands in one of two LDS buffers
// while the other's tile is in use.  With K in binary16 the scores need no joining of
// digits: two products, one accumulator.  Bound by the matrix units and the VALU in
// turn: 8 x 512 rows at 4000 tokens, 28/4 heads of 128, in 434 to 457 us by the card and
// its clock (513 in a profiler's few dispatches, at 1.97 GHz), 0.48 to 0.51 PFLOP/s of the
// formula's work, twice that executed (q and the weights in two parts; a large binary16
// product reaches 1.1 to 1.2 here); matrix units busy for 0.41 of the cycles, the VALU for
// 0.53.  What brought it down from 783 us: K and V through LDS
// (565), no masks where all rows see a tile, operands converted once and no load waited
// for where branches meet (520), a softmax reference that seldom moves (480).  64 columns
// per workgroup (16 per wave) took as long as 16 or longer.  The same rows with a cap of
// 30 take 855 us, with a window of 1000 tokens 170.
template <int D, int NT, bool X>
__device__ __forceinline__ void attn8_wide_body(const lgx_attn8_args& a) {
    constexpr int NS = D / 64, NH = D / 32, ND = D / 16, NF = 4 * NS + ND, FW = NF / 4;
    static_assert(4 * NS == ND, "waves 0 and 1 bring K, 2 and 3 bring V");
    __shared__ __align__(16) uint4 f_s[2][2 * NF * 64], raw_s[NF * 64];
    const int lane = threadIdx.x & 63, col = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    A8<64 * NT, X> w{a, {}};
    if (!w.place()) return;                       // uniform
    const int b = w.k.b, g = w.k.g, G = w.k.G;
    const int wcol = w.k.c0 + wave * 16 * NT;     // the wave's first column
    const bool any = wcol < w.k.ncols;            // uniform per wave
    const int wlast = min(wcol + 16 * NT, w.k.ncols) - 1;
    const int wend = any ? w.last(wlast) : 0, wbeg = any ? w.first(wcol) : 0;
    const int32_t* ptab = a.page_table + (int64_t)b * a.maxp;
    const int end = w.k.tb1;
    // Loads are issued whether or not there is such a tile (the last one's again,
    // from the cache): a conditional load's register would be copied, and so waited
    // for, where the branches meet.
    auto page_ld = [&](int t) { return ptab[min(4 * max(min(t, end - 1), 0) + (wave < 2 ? col >> 2 : kg), a.maxp - 1)]; };
    auto page_sc = [&](int t) { return ptab[min(4 * max(min(t, end - 1), 0) + kg, a.maxp - 1)]; };
    auto block = [&](int p) { return (int64_t)min(max(p, 0), a.num_pages - 1) * a.hkv + g; };
    uint4* const raw = raw_s + wave * FW * 64;
    // the wave's fragments of a tile, p its page
    auto load = [&](int p) __attribute__((always_inline)) {
        const int64_t blk = block(p);
        const int8_t* src = wave < 2 ? a.k + (blk * LGX_PAGE + (col & 3)) * D + 16 * kg : a.v + (blk * D + col) * LGX_PAGE;
#pragma unroll
        for (int j = 0; j < FW; ++j) {
            const int f = (wave & 1) * FW + j;
            load_lds_16(src + (wave < 2 ? 4 * (f / NS) * D + 64 * (f % NS) : 16 * f * LGX_PAGE), (lds_void*)(raw + j * 64));
        }
    };
    // them as operands: 2 f and 2 f + 1 of fragment f
    auto convert = [&](uint4* buf) __attribute__((always_inline)) {
        uint4* dst = buf + wave * 2 * FW * 64 + lane;
#pragma unroll
        for (int j = 0; j < FW; ++j) {
            uint4 h0, h1;
            i8_to_v8h(raw[j * 64 + lane], h0, h1);
            dst[2 * j * 64] = h0;
            dst[(2 * j + 1) * 64] = h1;
        }
    };
    load(page_ld(w.k.tb0));
    int pl_ = page_ld(w.k.tb0 + 1), ps_ = page_sc(w.k.tb0 + 1);
    float ks, vs;
    {
        const int64_t sb = block(page_sc(w.k.tb0));
        ks = a.ks[sb];
        vs = a.vs[sb];
    }
    A8Col k[NT];
    v8h qh[NT][2][NH];
    auto orow = [&](int c) { return ((int64_t)b * a.P + c / G) * a.hq + g * G + c % G; };
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int c = wcol + 16 * n + col, cc = min(c, w.k.ncols - 1);
        a8_reset(k[n]);
        k[n].L = w.last(cc);                      // columns past the last repeat it
        k[n].lo = w.first(cc);
        k[n].slope = X && a.slopes ? a.slopes[g * G + cc % G] : 0.0f;
        k[n].f = a8_query16<D, X>(a, a.q + orow(cc) * D + 16 * kg, qh[n]);
    }
    v4f o[NT][ND];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < ND; ++i) o[n][i] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
    auto tile = [&](int t, auto form) __attribute__((always_inline)) {
        constexpr bool edge = decltype(form)::value;
        const int cur = (t - w.k.tb0) & 1;
        publish_lds_loads();                      // tile t is whole, tile t - 1 read, t + 1's quants landed
        convert(f_s[cur ^ 1]);
        __builtin_amdgcn_sched_barrier(0);
        load(pl_);
        pl_ = page_ld(t + 3);
        const float ksn = ks, vsn = vs;
        const int64_t sb = block(ps_);
        ks = a.ks[sb];
        vs = a.vs[sb];
        ps_ = page_sc(t + 2);
        __builtin_amdgcn_sched_barrier(0);
        const int t0 = t * LGX_A8_TILE, pt = t0 + 16 * kg;
        if (!any || (edge && (t0 >= wend || t0 + LGX_A8_TILE <= wbeg))) return;   // uniform per wave
        const uint4* fr = f_s[cur] + lane;
        float S[NT][16];
        {
            // fragments PF ahead of their products: an LDS read takes as long as
            // two fragments' products
            constexpr int PF = 3;
            v8h kf[4 * NH];
            v4f acc[4][NT];
#pragma unroll
            for (int i = 0; i < PF; ++i) kf[i] = as_v8h(fr[i * 64]);
#pragma unroll
            for (int i = 0; i < 4 * NH; ++i) {
                const int u = i / NH, h = i % NH;
                if (i + PF < 4 * NH) kf[i + PF] = as_v8h(fr[(i + PF) * 64]);
#pragma unroll
                for (int part = 1; part >= 0; --part)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        acc[u][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            kf[i], qh[n][part][h], h == 0 && part == 1 ? (v4f){0.0f, 0.0f, 0.0f, 0.0f} : acc[u][n], 0, 0, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x100, PF, 0);
#pragma unroll
            for (int i = 0; i < 4 * NH; ++i) {
                if (i + PF < 4 * NH) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, 2 * NT, 0);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 16; ++e) S[n][e] = acc[e >> 2][n][e & 3];
        }
        v8h ph[NT][2], pl[NT][2];
        a8_weights<X, edge, NT, ND>(a, S, k, ksn, vsn, pt, ph, pl, o);
        {
            constexpr int PF = 3;
            const uint4* vr = fr + 2 * 4 * NS * 64;
            v8h vf[2 * ND];
            v4f t[ND][NT];
#pragma unroll
            for (int i = 0; i < PF; ++i) vf[i] = as_v8h(vr[i * 64]);
#pragma unroll
            for (int i = 0; i < 2 * ND; ++i) {
                if (i + PF < 2 * ND) vf[i + PF] = as_v8h(vr[(i + PF) * 64]);
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    t[i / 2][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[i], pl[n][i & 1],
                                                                         i & 1 ? t[i / 2][n] : (v4f){0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    t[i / 2][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[i], ph[n][i & 1], t[i / 2][n], 0, 0, 0);
                // a tile's sum from zero (a8_pv), of dimensions whose products have ended
                if (i >= 3 && i & 1) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) o[n][i / 2 - 1] += t[i / 2 - 1][n];
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) o[n][ND - 1] += t[ND - 1][n];
        }
    };
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    convert(f_s[0]);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the quants are read before the next overwrite them
    load(pl_);
    pl_ = page_ld(w.k.tb0 + 2);
    // the tiles that every column of the workgroup sees whole, then the others
    int t = w.k.tb0;
    if constexpr (!X) {
#pragma unroll 1
        for (const int whole = min(end, w.last(w.k.c0) / LGX_A8_TILE); t < whole; ++t) tile(t, A8Whole());
    }
#pragma unroll 1
    for (; t < end; ++t) tile(t, A8Edge());
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // no load into LDS outlives the wave
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int c = wcol + 16 * n + col;
        k[n].l = col_sum(k[n].l);
        if (c < w.k.ncols) a8_store<64 * NT, ND>(a, w.k, orow(c), c, k[n], kg, o[n]);
    }
}

// Joins the splits of one (row, head): D / 4 threads per split, TH / (D / 4) splits at
// a time.  TH: 256 threads, or a wave where there are many rows and so few splits
// each.  Three memory rounds behind a launch: 4 us; a thread per dimension, one split
// after the other, took 10 us for 32 splits and 36 for 125.
template <int D, int TH>
__device__ __forceinline__ void attn8_join_body(const lgx_attn8_args& a) {
    constexpr int Q = D / 4, NG = TH / Q, NW = TH / 64;
    __shared__ v4f o_s[NW > 1 ? NG * Q : 1];
    __shared__ float ml_s[2 * NW];
    const int tid = threadIdx.x % TH;
    const int64_t rh = (int64_t)blockIdx.x * (256 / TH) + threadIdx.x / TH;
    if (rh >= (int64_t)a.rows * a.hq) return;     // uniform per wave
    const int row = (int)(rh / a.hq), h = (int)(rh - (int64_t)row * a.hq), b = row / a.P, j = row - b * a.P;
    if (a.n_new && j >= a.n_new[b]) return;
    const int G = a.hq / a.hkv, g = h / G, c = j * G + h - g * G, cb = c / a.cols;
    const int u = b * a.ncb + cb, pos = a.plan[2 * u], ns = a.plan[2 * u + 1];
    if (ns < 2) return;
    auto at = [&](int s) { return ((int64_t)(pos + s) * a.hkv + g) * a.cols + c - cb * a.cols; };
    float m = -__builtin_inff(), l = 0.0f;
    for (int s = tid; s < ns; s += TH) m = fmaxf(m, a.ml[2 * at(s)]);
    m = wave_max(m);
    if (NW > 1) {
        if ((tid & 63) == 0) ml_s[tid >> 6] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NW; ++i) m = fmaxf(m, ml_s[i]);
    }
    // a split's sum of weights by the common maximum; an empty one's own is -inf
    auto weight = [&](int64_t i) {
        const float2 x = *(const float2*)(a.ml + 2 * i);
        return (x.x == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(x.x - m)) * x.y;
    };
    for (int s = tid; s < ns; s += TH) l += weight(at(s));
#pragma unroll
    for (int s = 32; s; s >>= 1) l += shfl_xor_f(l, s);
    if (NW > 1) {
        if ((tid & 63) == 0) ml_s[NW + (tid >> 6)] = l;
        __syncthreads();
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < NW; ++i) l += ml_s[NW + i];
    }
    const float r = l == 0.0f ? 0.0f : 1.0f / l;  // ahead of the sum, which then stays within V's values
    const int q = tid % Q, sg = tid / Q;
    v4f o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int s = sg; s < ns; s += NG) {
        const int64_t i = at(s);
        o += *((const v4f*)(a.part + i * D) + q) * (weight(i) * r);
    }
    if (NW > 1) {
        o_s[tid] = o;
        __syncthreads();
        if (tid >= Q) return;
#pragma unroll
        for (int i = 1; i < NG; ++i) o += o_s[tid + i * Q];
    } else {
#pragma unroll
        for (int s = Q; s < 64; s <<= 1)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += shfl_xor_f(o[e], s);
        if (tid >= Q) return;
    }
    *((v4f*)(a.out + rh * D) + q) = o;
}
extern "C" __global__ __launch_bounds__(256) void lgx_k_attn8_join_d64(const lgx_attn8_args a) { attn8_join_body<64, 256>(a); }
extern "C" __global__ __launch_bounds__(256) void lgx_k_attn8_join_d128(const lgx_attn8_args a) { attn8_join_body<128, 256>(a); }
extern "C" __global__ __launch_bounds__(256) void lgx_k_attn8_joinw_d64(const lgx_attn8_args a) { attn8_join_body<64, 64>(a); }
extern "C" __global__ __launch_bounds__(256) void lgx_k_attn8_joinw_d128(const lgx_attn8_args a) { attn8_join_body<128, 64>(a); }

#define LGX_A8_KERNELS(D, C, BODY, NT)                                                                                 \
    extern "C" __global__ __launch_bounds__(256, 2) void lgx_k_attn8_d##D##_c##C(const lgx_attn8_args a) {             \
        BODY<D, NT, false>(a);                                                                                         \
    }                                                                                                                  \
    extern "C" __global__ __launch_bounds__(256, 2) void lgx_k_attn8x_d##D##_c##C(const lgx_attn8_args a) {            \
        BODY<D, NT, true>(a);                                                                                          \
    }
LGX_A8_KERNELS(64, 16, attn8_narrow_body, 1)
LGX_A8_KERNELS(64, 32, attn8_narrow_body, 2)
LGX_A8_KERNELS(64, 128, attn8_wide_body, 2)
LGX_A8_KERNELS(128, 16, attn8_narrow_body, 1)
LGX_A8_KERNELS(128, 32, attn8_narrow_body, 2)
LGX_A8_KERNELS(128, 128, attn8_wide_body, 2)
