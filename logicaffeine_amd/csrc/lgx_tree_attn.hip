// lgx_tree_attn.hip -- attention of a tree of drafted tokens over the paged binary16
// cache.
#include "lgx_device.h"

// ---------------------------------------------------------------------------
// Sequence b has sl cached tokens and n nodes behind them, token sl + i being node i.  Node
// j stands at position sl + depth[j] and sees the cached tokens (within the window,
// if there is one) and the nodes of its mask.  The (node, query head) pairs of one
// KV head are the columns of the products, 16 to a matrix instruction; a tile is 64
// tokens, four pages.
//   scores   S^T[token][column] = K . Q^T on v_mfma_f32_16x16x32_f16.  q is scaled by a
//            power of two that brings its row's largest value to 2^14 .. 2^15 and is
//            the sum of two binary16 numbers, 22 bits (2^-25 of the row's largest where
//            it is far below): two products.
//   softmax  running maximum and sum per column, in base 2, binary32.
//   PV       O^T[dim][column] += V^T . P^T on the same instruction: a weight times 2^10 is
//            the sum of two binary16 numbers, 22 bits, or to 2^-35 of the largest where it
//            is smaller.  The matrix unit sums a tile, the VALU the tiles.
// So the results are as exact as binary32 products would be, 1e-7 to 4e-7 of the 64-bit
// result: a draft is accepted by what a decode step would have said, not by its rounding.
//
// Lane (column, kg) gets the scores of tokens 16 u + 4 kg + 0..3 of sub-tile u, and V's
// transposing LDS loads give lane (dimension, kg) the same four tokens of it: two
// sub-tiles' weights are the 8 values of a PV operand as they stand.
//
// A token that a column does not see has weight 0 and may hold anything: K's score is
// replaced; V rows behind the last node are cleared; and an infinity or a NaN among the
// others, which 0 would not hide, leaves a result that is not finite, upon which the
// column is done over token by token (tree_column).
//
// A workgroup has 64 columns, 16 per wave, and passes tiles of K and V through LDS, where all
// four waves read them.  Measured against it (128 dimensions, 28 heads of 4):
//   16 columns per workgroup, the waves sharing the tiles, for up to 16 columns: one token
//     of 64 sequences of up to 4000 tokens 75 against 70 us, of one of 8000 15.8 against
//     14.1: a workgroup's waves have more loads in flight where all of them load one tile.
//   128 columns, 32 per wave, half the LDS reads per product: 64 nodes over 8000 tokens
//     36.8 against 34.2 us, 100 nodes of 8 sequences of 1000 55 against 44; only 200 nodes
//     of 2 sequences of 5200 gain (113 against 136), where 22 blocks read the same K and V.
// What bounds it: few nodes, the cache's bytes (one token of 64 sequences: 4.2 TB/s of
// the 4.7 that a copy reaches); many, that a wave's LDS reads, products and softmax follow
// each other and the SIMD's other wave does not fill the gaps: of the compute units' busy
// cycles the matrix unit is busy in 31 to 32 %, VALU instructions are under way in 42 to 48
// % (64 nodes over 8000 tokens, 32 x 16 over up to 4096, 8 x 100 over 1000; no LDS bank
// conflicts), and with capped scores in 16 and 57 % (9 x 201 over 1500); short calls, the
// launch and the splits' join.
// ---------------------------------------------------------------------------
typedef __attribute__((address_space(3))) uint16_t lds_u16;
typedef __attribute__((address_space(4))) const int32_t const_i32;

#define TREE_UP 10             // weights as operands: times 2^10

// What a workgroup works on: a sequence, a KV head, a block of columns, a run of tiles.
struct Tree {
    const lgx_tree_attn_args& a;
    int b, g, G, c0, ncols, sl, n;
    int tb0, tb1;              // tiles
    int unit;                  // b * ncb + column block
    int pos, ns;               // number of the split among all, and splits of the column block

    __device__ __forceinline__ int nodes(int b) const { return a.n_nodes ? min(max(a.n_nodes[b], 0), a.N) : a.N; }
    __device__ __forceinline__ int length(int b) const { return min(max(a.seq_len[b], 0), a.maxlen); }
    // first and last + 1 tile that a sequence's nodes can see (depths are not negative)
    __device__ __forceinline__ int2 tiles(int sl, int n) const {
        const int first = a.window ? max((int)max((int64_t)sl - a.window + 1, (int64_t)0), 0) : 0;
        return make_int2(first / LGX_TREE_TILE, (sl + n + LGX_TREE_TILE - 1) / LGX_TREE_TILE);
    }
    // Column blocks of n nodes.
    __device__ __forceinline__ int blocks(int n) const { return (n * G + LGX_TREE_COLS - 1) / LGX_TREE_COLS; }
    // Workgroup ids go round-robin over the 8 XCDs, each with an L2 of its own: consecutive
    // places, whose column blocks share K and V, go to one XCD.  -1: none of the `all`.
    static __device__ __forceinline__ int place_of(int id, int all) {
        const int each = (all + 7) >> 3, at = (id & 7) * each + (id >> 3);
        return id >> 3 < each && at < all ? at : -1;
    }
    // false: nothing to do.  Places are in order of (sequence, run of tiles, KV head, column
    // block).  With a.per all sequences' tiles go in about equal runs to the workgroups:
    // every wave computes the run length from all lengths (four sequences per lane),
    // nearly the least with which all (run, column block)s fit into a.per, then finds the
    // sequence and the run of its place in the sums over the sequences.
    __device__ __forceinline__ bool place() {
        G = a.hq / a.hkv;
        int s = 0, run = 0, cb;
        const int id = __builtin_amdgcn_readfirstlane(blockIdx.x);
        if (a.per) {
            const int lane = threadIdx.x & 63;
            int t[4], len[4], cnt[4], all = 0, nb = 0, longest = 0;   // tiles of the lane's sequences; 0: no nodes
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int u = 4 * lane + i, bb = min(u, a.units - 1);
                cnt[i] = u < a.units ? nodes(bb) : 0;
                len[i] = length(bb);
                const int2 tt = tiles(len[i], cnt[i]);
                t[i] = cnt[i] ? tt.y - tt.x : 0;
                all += t[i] * blocks(cnt[i]);
                nb += blocks(cnt[i]);
                longest = max(longest, t[i]);
            }
            const int total = __builtin_amdgcn_readlane(wave_scan(all), 63);
            run = max(LGX_TREE_MIN, (int)((unsigned)(total + a.per - 1) / (unsigned)a.per));
            const int blks = __builtin_amdgcn_readlane(wave_scan(nb), 63);
            const int top = __builtin_amdgcn_readfirstlane((int)wave_max((float)longest));   // exact: at most 2^24
            // Whole sequences where they fill the device and are about equally long: then a
            // split gains less than its results' way through memory costs (b8-n100-l1000
            // on 28 heads of 4: 51 us whole, 54 split).
            if (2 * blks >= a.per && (int64_t)4 * top * blks <= (int64_t)5 * total) run = max(run, top);
            int m[4], upto, used;
            for (;;) {
                int c = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    m[i] = (int)((unsigned)(t[i] + run - 1) / (unsigned)run);
                    c += m[i] * blocks(cnt[i]);
                }
                upto = wave_scan(c);
                used = __builtin_amdgcn_readlane(upto, 63);
                if (used <= a.per) break;
                run += max(1, run >> 4);          // ends: a.per holds every column block
            }
            const int at = place_of(id, used * a.hkv);
            if (at < 0) return false;
            const int p = (int)((unsigned)at / (unsigned)a.hkv);
            const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > p));
            int first = 0, i = 0;                 // of the sequence among the (run, column block)s
            auto pick = [&](const int (&v)[4]) {
                const int v0 = __builtin_amdgcn_readlane(v[0], l), v1 = __builtin_amdgcn_readlane(v[1], l);
                const int v2 = __builtin_amdgcn_readlane(v[2], l), v3 = __builtin_amdgcn_readlane(v[3], l);
                return i == 0 ? v0 : i == 1 ? v1 : i == 2 ? v2 : v3;
            };
            int c[4], sum = 0;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                c[q] = m[q] * blocks(cnt[q]);
                sum += c[q];
            }
            first = __builtin_amdgcn_readlane(upto - sum, l);
#pragma unroll
            for (int q = 0; q < 3; ++q) {
                const int cq = __builtin_amdgcn_readlane(c[q], l);
                const bool next = i == q && p >= first + cq;
                first += next ? cq : 0;
                i += next ? 1 : 0;
            }
            ns = pick(m);
            sl = pick(len);
            n = pick(cnt);
            b = 4 * l + i;
            const int ncb = blocks(n), rest = at - first * a.hkv;
            s = rest / (ncb * a.hkv);
            const int gc = rest - s * ncb * a.hkv;
            g = gc / ncb;
            cb = gc - g * ncb;
            pos = first + cb * ns + s;            // the column block's splits side by side
            unit = b * a.ncb + cb;
            if (s == 0 && g == 0 && threadIdx.x == 0) {
                a.plan[2 * unit] = pos;
                a.plan[2 * unit + 1] = ns;
            }
        } else {
            const int at = place_of(id, a.units * a.hkv * a.ncb);
            if (at < 0) return false;
            const int bg = at / a.ncb;
            cb = at - bg * a.ncb;
            b = bg / a.hkv;
            g = bg - b * a.hkv;
            pos = 0;
            ns = 1;
        }
        b = __builtin_amdgcn_readfirstlane(b);
        g = __builtin_amdgcn_readfirstlane(g);
        c0 = __builtin_amdgcn_readfirstlane(cb) * LGX_TREE_COLS;
        if (!a.per) {
            n = __builtin_amdgcn_readfirstlane(nodes(b));
            sl = __builtin_amdgcn_readfirstlane(length(b));
        }
        ncols = n * G;
        if (c0 >= ncols) return false;
        const int2 t = tiles(sl, n);
        tb0 = t.x + s * run;
        tb1 = a.per ? min(t.y, tb0 + run) : t.y;
        return true;
    }
    __device__ __forceinline__ int64_t row(int c) const { return (int64_t)b * a.N + c / G; }
    __device__ __forceinline__ int64_t orow(int c) const { return row(c) * a.hq + g * G + c % G; }
    // positions end at 2^31 - 1, so that their distances have 31 bits
    __device__ __forceinline__ int depth(int i) const {
        return a.depth ? min(max(a.depth[(int64_t)b * a.N + i], 0), 0x7fffffff - sl) : i;
    }
    // bit i: node j sees token t0 + i (but for a window among the nodes: in_window)
    __device__ __forceinline__ uint64_t sees(int t0, int j, int dj) const {
        const int base = t0 - sl;                 // node of bit 0
        uint64_t m = 0;
        if (base < 0) {
            m = base <= -64 ? ~0ull : (1ull << -base) - 1;
            const int64_t lo = a.window ? (int64_t)sl + dj - a.window + 1 - t0 : 0;
            if (lo > 0) m = lo >= 64 ? 0 : m & ~0ull << lo;
        }
        if (base > -64) {
            const int end = (a.mask ? n : j + 1) - base;   // bits from here on are no nodes
            uint64_t d = ~0ull;
            if (a.mask) {
                const uint64_t* w = a.mask + row(j * G) * a.words;
                if (base < 0) {
                    d = w[0] << -base;
                } else {
                    const int i = base >> 6, s = base & 63;
                    d = i < a.words ? w[i] >> s : 0;
                    if (s && i + 1 < a.words) d |= w[i + 1] << (64 - s);
                }
            } else if (base < 0) {
                d <<= -base;
            }
            m |= end >= 64 ? d : end > 0 ? d & ((1ull << end) - 1) : 0;
        }
        return m;
    }
    // position of the column's node less that of token t
    __device__ __forceinline__ int back(int t, int dj) const { return t < sl ? sl + dj - t : dj - depth(min(t - sl, n - 1)); }
};

// One column: q's scale, the distance slope, its node and depth; running maximum (base 2), and
// sum of weights times 2^10.
struct TreeCol {
    float f, slope, m, l;
    int j, dj;
};
struct TreeEdge { static constexpr bool value = true; };
struct TreeWhole { static constexpr bool value = false; };

// a8_tanh with its quotient by the reciprocal and one correction (1.6 units of the last
// place): the exact division takes a third of the capped scores' time.
__device__ __forceinline__ float tree_tanh(float x) {
    const float ax = fabsf(x), t = __builtin_amdgcn_exp2f(-2.8853900817779268f * ax);
    const float n = 1.0f - t, d = 1.0f + t, r = __builtin_amdgcn_rcpf(d), q = n * r;
    const float big = copysignf(fmaf(fmaf(-q, d, n), r, q), x);
    const float y = x * x;
    float p = fmaf(y, -1382.0f / 155925.0f, 62.0f / 2835.0f);
    p = fmaf(y, p, -17.0f / 315.0f);
    p = fmaf(y, p, 2.0f / 15.0f);
    p = fmaf(y, p, -1.0f / 3.0f);
    return ax < 0.35f ? fmaf(x * y, p, x) : big;
}

// The query of a lane's column in two binary16 parts, dimensions 32 s + 8 kg .. in step s;
// the factor that makes a score (in base 2 unless X) of a product.
template <int D, bool X>
__device__ __forceinline__ float tree_query(const lgx_tree_attn_args& a, const float* qr, v8h (&qh)[2][D / 32]) {
    constexpr int NS = D / 32;
    float x[NS][8], am = 0.0f;
    bool bad = false;
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
            const float4 v = *(const float4*)(qr + 32 * s + e);
            x[s][e] = v.x;
            x[s][e + 1] = v.y;
            x[s][e + 2] = v.z;
            x[s][e + 3] = v.w;
        }
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            am = fmaxf(am, fabsf(x[s][e]));
            bad = bad || !(fabsf(x[s][e]) < __builtin_inff());
        }
    am = col_max(am);
    const bool isbad = col_max(bad ? 1.0f : 0.0f) != 0.0f;
    // a power of two; up to 2^122, where scale / up is still a normal number
    const float up = __uint_as_float(__float_as_uint(fminf(32768.0f / am, 0x1p122f)) & 0x7f800000u);
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        uint32_t hw[4], lw[4];
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const float y0 = isbad ? 0.0f : x[s][e] * up, y1 = isbad ? 0.0f : x[s][e + 1] * up;
            hw[e / 2] = f16_pair(y0, y1);
            lw[e / 2] = f16_pair(minus_half<0>(y0, hw[e / 2]), minus_half<1>(y1, hw[e / 2]));
        }
        qh[0][s] = as_v8h(make_uint4(hw[0], hw[1], hw[2], hw[3]));
        qh[1][s] = as_v8h(make_uint4(lw[0], lw[1], lw[2], lw[3]));
    }
    return isbad ? __builtin_nanf("") : a.scale / up * (X ? 1.0f : 1.44269504088896341f);
}

// From the products of a column tile to its weights as operands; o is brought to the new
// reference where it moves.  EDGE: some column does not see the whole tile, or the scores
// are capped, biased or windowed (X).  S[4 u + v]: token t0 + 16 u + 4 kg + v.
template <bool X, bool EDGE, int ND>
__device__ __forceinline__ void tree_weights(const Tree& w, float (&S)[16], TreeCol& k, int t0, int kg, v8h (&ph)[2], v8h (&pl)[2],
                                             v4f (&o)[ND]) {
    static_assert(EDGE || !X, "other scores are formed ahead of the maximum");
    constexpr float kLog2e = 1.44269504088896341f;
    const lgx_tree_attn_args& a = w.a;
    const float inf = __builtin_inff();
    if (EDGE) {
        if constexpr (X) {
#pragma unroll
            for (int e = 0; e < 16; ++e) S[e] *= k.f;
            if (a.softcap > 0.0f) {
                const float inv = 1.0f / a.softcap;
#pragma unroll
                for (int e = 0; e < 16; ++e) S[e] = a.softcap * tree_tanh(S[e] * inv);
            }
            const bool tree = t0 + LGX_TREE_TILE > w.sl;   // uniform: nodes among the tokens
            if (a.slopes || (tree && a.window)) {          // uniform
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int t = t0 + 16 * (e >> 2) + 4 * kg + (e & 3);
                    const int back = tree ? w.back(t, k.dj) : w.sl + k.dj - t;
                    S[e] -= k.slope * (float)back;
                    if (tree && a.window && back >= a.window) S[e] = -inf;
                }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) S[e] *= kLog2e;
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) S[e] *= k.f;
        }
        if (!X || a.window || t0 + LGX_TREE_TILE > w.sl) {   // uniform; else all see the whole tile
            const uint64_t sees = w.sees(t0, k.j, k.dj) >> (4 * kg);
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (!(sees >> (16 * (e >> 2) + (e & 3)) & 1)) S[e] = -inf;
        }
    }
    float m = fmaxf(fmaxf(S[0], S[1]), S[2]);
#pragma unroll
    for (int e = 3; e < 15; e += 2) m = fmaxf(fmaxf(m, S[e]), S[e + 1]);
    m = fmaxf(m, S[15]);
    if (!EDGE) m *= k.f;                          // > 0 or NaN
    const float mt = col_max(m);
    // the reference moves when a maximum passes it by more than 2^4: most tiles leave
    // what was summed as it is
    const bool moves = mt > k.m + 4.0f;
    if (__builtin_amdgcn_ballot_w64(moves)) {
        const float mn = moves ? mt : k.m;
        const float down = k.m == -inf ? 0.0f : __builtin_amdgcn_exp2f(k.m - mn);
#pragma unroll
        for (int i = 0; i < ND; ++i) o[i] *= down;
        k.l *= down;
        k.m = mn;
    }
    const float off = TREE_UP - (k.m == -inf ? 0.0f : k.m);   // nothing seen yet: weights of 0
    float ps[2] = {0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        S[e] = __builtin_amdgcn_exp2f(EDGE ? S[e] + off : fmaf(S[e], k.f, off));
        ps[e & 1] += S[e];
    }
    k.l += ps[0] + ps[1];
    uint32_t hw[8], lw[8];
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
        const uint32_t h = f16_pair(S[e], S[e + 1]);
        hw[e >> 1] = h;
        lw[e >> 1] = f16_pair(minus_half<0>(S[e], h), minus_half<1>(S[e + 1], h));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        ph[i] = as_v8h(make_uint4(hw[4 * i], hw[4 * i + 1], hw[4 * i + 2], hw[4 * i + 3]));
        pl[i] = as_v8h(make_uint4(lw[4 * i], lw[4 * i + 1], lw[4 * i + 2], lw[4 * i + 3]));
    }
}

// Column c over its run of tiles, token by token, by one wave: only seen tokens are
// multiplied.  m, l: the column's reference and sum (> 0).
template <int D, bool X>
__device__ void tree_column(const Tree& w, int c, float m, float l, float* dst) {
    constexpr float kLog2e = 1.44269504088896341f;
    const lgx_tree_attn_args& a = w.a;
    const int lane = threadIdx.x & 63, j = c / w.G, dj = w.depth(j);
    const float* q = a.q + w.orow(c) * D;
    const float slope = X && a.slopes ? a.slopes[w.g * w.G + c % w.G] : 0.0f;
    float o[D / 64] = {};
    for (int t0 = w.tb0 * LGX_TREE_TILE; t0 < w.tb1 * LGX_TREE_TILE; t0 += 64) {
        const int t = t0 + lane;
        const int page = min(max(a.page_table[(int64_t)w.b * a.maxp + min(t / LGX_PAGE, a.maxp - 1)], 0), a.num_pages - 1);
        const int64_t at = (((int64_t)page * a.hkv + w.g) * LGX_PAGE + t % LGX_PAGE) * D;
        bool on = w.sees(t0, j, dj) >> lane & 1;
        float s = 0.0f;
        if (on) {
            for (int i = 0; i < D; ++i) s = fmaf(q[i], h2f(a.k[at + i]), s);
            s *= a.scale;
            if (X) {
                if (a.softcap > 0.0f) s = a.softcap * a8_tanh(s / a.softcap);
                const int back = w.back(t, dj);
                s -= slope * (float)back;
                on = !a.window || back < a.window;
            }
            s = __builtin_amdgcn_exp2f(s * kLog2e - m);
        }
        uint64_t todo = __builtin_amdgcn_ballot_w64(on);
        while (todo) {
            const int i = __builtin_ctzll(todo);
            todo &= todo - 1;
            const float wt = __shfl(s, i, 64);
            const int64_t vat = __shfl((long long)at, i, 64);
#pragma unroll
            for (int e = 0; e < D / 64; ++e) o[e] = fmaf(wt, h2f(a.v[vat + 64 * e + lane]), o[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < D / 64; ++e) dst[64 * e + lane] = o[e] / l;
}

// A column's result, or its split's (divided by the split's own sum of weights).
template <int D, bool X>
__device__ __forceinline__ void tree_store(const Tree& w, int c, const TreeCol& k, int kg, const v4f (&o)[D / 16]) {
    const lgx_tree_attn_args& a = w.a;
    const bool part = w.ns > 1, on = c < w.ncols;
    const int64_t at = part ? ((int64_t)w.pos * a.hkv + w.g) * LGX_TREE_COLS + c - w.c0 : w.orow(on ? c : 0);
    float* dst = (part ? a.part : a.out) + at * D;
    const float r = 1.0f / k.l, l = k.l * (1.0f / (1 << TREE_UP));
    // Nothing seen (here: another split may see some) gives zeros by selection, not by a factor:
    // o is NaN where an unseen token's V is not finite, and so would be the joined result.
    const bool none = k.l == 0.0f;
    bool bad = false;
    if (on) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            const v4f x = none ? (v4f){0.0f, 0.0f, 0.0f, 0.0f} : o[i] * r;
            *(float4*)(dst + 16 * i + 4 * kg) = make_float4(x[0], x[1], x[2], x[3]);
            bad = bad || !(fabsf(x[0]) + fabsf(x[1]) + fabsf(x[2]) + fabsf(x[3]) < __builtin_inff());
        }
        if (part && kg == 0) *(float2*)(a.ml + 2 * at) = make_float2(k.m, l);
    }
    uint64_t again = __builtin_amdgcn_ballot_w64(bad && l == l);
    again = (again | again >> 16 | again >> 32 | again >> 48) & 0xffff;
    if (again) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the first results are written
    while (again) {
        const int i = __builtin_ctzll(again);
        again &= again - 1;
        tree_column<D, X>(w, __shfl(c, i, 64), __shfl(k.m, i, 64), __shfl(l, i, 64),
                          (float*)__shfl((unsigned long long)(uintptr_t)dst, i, 64));
    }
}

// V operands of dimensions 16 i .. from the LDS rows of a tile: tokens of sub-tiles 2 h and
// 2 h + 1.  Lane (col, kg) loads token 16 u + 4 kg + col / 4, dimensions 16 i + 4 (col % 4) ..,
// and receives dimension 16 i + col of tokens 16 u + 4 kg .. + 3.  Pieces of a row change
// places by the token, so that the rows of a load fall on different banks.
template <int D>
struct TreeV {
    static constexpr int CH = D / 8, SW = CH / 2 - 1;
    static __device__ __forceinline__ int piece(int t, int c) { return c ^ ((t & SW) << 1); }
    static __device__ __forceinline__ v8h operand(const lds_u16* v, int i, int h, int col, int kg) {
        uint2 x[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int t = 16 * (2 * h + u) + 4 * kg + (col >> 2);
            x[u] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                 (lds_v4s*)(v + t * D + piece(t, 2 * i + ((col >> 1) & 1)) * 8 + (col & 1) * 4)));
        }
        return as_v8h(make_uint4(x[0].x, x[0].y, x[1].x, x[1].y));
    }
};
// Its K operands: row (token) 16 u + col, dimensions 32 s + 8 kg ..
template <int D>
struct TreeK {
    static constexpr int CH = D / 8;
    static __device__ __forceinline__ int piece(int t, int c) { return c ^ (t & (CH - 1)); }
    static __device__ __forceinline__ v8h operand(const lds_u16* k, int u, int s, int col, int kg) {
        typedef __attribute__((address_space(3))) const u32x4 lds_u4;
        const int t = 16 * u + col;
        return __builtin_bit_cast(v8h, *(lds_u4*)(k + t * D + piece(t, 4 * s + kg) * 8));
    }
};

// 16 columns per wave: tiles of K and V pass through LDS, the next one in flight from the
// barrier that publishes this one on.
template <int D, bool X>
__device__ __forceinline__ void tree_body(const lgx_tree_attn_args& a) {
    constexpr int NS = D / 32, ND = D / 16, CH = D / 8;
    constexpr int TPI = 64 / CH, NI = LGX_TREE_TILE / TPI;   // tokens of a 1 KiB load, loads of a tile's K or V
    __shared__ __align__(16) uint16_t kv_s[2][2][LGX_TREE_TILE * D];
    const int lane = threadIdx.x & 63, col = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Tree w{a};
    if (!w.place()) return;                       // uniform
    const_i32* table = (const_i32*)(a.page_table + (int64_t)w.b * a.maxp);   // through the scalar cache
    struct Pages {
        int p[LGX_TREE_TILE / LGX_PAGE];
    };
    auto pages = [&](int t) {
        Pages r;
#pragma unroll
        for (int u = 0; u < 4; ++u) r.p[u] = table[min(4 * t + u, a.maxp - 1)];
        return r;
    };
    // waves 0 and 1 bring K, 2 and 3 V
    auto load = [&](int buf, const Pages& p) __attribute__((always_inline)) {
        lds_u16* to = (lds_u16*)kv_s[buf][wave >> 1];
#pragma unroll
        for (int j = 0; j < NI / 2; ++j) {
            const int i = (wave & 1) * (NI / 2) + j;
            const int u = i * TPI / LGX_PAGE, r = i * TPI % LGX_PAGE + lane / CH;   // page, row
            const int pg = u == 0 ? p.p[0] : u == 1 ? p.p[1] : u == 2 ? p.p[2] : p.p[3];
            const int64_t blk = ((int64_t)min(max(pg, 0), a.num_pages - 1) * a.hkv + w.g) * (LGX_PAGE * D);
            const int c = wave < 2 ? TreeK<D>::piece(r, lane % CH) : TreeV<D>::piece(r, lane % CH);
            load_lds_16((wave < 2 ? a.k : a.v) + blk + (r * D + c * 8), (lds_void*)(to + i * 512));
        }
    };
    const int end = w.tb1, T = w.sl + w.n;
    int t = w.tb0;
    load(0, pages(t));
    Pages p = pages(min(t + 1, end - 1));
    const int wcol = w.c0 + wave * 16;
    const bool any = wcol < w.ncols;              // else the wave only loads
    v4f o[ND];
#pragma unroll
    for (int i = 0; i < ND; ++i) o[i] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
    TreeCol k;
    v8h qh[2][NS];
    {
        const int c = min(wcol + col, w.ncols - 1);   // columns past the last repeat it
        k = {0.0f, X && a.slopes ? a.slopes[w.g * w.G + c % w.G] : 0.0f, -__builtin_inff(), 0.0f, c / w.G, 0};
        k.dj = w.depth(k.j);
        k.f = tree_query<D, X>(a, a.q + w.orow(c) * D + 8 * kg, qh);
    }
    auto tile = [&](auto form) __attribute__((always_inline)) {
        constexpr bool edge = decltype(form)::value;
        const int t0 = t * LGX_TREE_TILE, cur = (t - w.tb0) & 1;
        publish_lds_loads();                      // this tile is there, the last one read
        if (edge && t0 + LGX_TREE_TILE > T) {         // uniform
            // rows behind the last node: weight 0 times whatever they hold
            for (int i = threadIdx.x; i < LGX_TREE_TILE * CH; i += 256)
                if (t0 + i / CH >= T) *(uint4*)(kv_s[cur][1] + i * 8) = make_uint4(0u, 0u, 0u, 0u);
            __syncthreads();
        }
        if (t + 1 < end) {                        // uniform
            load(cur ^ 1, p);
            p = pages(min(t + 2, end - 1));
        }
        if (!any) return;
        const lds_u16* ks = (const lds_u16*)kv_s[cur][0];
        const lds_u16* vs = (const lds_u16*)kv_s[cur][1];
        float S[16];
        {
            // the four sub-tiles' chains side by side, operands a step ahead
            v4f acc[4];
            v8h kf[2][4];
#pragma unroll
            for (int u = 0; u < 4; ++u) kf[0][u] = TreeK<D>::operand(ks, u, 0, col, kg);
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                if (s + 1 < NS) {
#pragma unroll
                    for (int u = 0; u < 4; ++u) kf[(s + 1) & 1][u] = TreeK<D>::operand(ks, u, s + 1, col, kg);
                }
#pragma unroll
                for (int part = 1; part >= 0; --part)
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        acc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            kf[s & 1][u], qh[part][s], s == 0 && part == 1 ? (v4f){0.0f, 0.0f, 0.0f, 0.0f} : acc[u], 0, 0, 0);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) S[e] = acc[e >> 2][e & 3];
        }
        v8h ph[2], pl[2];
        tree_weights<X, edge, ND>(w, S, k, t0, kg, ph, pl, o);
        // 64 dimensions at a time, their chains side by side, operands a step ahead
        v8h vf[2][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) vf[0][i] = TreeV<D>::operand(vs, i, 0, col, kg);
#pragma unroll
        for (int g = 0; g < ND / 4; ++g) {
            v4f r[4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (h == 0 || g + 1 < ND / 4) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) vf[h ^ 1][i] = TreeV<D>::operand(vs, 4 * (g + h) + i, h ^ 1, col, kg);
                }
#pragma unroll
                for (int part = 1; part >= 0; --part)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        r[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            vf[h][i], part ? pl[h] : ph[h], h == 0 && part == 1 ? (v4f){0.0f, 0.0f, 0.0f, 0.0f} : r[i], 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) o[4 * g + i] += r[i];
        }
    };
    // the tiles of cached tokens alone, then the others
    if constexpr (!X) {
#pragma unroll 1
        for (const int whole = min(end, w.sl / LGX_TREE_TILE); t < whole; ++t) tile(TreeWhole());
    }
#pragma unroll 1
    for (; t < end; ++t) tile(TreeEdge());
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // no load into LDS outlives the wave
    if (!any) return;
    k.l = col_sum(k.l);
    tree_store<D, X>(w, wcol + col, k, kg, o);
}

#define LGX_TREE_KERNEL(NAME, BODY) \
    extern "C" __global__ __launch_bounds__(256, 2) void NAME(const lgx_tree_attn_args a) { BODY(a); }
LGX_TREE_KERNEL(lgx_k_tree_attn_d64, (tree_body<64, false>))
LGX_TREE_KERNEL(lgx_k_tree_attnx_d64, (tree_body<64, true>))
LGX_TREE_KERNEL(lgx_k_tree_attn_d128, (tree_body<128, false>))
LGX_TREE_KERNEL(lgx_k_tree_attnx_d128, (tree_body<128, true>))

// Joins the splits of each (node, query head): D / 4 lanes hold its dimensions, NG such
// groups take its splits in turn, four in flight, and meet in LDS.  A row is its plan's
// memory round, then one for each four splits of a group.
template <int D, int NG>
__device__ __forceinline__ void tree_join_body(const lgx_tree_attn_args& a) {
    constexpr int Q = D / 4, IT = 256 / (Q * NG);  // items of a workgroup
    __shared__ v4f o_s[NG > 1 ? NG * Q : 1];
    __shared__ float2 ml_s[NG > 1 ? NG : 1];
    const int q = threadIdx.x % Q, sg = NG > 1 ? threadIdx.x / Q : 0;
    const unsigned item = blockIdx.x * IT + (NG > 1 ? 0 : threadIdx.x / Q);
    if (item >= (unsigned)a.rows * (unsigned)a.hq) return;
    const unsigned row = item / (unsigned)a.hq, b = row / (unsigned)a.N;
    const int h = (int)(item - row * a.hq), j = (int)(row - b * a.N), G = a.hq / a.hkv;
    const int g = h / G, c = j * G + h - g * G, u = (int)b * a.ncb + c / LGX_TREE_COLS;
    const int n = a.n_nodes ? a.n_nodes[b] : a.N;
    const int2 plan = *(const int2*)(a.plan + 2 * u);
    if (j >= n || plan.y < 2) return;             // with NG > 1 uniform
    const float inf = __builtin_inff();
    const int64_t at0 = ((int64_t)plan.x * a.hkv + g) * LGX_TREE_COLS + c % LGX_TREE_COLS, step = (int64_t)a.hkv * LGX_TREE_COLS;
    float m = -inf, l = 0.0f;
    v4f o = {0.0f, 0.0f, 0.0f, 0.0f};
    // ls times the mean os, by the maximum ms (an empty split's is -inf; so is a NaN one's, whose ls is NaN)
    auto join = [&](float ms, float ls, v4f os) {
        const float mn = fmaxf(m, ms);
        const float u0 = m == -inf ? 0.0f : __builtin_amdgcn_exp2f(m - mn), u1 = (ms == -inf ? 0.0f : __builtin_amdgcn_exp2f(ms - mn)) * ls;
        o = o * u0 + os * u1;
        l = l * u0 + u1;
        m = mn;
    };
    for (int s0 = sg; s0 < plan.y; s0 += 4 * NG) {
        float2 ml[4];
        v4f p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t at = at0 + min(s0 + i * NG, plan.y - 1) * step;
            ml[i] = *(const float2*)(a.ml + 2 * at);
            p[i] = *((const v4f*)(a.part + at * D) + q);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (s0 + i * NG < plan.y) join(ml[i].x, ml[i].y, p[i]);
    }
    if constexpr (NG > 1) {
        o_s[threadIdx.x] = o;                     // not yet divided by l
        if (q == 0) ml_s[sg] = make_float2(m, l);
        __syncthreads();
        if (sg) return;
        float mx = m;
#pragma unroll
        for (int i = 1; i < NG; ++i) mx = fmaxf(mx, ml_s[i].x);
        l = 0.0f;
        o = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const float w = ml_s[i].x == -inf ? 0.0f : __builtin_amdgcn_exp2f(ml_s[i].x - mx);
            l += ml_s[i].y * w;
            o += o_s[i * Q + q] * w;
        }
    }
    const float r = l == 0.0f ? 0.0f : 1.0f / l;
    *((v4f*)(a.out + (int64_t)item * D) + q) = o * r;
}
extern "C" __global__ __launch_bounds__(256) void lgx_k_tree_join_d64(const lgx_tree_attn_args a) { tree_join_body<64, 16>(a); }
extern "C" __global__ __launch_bounds__(256) void lgx_k_tree_joinr_d64(const lgx_tree_attn_args a) { tree_join_body<64, 1>(a); }
extern "C" __global__ __launch_bounds__(256) void lgx_k_tree_join_d128(const lgx_tree_attn_args a) { tree_join_body<128, 8>(a); }
extern "C" __global__ __launch_bounds__(256) void lgx_k_tree_joinr_d128(const lgx_tree_attn_args a) { tree_join_body<128, 1>(a); }
