// lgx_tree.hip -- several drafted tokens per sequence and step: their rows appended to
// the binary16 cache, which of them hold, and the cache closed up behind those.
#include "lgx_device.h"

// ---------------------------------------------------------------------------
// Append.  Row j of sequence b is token slot seq_len + j, at position seq_len +
// depth[j] (siblings share a position, each has a slot).  Arithmetic as in
// lgx_k_qkv_rope_append: binary32, each product rounded on its own, K and V rounded to
// nearest binary16; with rot = d and halves as pairs the results are that kernel's.
//
// A thread holds 4 pairs of a head: pair p < rot / 2 is (p, p + rot / 2), or (2p, 2p + 1)
// when interleaved, and turns; the others are (2p, 2p + 1) and do not.
//
// Bound by memory: 64 sequences of up to 33 rows of 36 heads of 128 (38 MB where half the
// rows are padding) take 13.2 to 15.9 us, 2.4 to 2.9 TB/s, after two dependent rounds for a
// row's number, length and angle.  A small call is those rounds: 3.6 us for 6 rows.  (Two
// heads of a row per thread, with half the rounds of workgroups: 18.6 and 4.4 us.)
// ---------------------------------------------------------------------------
template <int D>
__device__ __forceinline__ void append_rows_body(const lgx_append_rows_args& a) {
    constexpr int TPH = D / 8;                    // threads of a head
    const int nh = a.hq + 2 * a.hkv;
    // the workgroup's first head by one division of 64 bits (uniform), the thread's by 32
    const int64_t item0 = (int64_t)blockIdx.x * (256 / TPH), r0 = item0 / nh;
    const int of = threadIdx.x / TPH;
    if (item0 + of >= a.items) return;
    const unsigned from = (unsigned)(item0 - r0 * nh) + of, down = from / (unsigned)nh;
    const int64_t r = r0 + down;                  // below 2^31
    const int h = (int)(from - down * nh), b = (int)((unsigned)r / (unsigned)a.N), j = (int)((unsigned)r - (unsigned)b * a.N);
    if (a.n_new && j >= a.n_new[b]) return;
    const bool isv = h >= a.hq + a.hkv;
    const int rot = isv ? 0 : a.rot, half = rot / 2, p = (threadIdx.x % TPH) * 4;
    const int64_t sl = min(max(a.seq_len[b], 0), a.maxp * LGX_PAGE);
    const float* x = a.x + r * ((int64_t)nh * D) + h * D;
    const float* bias = a.bias ? a.bias + h * D : nullptr;
    // first dimensions of the members of pair p + i
    const bool apart = !a.interleaved;
    int d0[4], d1[4];
    float x0[4], x1[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool split = apart && p + i < half;
        d0[i] = split ? p + i : 2 * (p + i);
        d1[i] = split ? p + i + half : 2 * (p + i) + 1;
    }
    const bool split = apart && p < half;         // with vec, of all four pairs
    if (a.vec) {
        const float4 u = *(const float4*)(x + (split ? p : 2 * p)), w = *(const float4*)(x + (split ? p + half : 2 * p + 4));
        x0[0] = u.x, x0[1] = split ? u.y : u.z, x0[2] = split ? u.z : w.x, x0[3] = split ? u.w : w.z;
        x1[0] = split ? w.x : u.y, x1[1] = split ? w.y : u.w, x1[2] = split ? w.z : w.y, x1[3] = w.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x0[i] = x[d0[i]], x1[i] = x[d1[i]];
    }
    if (bias) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x0[i] = x0[i] + bias[d0[i]], x1[i] = x1[i] + bias[d1[i]];
    }
    if (p < half) {
        const int64_t dep = a.depth ? a.depth[r] : j;
        const int64_t pos = min(max(sl + dep, (int64_t)0), (int64_t)a.max_pos - 1) * half + p;
        float c[4], s[4];
        if (a.vec) {
            *(float4*)c = *(const float4*)(a.cos_t + pos);
            *(float4*)s = *(const float4*)(a.sin_t + pos);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                c[i] = p + i < half ? a.cos_t[pos + i] : 1.0f;
                s[i] = p + i < half ? a.sin_t[pos + i] : 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float t0 = x0[i] * c[i], t1 = x1[i] * s[i], t2 = x1[i] * c[i], t3 = x0[i] * s[i];
            // a pair that does not turn keeps its bits
            x0[i] = p + i < half ? t0 - t1 : x0[i];
            x1[i] = p + i < half ? t2 + t3 : x1[i];
        }
    }
    if (h < a.hq) {
        float* q = a.q_out + (r * a.hq + h) * D;
        if (a.vec) {
            *(float4*)(q + (split ? p : 2 * p)) = split ? make_float4(x0[0], x0[1], x0[2], x0[3]) : make_float4(x0[0], x1[0], x0[1], x1[1]);
            *(float4*)(q + (split ? p + half : 2 * p + 4)) =
                split ? make_float4(x1[0], x1[1], x1[2], x1[3]) : make_float4(x0[2], x1[2], x0[3], x1[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) q[d0[i]] = x0[i], q[d1[i]] = x1[i];
        }
        return;
    }
    const int64_t t = sl + j;
    if (t >= (int64_t)a.maxp * LGX_PAGE) return;
    const int page = a.page_table[(int64_t)b * a.maxp + t / LGX_PAGE];
    if (page < 0 || page >= a.num_pages) return;
    const int g = h - a.hq - (isv ? a.hkv : 0);
    uint16_t* row = (isv ? a.v : a.k) + (((int64_t)page * a.hkv + g) * LGX_PAGE + t % LGX_PAGE) * D;
    if (a.vec) {
        const uint2 lo = split ? make_uint2(f16_pair(x0[0], x0[1]), f16_pair(x0[2], x0[3])) : make_uint2(f16_pair(x0[0], x1[0]), f16_pair(x0[1], x1[1]));
        const uint2 hi = split ? make_uint2(f16_pair(x1[0], x1[1]), f16_pair(x1[2], x1[3])) : make_uint2(f16_pair(x0[2], x1[2]), f16_pair(x0[3], x1[3]));
        if (split) {
            *(uint2*)(row + p) = lo;
            *(uint2*)(row + p + half) = hi;
        } else {
            *(uint4*)(row + 2 * p) = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) row[d0[i]] = f2h(x0[i]), row[d1[i]] = f2h(x1[i]);
    }
}
extern "C" __global__ __launch_bounds__(256) void lgx_k_append_rows_d64(const lgx_append_rows_args a) { append_rows_body<64>(a); }
extern "C" __global__ __launch_bounds__(256) void lgx_k_append_rows_d128(const lgx_append_rows_args a) { append_rows_body<128>(a); }

// ---------------------------------------------------------------------------
// Trees.  parent[j] < j, or -1 where node j hangs from the sequence's last token; any
// other value counts as -1.  Bound by chains of dependent steps, one for each generation.
// The plan, an LDS read a step: 1.6 us for a chain of 6 nodes, 3.1 for 32 trees of 24, 5.5 for a
// chain of 64, 18 for one of 256 (19.6 for 64 of them; 4.6 for a tree of 256 nodes with
// parents among the last 12).  The walk, some VALU operations a step: 2.5 us for one tree of 6
// nodes, 5.0 for 32 of 24.
// ---------------------------------------------------------------------------
__device__ __forceinline__ int tree_parent(int p, int j) { return p >= 0 && p < j ? p : -1; }

// A workgroup per sequence, a thread per node, which walks up to its root.
extern "C" __global__ __launch_bounds__(LGX_TREE_NODES) void lgx_k_tree_plan(const lgx_tree_plan_args a) {
    __shared__ int par[LGX_TREE_NODES];
    const int b = blockIdx.x, j = threadIdx.x;
    const int n = a.n_nodes ? min(max(a.n_nodes[b], 0), a.N) : a.N;
    if (j < n) par[j] = tree_parent(a.parent[(int64_t)b * a.N + j], j);
    __syncthreads();
    if (j >= n) return;
    uint64_t m[LGX_TREE_NODES / 64] = {};
    int depth = -1;
    for (int i = j; i >= 0; i = par[i]) {         // ends: parents come before their children
        ++depth;
#pragma unroll
        for (int w = 0; w < LGX_TREE_NODES / 64; ++w)
            if (i >> 6 == w) m[w] |= 1ull << (i & 63);
    }
    const int64_t row = (int64_t)b * a.N + j;
    a.depth[row] = depth;
#pragma unroll
    for (int w = 0; w < LGX_TREE_NODES / 64; ++w)
        if (w < a.words) a.mask[row * a.words + w] = m[w];
}

// A wave per sequence: from node 0 on to the first child (the lowest) whose token was
// picked behind the node.
extern "C" __global__ __launch_bounds__(64) void lgx_k_tree_accept(const lgx_tree_accept_args a) {
    constexpr int W = LGX_TREE_NODES / 64;
    const int b = blockIdx.x, lane = threadIdx.x;
    const int n = a.n_nodes ? min(max(a.n_nodes[b], 0), a.N) : a.N;
    const int64_t at = (int64_t)b * a.N;
    int par[W], tok[W], pick[W];
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const int j = 64 * w + lane;
        par[w] = j < n ? tree_parent(a.parent[at + j], j) : -1;
        tok[w] = j < n ? a.tokens[at + j] : 0;
        pick[w] = j < n ? a.picked[at + j] : 0;
    }
    int cur = n > 0 ? 0 : -1, count = 0, last = 0;
    while (cur >= 0) {                            // uniform; ends: cur grows
        if (lane == 0) a.path[at + count] = cur;
        ++count;
        int t = 0;
#pragma unroll
        for (int w = 0; w < W; ++w)
            if (cur >> 6 == w) t = __builtin_amdgcn_readlane(pick[w], cur & 63);
        last = t;
        int child = -1;
#pragma unroll
        for (int w = W - 1; w >= 0; --w) {
            const uint64_t hit = __builtin_amdgcn_ballot_w64(par[w] == cur && tok[w] == t);
            if (hit) child = 64 * w + __builtin_ctzll(hit);
        }
        cur = child;
    }
    for (int j = count + lane; j < a.N; j += 64) a.path[at + j] = -1;
    if (lane == 0) {
        a.count[b] = count;
        if (n > 0) a.next[b] = last;
        if (a.new_len) a.new_len[b] = a.seq_len[b] + count;
    }
}

// Rows start + keep[i] of a sequence become rows start + i, a wave per (sequence, K or V
// array of a layer, KV head).  keep ascends, so that a row's new place is never behind
// its old one, and never a later row's old one: 16 / (D / 64) rows are read before any of
// them is written, then the next ones.  A small call is four dependent rounds (3.3 us for 6
// nodes in 24 layers); 28 layers of 32 sequences, 17 MB, take 6.9 to 7.3 us.
template <int D>
__device__ __forceinline__ void kv_keep_body(const lgx_kv_keep_args& a) {
    constexpr int CH = D / 8, RW = 64 / CH, U = 4;   // pieces of a row, rows of a load, loads in flight
    const int lane = threadIdx.x & 63, b = blockIdx.x;
    const int g = blockIdx.z * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (g >= a.hkv) return;
    const int n = min(max(a.n_keep[b], 0), a.N);
    const int64_t start = max(a.start[b], 0);
    const int32_t* table = a.page_table + (int64_t)b * a.maxp;
    const int32_t* keep = a.keep + (int64_t)b * a.N;
    uint16_t* base = a.base[blockIdx.y];
    // piece of token t, or null
    auto at = [&](int64_t t) -> uint4* {
        if (t >= (int64_t)a.maxp * LGX_PAGE) return nullptr;
        const int page = table[t / LGX_PAGE];
        if (page < 0 || page >= a.num_pages) return nullptr;
        return (uint4*)(base + (((int64_t)page * a.hkv + g) * LGX_PAGE + t % LGX_PAGE) * D) + lane % CH;
    };
    for (int i0 = 0; i0 < n; i0 += RW * U) {
        uint4 v[U];
        bool on[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * RW + lane / CH;
            const int from = i < n ? keep[i] : -1;
            const uint4* src = from >= 0 && from != i ? at(start + from) : nullptr;
            on[u] = src != nullptr;
            v[u] = on[u] ? *src : make_uint4(0u, 0u, 0u, 0u);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // every row is read before one is written
#pragma unroll
        for (int u = 0; u < U; ++u) {
            uint4* dst = on[u] ? at(start + i0 + u * RW + lane / CH) : nullptr;
            if (dst) *dst = v[u];
        }
    }
}
extern "C" __global__ __launch_bounds__(256) void lgx_k_kv_keep_d64(const lgx_kv_keep_args a) { kv_keep_body<64>(a); }
extern "C" __global__ __launch_bounds__(256) void lgx_k_kv_keep_d128(const lgx_kv_keep_args a) { kv_keep_body<128>(a); }
