// lgx_tree.cpp -- drafted tokens: rows appended to the binary16 cache, trees of drafts,
// the walk over those that hold, the cache closed up behind it (kernels in
// lgx_tree.hip); sampling with per-row settings (lgx_filter.hip).
#include "lgx_internal.h"

using namespace lgxi;

namespace {

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

lgx_status check_kv(const lgx_kv_f16* kv, int32_t maxp) {
    if (!kv) return fail(LGX_NULL_POINTER, "kv is NULL");
    if (!kv->k || !kv->v) return fail(LGX_NULL_POINTER, "NULL cache pointer");
    if (kv->num_pages <= 0 || kv->hkv <= 0 || maxp <= 0 || maxp > 1 << 26)
        return fail(LGX_INVALID_ARGUMENT, "num_pages=%d hkv=%d maxp=%d", kv->num_pages, kv->hkv, maxp);
    if (kv->d != 64 && kv->d != 128) return fail(LGX_UNSUPPORTED, "head_dim %d (64 or 128)", kv->d);
    if (!aligned16(kv->k) || !aligned16(kv->v))
        return fail(LGX_INVALID_ARGUMENT, "cache pages must be 16-byte aligned");
    return LGX_OK;
}

// An output that another row's thread still reads, or that is read again (tree_column).
bool overlap(const float* a, int64_t na, const float* b, int64_t nb) { return a < b + nb && b < a + na; }

lgx_status check_tree(int32_t B, int32_t N) {
    if (B <= 0 || N <= 0 || N > LGX_TREE_NODES)
        return fail(LGX_INVALID_ARGUMENT, "B=%d, %d nodes (1..%d)", B, N, LGX_TREE_NODES);
    return LGX_OK;
}

// Launch over B sequences.  Where there are fewer (sequence, KV head, column block)s
// than two to a compute unit, their tiles are split among that many workgroups; the
// splitting itself is done on the device, by the lengths.  Splits for one to a compute unit
// against two (28 heads of 4, 128 dimensions): 85 against 69 us for 32 ragged sequences
// of up to 4096 tokens and 16 nodes, 66 against 56 for 64 of 3000 and 2; but 25.9 against
// 27.5 for 16 of 2000 and 8.  The joining of the splits is that of the 8-bit cache's attention.
lgx_status run_tree(lgx_ctx* c, lgx_tree_attn_args& a, int B, int d, bool x, void* stream) {
    const int64_t cols = (int64_t)a.N * (a.hq / a.hkv), heads = (int64_t)B * a.hkv;
    // the most tiles that a sequence's nodes can see
    int64_t tiles = cdiv((int64_t)a.maxlen + a.N, LGX_TREE_TILE);
    if (a.window) tiles = std::min<int64_t>(tiles, ((int64_t)a.window + a.N) / LGX_TREE_TILE + 2);
    const int64_t ncb = cdiv(cols, LGX_TREE_COLS), units = B * ncb, blocks = heads * ncb;
    a.ncb = (int)ncb;
    a.units = B;
    a.rows = B * a.N;
    const int64_t per = (int64_t)c->tree_wgs * c->ncu / a.hkv;
    const bool split = tiles > LGX_TREE_MIN && B <= LGX_TREE_UNITS && units < per && units * tiles <= INT32_MAX;
    lgx_status st;
    if (split) {
        const int64_t slots = per * a.hkv * LGX_TREE_COLS;
        float* ws = nullptr;
        if ((st = ensure_ws(c, (size_t)(slots * (d + 2) + 2 * units) * sizeof(float), stream, &ws)) != LGX_OK) return st;
        a.per = (int)per;
        a.part = ws;
        a.ml = ws + slots * d;
        a.plan = (int32_t*)(a.ml + 2 * slots);
    }
    const int64_t grid = ((split ? per * a.hkv : blocks) + 7) / 8 * 8;   // an eighth per XCD
    if (grid > UINT32_MAX / 256) return fail(LGX_OUT_OF_BOUNDS, "attention of %lld workgroups", (long long)grid);
    const int k = (d == 64 ? K_TREE_ATTN_D64 : K_TREE_ATTN_D128) + (x ? 1 : 0);
    if ((st = launch(c, (Kern)k, dim3((unsigned)grid), dim3(256), a, stream)) != LGX_OK || !split) return st;
    const int64_t rh = (int64_t)B * a.N * a.hq;
    // one group of lanes for all splits of a (node, query head) from 8 of them to a compute unit
    // on (14336 of them with 2 or 3 splits: the whole call 66.6 against 75.7 us), several below
    // (1792 with 18: 33.2 against 34.8)
    const int w = rh >= 8 * (int64_t)c->ncu ? 1 : 0;
    return launch(c, (Kern)((d == 64 ? K_TREE_JOIN_D64 : K_TREE_JOIN_D128) + w), dim3(w ? cdiv(rh * (d / 4), 256) : (unsigned)rh),
                  dim3(256), a, stream);
}

}  // namespace

extern "C" {

lgx_status lgx_gqa_tree_attn(lgx_ctx* c, const float* q, const lgx_kv_f16* kv, const int32_t* page_table,
                             const int32_t* seq_len, const int32_t* n_nodes, const int32_t* depth, const uint64_t* mask,
                             int32_t B, int32_t N, int32_t hq, int32_t maxp, int32_t max_seq_len, const lgx_attn_opts* opts,
                             float* out, void* stream) {
    return guarded(__func__, [&]() -> lgx_status {
        lgx_status st = enter(c);
        if (st != LGX_OK) return st;
        if ((st = check_kv(kv, maxp)) != LGX_OK) return st;
        if (!q || !page_table || !seq_len || !out) return fail(LGX_NULL_POINTER, "NULL tensor pointer");
        if ((st = check_tree(B, N)) != LGX_OK) return st;
        if (hq <= 0 || hq % kv->hkv != 0) return fail(LGX_INVALID_ARGUMENT, "hq=%d hkv=%d", hq, kv->hkv);
        if (hq / kv->hkv > 16) return fail(LGX_UNSUPPORTED, "%d query heads per KV head (1..16)", hq / kv->hkv);
        if (max_seq_len < 0 || max_seq_len > maxp * LGX_PAGE - N)
            return fail(LGX_OUT_OF_BOUNDS, "max_seq_len %d outside [0, %d]", max_seq_len, maxp * LGX_PAGE - N);
        if ((int64_t)B * N * hq > INT32_MAX / 128) return fail(LGX_OUT_OF_BOUNDS, "B*N*hq too large");
        if (!aligned16(q) || !aligned16(out)) return fail(LGX_INVALID_ARGUMENT, "q and out must be 16-byte aligned");
        const int64_t n = (int64_t)B * N * hq * kv->d;
        if (overlap(q, n, out, n)) return fail(LGX_INVALID_ARGUMENT, "q and out overlap");
        lgx_tree_attn_args a{};
        a.scale = (float)(1.0 / std::sqrt((double)kv->d));
        if (opts) {
            if (!std::isfinite(opts->scale) || !std::isfinite(opts->softcap) ||
                (opts->softcap != 0.0f && !(opts->softcap >= 0x1p-100f)) || opts->window < 0)
                return fail(LGX_INVALID_ARGUMENT, "scale %g, softcap %g, window %d", (double)opts->scale,
                            (double)opts->softcap, opts->window);
            if (opts->scale != 0.0f) a.scale = opts->scale;
            a.softcap = opts->softcap;
            a.window = opts->window;
            a.slopes = opts->slopes;
        }
        a.q = q;
        a.k = kv->k;
        a.v = kv->v;
        a.page_table = page_table;
        a.seq_len = seq_len;
        a.n_nodes = n_nodes;
        a.depth = depth;
        a.mask = mask;
        a.out = out;
        a.N = N;
        a.words = (N + 63) / 64;
        a.hq = hq;
        a.hkv = kv->hkv;
        a.maxp = maxp;
        a.num_pages = kv->num_pages;
        a.maxlen = max_seq_len;
        return run_tree(c, a, B, kv->d, a.softcap > 0.0f || a.window > 0 || a.slopes != nullptr || a.scale < 0.0f, stream);
    });
}

lgx_status lgx_rope_kv_append_rows(lgx_ctx* c, const float* qkv, const float* bias, const lgx_rope* rope,
                                   const int32_t* seq_len, const int32_t* depth, const int32_t* n_new,
                                   const int32_t* page_table, const lgx_kv_f16* kv, float* q_out, int32_t B, int32_t N,
                                   int32_t hq, int32_t maxp, void* stream) {
    return guarded(__func__, [&]() -> lgx_status {
        lgx_status st = enter(c);
        if (st != LGX_OK) return st;
        if ((st = check_kv(kv, maxp)) != LGX_OK) return st;
        if (!qkv || !rope || !seq_len || !page_table || !q_out) return fail(LGX_NULL_POINTER, "NULL tensor pointer");
        if (rope->rot > 0 && (!rope->cos_t || !rope->sin_t)) return fail(LGX_NULL_POINTER, "NULL cos / sin table");
        if (B <= 0 || N <= 0 || hq <= 0 || hq % kv->hkv != 0)
            return fail(LGX_INVALID_ARGUMENT, "B=%d N=%d hq=%d hkv=%d", B, N, hq, kv->hkv);
        if (rope->rot < 0 || rope->rot > kv->d || rope->rot % 2 || rope->max_pos <= 0 || rope->interleaved < 0 ||
            rope->interleaved > 1)
            return fail(LGX_INVALID_ARGUMENT, "rot %d of %d dimensions, max_pos %d, interleaved %d", rope->rot, kv->d,
                        rope->max_pos, rope->interleaved);
        const int64_t heads = (int64_t)hq + 2 * (int64_t)kv->hkv, rows = (int64_t)B * N;
        if (rows > INT32_MAX || heads > INT32_MAX / kv->d || rows > ((int64_t)1 << 33) / heads)
            return fail(LGX_OUT_OF_BOUNDS, "append of %lld rows of %lld heads", (long long)rows, (long long)heads);
        if (overlap(qkv, rows * heads * kv->d, q_out, rows * hq * kv->d))
            return fail(LGX_INVALID_ARGUMENT, "qkv and q_out overlap");
        const int per = 2048 / kv->d;                 // heads of a workgroup
        const int64_t wgs = (rows * heads + per - 1) / per;
        if (wgs > UINT32_MAX / 256) return fail(LGX_OUT_OF_BOUNDS, "append of %lld heads", (long long)(rows * heads));
        const int vec = rope->rot % 8 == 0 && aligned16(qkv) && aligned16(rope->cos_t) && aligned16(rope->sin_t) &&
                        aligned16(q_out);
        lgx_append_rows_args a{qkv, bias, rope->cos_t, rope->sin_t, seq_len, depth, n_new, page_table, kv->k, kv->v, q_out,
                               rows * heads, N, hq, kv->hkv, maxp, kv->num_pages, rope->max_pos, rope->rot,
                               rope->interleaved, vec};
        return launch(c, kv->d == 64 ? K_APPEND_ROWS_D64 : K_APPEND_ROWS_D128, dim3((unsigned)wgs), dim3(256), a, stream);
    });
}

lgx_status lgx_tree_plan(lgx_ctx* c, const int32_t* parent, const int32_t* n_nodes, int32_t B, int32_t N, int32_t* depth,
                         uint64_t* mask, void* stream) {
    return guarded(__func__, [&]() -> lgx_status {
        lgx_status st = enter(c);
        if (st != LGX_OK) return st;
        if (!parent || !depth || !mask) return fail(LGX_NULL_POINTER, "NULL tensor pointer");
        if ((st = check_tree(B, N)) != LGX_OK) return st;
        if (B > 1 << 23) return fail(LGX_OUT_OF_BOUNDS, "trees of %d sequences", B);
        lgx_tree_plan_args a{parent, n_nodes, depth, mask, N, (N + 63) / 64};
        return launch(c, K_TREE_PLAN, dim3((unsigned)B), dim3(LGX_TREE_NODES), a, stream);
    });
}

lgx_status lgx_tree_accept(lgx_ctx* c, const int32_t* tokens, const int32_t* parent, const int32_t* picked,
                           const int32_t* n_nodes, const int32_t* seq_len, int32_t B, int32_t N, int32_t* path,
                           int32_t* count, int32_t* next, int32_t* new_len, void* stream) {
    return guarded(__func__, [&]() -> lgx_status {
        lgx_status st = enter(c);
        if (st != LGX_OK) return st;
        if (!tokens || !parent || !picked || !path || !count || !next) return fail(LGX_NULL_POINTER, "NULL tensor pointer");
        if (new_len && !seq_len) return fail(LGX_NULL_POINTER, "new_len without seq_len");
        if ((st = check_tree(B, N)) != LGX_OK) return st;
        if (B > 1 << 25) return fail(LGX_OUT_OF_BOUNDS, "trees of %d sequences", B);
        lgx_tree_accept_args a{tokens, parent, picked, n_nodes, seq_len, path, count, next, new_len, N};
        return launch(c, K_TREE_ACCEPT, dim3((unsigned)B), dim3(64), a, stream);
    });
}

lgx_status lgx_kv_keep(lgx_ctx* c, const lgx_kv_f16* kv, int32_t layers, const int32_t* page_table, const int32_t* start,
                       const int32_t* keep, const int32_t* n_keep, int32_t B, int32_t N, int32_t maxp, void* stream) {
    return guarded(__func__, [&]() -> lgx_status {
        lgx_status st = enter(c);
        if (st != LGX_OK) return st;
        if (!kv) return fail(LGX_NULL_POINTER, "kv is NULL");
        if (!page_table || !start || !keep || !n_keep) return fail(LGX_NULL_POINTER, "NULL tensor pointer");
        if (layers <= 0 || B <= 0 || B > 1 << 23 || N <= 0 || N > 1 << 30)
            return fail(LGX_INVALID_ARGUMENT, "%d layers, B=%d, N=%d", layers, B, N);
        for (int i = 0; i < layers; ++i) {
            if ((st = check_kv(kv + i, maxp)) != LGX_OK) return st;
            if (kv[i].num_pages != kv->num_pages || kv[i].hkv != kv->hkv || kv[i].d != kv->d)
                return fail(LGX_INVALID_ARGUMENT, "layer %d's cache differs in shape", i);
        }
        if (kv->hkv > 4 * 65535) return fail(LGX_OUT_OF_BOUNDS, "%d heads", kv->hkv);
        for (int l0 = 0; l0 < layers; l0 += LGX_KEEP_PLANES / 2) {
            const int n = std::min(layers - l0, LGX_KEEP_PLANES / 2);
            lgx_kv_keep_args a{};
            for (int i = 0; i < n; ++i) {
                a.base[2 * i] = kv[l0 + i].k;
                a.base[2 * i + 1] = kv[l0 + i].v;
            }
            a.page_table = page_table;
            a.start = start;
            a.keep = keep;
            a.n_keep = n_keep;
            a.N = N;
            a.hkv = kv->hkv;
            a.maxp = maxp;
            a.num_pages = kv->num_pages;
            if ((st = launch(c, kv->d == 64 ? K_KV_KEEP_D64 : K_KV_KEEP_D128, dim3((unsigned)B, 2 * n, cdiv(kv->hkv, 4)),
                             dim3(256), a, stream)) != LGX_OK)
                return st;
        }
        return LGX_OK;
    });
}

lgx_status lgx_sample_filtered(lgx_ctx* c, const float* logits, int64_t ld, int32_t m, int32_t vocab,
                               const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                               const float* u, int32_t* out, float* prob, void* stream) {
    return guarded(__func__, [&]() -> lgx_status {
        lgx_status st = enter(c);
        if (st != LGX_OK) return st;
        if (!logits || !u || !out) return fail(LGX_NULL_POINTER, "NULL tensor");
        if (m <= 0 || m > 65535) return fail(LGX_INVALID_ARGUMENT, "m = %d", m);
        if (vocab <= 0 || vocab > LGX_SF_VOCAB)
            return fail(LGX_UNSUPPORTED, "vocab = %d outside [1, %d]", vocab, LGX_SF_VOCAB);
        if (ld < vocab || ld > INT64_MAX / 65536 / 4) return fail(LGX_INVALID_ARGUMENT, "rows %lld apart, vocab %d", (long long)ld, vocab);
        lgx_filter_args a{};
        a.logits = logits;
        a.temperature = temperature;
        a.top_k = top_k;
        a.top_p = top_p;
        a.min_p = min_p;
        a.u = u;
        a.out = out;
        a.prob = prob;
        a.ld = ld;
        a.m = m;
        a.vocab = vocab;
        a.nslices = (vocab + LGX_SF_SLICE - 1) / LGX_SF_SLICE;
        a.vec = ld % 4 == 0 && aligned16(logits);
        // room for the bins of as many wide rows as 64 MiB hold; the others take longer
        const size_t ns = (size_t)m * a.nslices, slot = (size_t)a.nslices * LGX_SF_BINS;
        // (a row of no more tokens than a workgroup lists is never wide)
        if ((top_p || min_p) && vocab > LGX_SF_LIST)
            a.slots = (int)std::min<size_t>(m, std::max<size_t>(((size_t)64 << 20) / 8 / slot, 1));
        const size_t eights = ns + m + (size_t)a.slots * slot;
        const size_t fours = ns * (1 + LGX_SF_SLICE / LGX_SF_CHUNK) + 2 * (size_t)m + 1 + a.slots;
        float* ws = nullptr;
        if ((st = ensure_ws(c, 8 * eights + 4 * fours, stream, &ws)) != LGX_OK) return st;
        a.sum = (double*)ws;
        a.wide_all = a.sum + ns;
        a.hist = (uint64_t*)(a.wide_all + m);
        a.smax = (float*)(a.hist + (size_t)a.slots * slot);
        a.cmax = a.smax + ns;
        a.wide_tau = a.cmax + ns * (LGX_SF_SLICE / LGX_SF_CHUNK);
        a.wide_row = (int32_t*)(a.wide_tau + m);
        a.wide_done = a.wide_row + m;
        a.wide_n = a.wide_done + a.slots;
        if ((st = launch(c, K_FILTER_SCAN, dim3((unsigned)a.nslices, (unsigned)m), dim3(256), a, stream)) != LGX_OK) return st;
        if ((st = launch(c, K_FILTER_PICK, dim3((unsigned)m), dim3(1024), a, stream)) != LGX_OK || !a.slots) return st;
        return launch(c, K_FILTER_WIDE, dim3((unsigned)std::min<size_t>(ns, 2 * (size_t)c->ncu)), dim3(1024), a, stream);
    });
}

}  // extern "C"
