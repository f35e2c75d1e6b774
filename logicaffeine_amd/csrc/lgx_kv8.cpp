// lgx_kv8.cpp -- the 8-bit KV cache: rotary tables, append, read-back, and the
// attention of decode and prefill rows over it (kernels in lgx_kv8.hip).
#include <algorithm>
#include <cmath>

#include "lgx_internal.h"

using namespace lgxi;

namespace {

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

lgx_status check_kv(const lgx_kv_i8* kv, int32_t maxp) {
    if (!kv) return fail(LGX_NULL_POINTER, "kv is NULL");
    if (!kv->k || !kv->v || !kv->k_scale || !kv->v_scale) return fail(LGX_NULL_POINTER, "NULL cache pointer");
    if (kv->num_pages <= 0 || kv->hkv <= 0 || maxp <= 0 || maxp > 1 << 26)
        return fail(LGX_INVALID_ARGUMENT, "num_pages=%d hkv=%d maxp=%d", kv->num_pages, kv->hkv, maxp);
    if (kv->d != 64 && kv->d != 128) return fail(LGX_UNSUPPORTED, "head_dim %d (64 or 128)", kv->d);
    if (!aligned16(kv->k) || !aligned16(kv->v))
        return fail(LGX_INVALID_ARGUMENT, "cache pages must be 16-byte aligned");
    return LGX_OK;
}

// Pages that n tokens from any slot on can touch.
int pages_touched(int n) { return (int)(((int64_t)n + LGX_PAGE - 2) / LGX_PAGE + 1); }

// (row, head) pairs of a workgroup, for `heads` (sequence, KV head) pairs of `cols`
// each over up to `tiles` tiles of 64 tokens (of max_seq_len: the lengths are on the
// device).  16 and 32 go over a tile's tokens with all four waves, 128 over its columns.
// Measured on the 0.5B-, 1.5B- and 7B-shaped heads (us with 16 / 32 / 128):
//  - 128 from 512 workgroups on, two per compute unit: 8 x 512 rows at 4000 tokens
//    (7B-shaped, 896 workgroups) 581 / 449 / 437, 8 x 1024 at 1100 (1792) 346 / 286 /
//    196; below 8 x 256 at 4000 (448) 299 / 237 / 231, 16 x 256 at 2000
//    (1.5B-shaped, 384) 149 / 116 / 121;
//  - 32, which read K and V half as often and convert V for twice the columns, from
//    about 12000 tiles of 16 columns on at head dimension 128: 16 x 64 at 500 (14300)
//    40.3 / 38.2, 8 x 64 at 2000 (28700) 53.2 / 43.6, 1 x 256 at 4000 (28200) 47.0 / 48.7;
//    below 16 x 64 at 700 (1.5B-shaped, 8400) 23.4 / 24.2, 2 x 64 at 2000 (7200)
//    22.4 / 26.7; at 64, where a tile's work is half as long, from about 65000: 8 x 512 at
//    2000 (0.5B-shaped, 115000) 87.0 / 86.0, 8 x 128 at 4000 (56000) 53.6 / 48.9, 4 x 256
//    at 1000 (14000) 18.8 / 19.4.
int attn8_cols(const lgx_ctx* c, int64_t heads, int64_t cols, int64_t tiles, int d) {
    if (c->attn8_cols == 16 || c->attn8_cols == 32 || c->attn8_cols == 128) return c->attn8_cols;
    if (cols <= 16) return 16;
    if (heads * ((cols + 127) / 128) >= 2 * (int64_t)c->ncu) return 128;
    return heads * ((cols + 15) / 16) * tiles >= (d == 64 ? 65536 : 12288) ? 32 : 16;
}

// Launch over B sequences.  Where there are fewer (sequence, KV head, column block)s
// than compute units (times attn8_wgs), their tiles are split among that many
// workgroups; the splitting itself is done on the device, by the lengths.  From there
// on each is one workgroup's, also a sequence far longer than the others.
lgx_status run_attn8(lgx_ctx* c, lgx_attn8_args& a, int B, int d, bool x, void* stream) {
    const int64_t cols = (int64_t)a.P * (a.hq / a.hkv), heads = (int64_t)B * a.hkv;
    // the most tiles that a block can see (its rows are at most 128 apart)
    int64_t tiles = cdiv(a.maxlen, LGX_A8_TILE);
    if (a.window) tiles = std::min<int64_t>(tiles, ((int64_t)a.window + 128) / LGX_A8_TILE + 2);
    const int nc = attn8_cols(c, heads, cols, tiles, d);
    const int64_t ncb = (cols + nc - 1) / nc, units = B * ncb, blocks = heads * ncb;
    a.ncb = (int)ncb;
    a.cols = nc;
    int64_t per = (int64_t)c->attn8_wgs * c->ncu / a.hkv;
    bool split = tiles > LGX_A8_MIN && units <= LGX_A8_UNITS && units < per;
    if (split && units == 1 && !a.window) {
        a.cps = (int)std::max<int64_t>(LGX_A8_MIN, ((tiles + per - 1) / per + 3) / 4 * 4);
        per = (tiles + a.cps - 1) / a.cps;
        if (per == 1) split = false, a.cps = 0;
    }
    lgx_status st;
    if (split) {
        const int64_t slots = per * a.hkv * nc;
        float* ws = nullptr;
        if ((st = ensure_ws(c, (size_t)(slots * (d + 2) + 2 * units) * sizeof(float), stream, &ws)) != LGX_OK) return st;
        a.per = (int)per;
        a.units = (int)units;
        a.part = ws;
        a.ml = ws + slots * d;
        a.plan = (int32_t*)(a.ml + 2 * slots);
    }
    const int64_t grid = split ? per * a.hkv : blocks;
    if (grid > UINT32_MAX / 256) return fail(LGX_OUT_OF_BOUNDS, "attention of %lld workgroups", (long long)grid);
    const int k = (d == 64 ? K_ATTN8_D64 : K_ATTN8_D128) + (nc == 16 ? 0 : nc == 32 ? 2 : 4) + (x ? 1 : 0);
    if ((st = launch(c, (Kern)k, dim3((unsigned)grid), dim3(256), a, stream)) != LGX_OK || !split) return st;
    // a wave joins a row's head where there are many; a workgroup, whose threads
    // read more splits at a time, where there are few
    const int64_t rh = (int64_t)a.rows * a.hq;
    const int w = rh >= 8 * (int64_t)c->ncu ? 1 : 0;
    return launch(c, (Kern)((d == 64 ? K_ATTN8_JOIN_D64 : K_ATTN8_JOIN_D128) + w), dim3(w ? cdiv(rh, 4) : (unsigned)rh),
                  dim3(256), a, stream);
}

lgx_status attn8(lgx_ctx* c, const float* q, const lgx_kv_i8* kv, const int32_t* page_table,
                 const int32_t* seq_len, const int32_t* n_new, int32_t B, int32_t P, int32_t hq, int32_t maxp,
                 int32_t max_seq_len, const lgx_attn_opts* opts, int len_add, float* out, void* stream) {
    lgx_status st = enter(c);
    if (st != LGX_OK) return st;
    if ((st = check_kv(kv, maxp)) != LGX_OK) return st;
    if (!q || !page_table || !seq_len || !out) return fail(LGX_NULL_POINTER, "NULL tensor pointer");
    if (B <= 0 || P <= 0 || hq <= 0 || hq % kv->hkv != 0)
        return fail(LGX_INVALID_ARGUMENT, "B=%d P=%d hq=%d hkv=%d", B, P, hq, kv->hkv);
    if (hq / kv->hkv > 16) return fail(LGX_UNSUPPORTED, "%d query heads per KV head (1..16)", hq / kv->hkv);
    if (max_seq_len <= 0 || max_seq_len > maxp * LGX_PAGE)
        return fail(LGX_OUT_OF_BOUNDS, "max_seq_len %d outside (0, %d]", max_seq_len, maxp * LGX_PAGE);
    if ((int64_t)B * P * hq > INT32_MAX / 128) return fail(LGX_OUT_OF_BOUNDS, "B*P*hq too large");
    if (!aligned16(q) || !aligned16(out)) return fail(LGX_INVALID_ARGUMENT, "q and out must be 16-byte aligned");
    lgx_attn8_args a{};
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
    a.ks = kv->k_scale;
    a.vs = kv->v_scale;
    a.page_table = page_table;
    a.seq_len = seq_len;
    a.n_new = n_new;
    a.out = out;
    a.P = P;
    a.hq = hq;
    a.hkv = kv->hkv;
    a.maxp = maxp;
    a.num_pages = kv->num_pages;
    a.maxlen = max_seq_len;
    a.len_add = len_add;
    a.rows = B * P;
    return run_attn8(c, a, B, kv->d, a.softcap > 0.0f || a.window > 0 || a.slopes != nullptr || a.scale < 0.0f, stream);
}

}  // namespace

extern "C" {

lgx_status lgx_rope_tables(int32_t max_pos, int32_t rot, double theta, const lgx_rope_scaling* sc, float* cos_t,
                           float* sin_t) {
    return guarded(__func__, [&]() -> lgx_status {
        g_has_error = false;
        if (!cos_t || !sin_t) return fail(LGX_NULL_POINTER, "NULL table");
        if (max_pos <= 0 || rot <= 0 || rot % 2 || !(theta > 0.0) || !std::isfinite(theta))
            return fail(LGX_INVALID_ARGUMENT, "max_pos %d, rot %d, theta %g", max_pos, rot, theta);
        const int kind = sc ? sc->kind : LGX_ROPE_PLAIN, half = rot / 2;
        if (kind < LGX_ROPE_PLAIN || kind > LGX_ROPE_PARTS)
            return fail(LGX_INVALID_ARGUMENT, "rotary scaling kind %d", kind);
        if (kind != LGX_ROPE_PLAIN && (!(sc->factor >= 1.0) || !std::isfinite(sc->factor)))
            return fail(LGX_INVALID_ARGUMENT, "rotary scaling factor %g (>= 1)", sc->factor);
        if (kind == LGX_ROPE_PARTS &&
            (sc->original_len <= 0 || !(sc->slow >= 0.0) || !(sc->fast > sc->slow) || !std::isfinite(sc->fast)))
            return fail(LGX_INVALID_ARGUMENT, "original_len %d, slow %g, fast %g", sc->original_len, sc->slow, sc->fast);
        if (kind == LGX_ROPE_BASE && rot > 2) theta *= std::pow(sc->factor, (double)rot / (rot - 2));
        std::vector<double> w(half);
        double amp = 1.0;
        for (int i = 0; i < half; ++i) {
            w[i] = std::pow(theta, -2.0 * i / rot);
            if (kind == LGX_ROPE_LINEAR) w[i] /= sc->factor;
            if (kind == LGX_ROPE_PARTS) {
                const double turns = sc->original_len * w[i] / (2.0 * M_PI);
                const double keep = std::min(std::max((turns - sc->slow) / (sc->fast - sc->slow), 0.0), 1.0);
                w[i] = w[i] * keep + w[i] / sc->factor * (1.0 - keep);
            }
        }
        if (kind == LGX_ROPE_PARTS) amp = 0.1 * std::log(sc->factor) + 1.0;
        for (int64_t p = 0; p < max_pos; ++p)
            for (int i = 0; i < half; ++i) {
                const double x = (double)p * w[i];
                cos_t[p * half + i] = (float)(amp * std::cos(x));
                sin_t[p * half + i] = (float)(amp * std::sin(x));
            }
        return LGX_OK;
    });
}

lgx_status lgx_rope_kv_append_i8(lgx_ctx* c, const float* qkv, const float* bias, const lgx_rope* rope,
                                 const int32_t* seq_len, const int32_t* n_new, const int32_t* page_table,
                                 const lgx_kv_i8* kv, float* q_out, int32_t B, int32_t P, int32_t hq, int32_t maxp,
                                 void* stream) {
    return guarded(__func__, [&]() -> lgx_status {
        lgx_status st = enter(c);
        if (st != LGX_OK) return st;
        if ((st = check_kv(kv, maxp)) != LGX_OK) return st;
        if (!qkv || !rope || !seq_len || !page_table || !q_out) return fail(LGX_NULL_POINTER, "NULL tensor pointer");
        if (rope->rot > 0 && (!rope->cos_t || !rope->sin_t)) return fail(LGX_NULL_POINTER, "NULL cos / sin table");
        if (B <= 0 || P <= 0 || hq <= 0 || hq % kv->hkv != 0)
            return fail(LGX_INVALID_ARGUMENT, "B=%d P=%d hq=%d hkv=%d", B, P, hq, kv->hkv);
        if (rope->rot < 0 || rope->rot > kv->d || rope->rot % 2 || rope->max_pos <= 0 || rope->interleaved < 0 ||
            rope->interleaved > 1)
            return fail(LGX_INVALID_ARGUMENT, "rot %d of %d dimensions, max_pos %d, interleaved %d", rope->rot, kv->d,
                        rope->max_pos, rope->interleaved);
        if (!aligned16(q_out)) return fail(LGX_INVALID_ARGUMENT, "q_out must be 16-byte aligned");
        const int64_t nblk = pages_touched(P), heads = (int64_t)hq + 2 * kv->hkv;
        if (B * nblk > UINT32_MAX / 256 || heads > 65535)
            return fail(LGX_OUT_OF_BOUNDS, "append of %d x %d rows, %lld heads", B, P, (long long)heads);
        lgx_kv8_append_args a{qkv, bias, rope->cos_t, rope->sin_t, seq_len, n_new, page_table, kv->k, kv->v,
                              kv->k_scale, kv->v_scale, q_out, P, hq, kv->hkv, maxp, kv->num_pages, rope->max_pos,
                              rope->rot, rope->interleaved, (int32_t)nblk, 0};
        const bool d64 = kv->d == 64;
        if (P == 1)
            return launch(c, d64 ? K_KV8_APPEND1_D64 : K_KV8_APPEND1_D128, dim3((unsigned)B, cdiv(heads, 4)), dim3(256), a,
                          stream);
        // a thread's d / 32 pairs in 16- or 8-byte pieces
        a.vec = rope->rot / 2 % (kv->d / 32) == 0 && aligned16(qkv) && aligned16(bias) && aligned16(rope->cos_t) &&
                aligned16(rope->sin_t);
        return launch(c, d64 ? K_KV8_APPEND_D64 : K_KV8_APPEND_D128,
                      dim3((unsigned)(B * nblk), cdiv(hq, LGX_KV8_QH) + 2 * kv->hkv), dim3(256), a, stream);
    });
}

lgx_status lgx_kv_read_i8(lgx_ctx* c, const lgx_kv_i8* kv, const int32_t* page_table, const int32_t* start, int32_t B,
                          int32_t n, int32_t maxp, float* k_out, float* v_out, void* stream) {
    return guarded(__func__, [&]() -> lgx_status {
        lgx_status st = enter(c);
        if (st != LGX_OK) return st;
        if ((st = check_kv(kv, maxp)) != LGX_OK) return st;
        if (!page_table || !start || !k_out || !v_out) return fail(LGX_NULL_POINTER, "NULL tensor pointer");
        if (B <= 0 || n <= 0) return fail(LGX_INVALID_ARGUMENT, "B=%d n=%d", B, n);
        if (!aligned16(k_out) || !aligned16(v_out))
            return fail(LGX_INVALID_ARGUMENT, "k_out and v_out must be 16-byte aligned");
        const int64_t nblk = pages_touched(n);
        if (B * nblk > UINT32_MAX / 256 || kv->hkv > 65535)
            return fail(LGX_OUT_OF_BOUNDS, "read of %d x %d tokens, %d heads", B, n, kv->hkv);
        lgx_kv8_read_args a{kv->k, kv->v, kv->k_scale, kv->v_scale, page_table, start, k_out, v_out,
                            n, kv->hkv, maxp, kv->num_pages, (int32_t)nblk};
        return launch(c, kv->d == 64 ? K_KV8_READ_D64 : K_KV8_READ_D128, dim3((unsigned)(B * nblk), (unsigned)kv->hkv),
                      dim3(256), a, stream);
    });
}

lgx_status lgx_gqa_decode_attn_i8(lgx_ctx* c, const float* q, const lgx_kv_i8* kv, const int32_t* page_table,
                                  const int32_t* seq_len, int32_t B, int32_t hq, int32_t maxp, int32_t max_seq_len,
                                  const lgx_attn_opts* opts, float* out, void* stream) {
    return guarded(__func__, [&] {
        return attn8(c, q, kv, page_table, seq_len, nullptr, B, 1, hq, maxp, max_seq_len, opts, 0, out, stream);
    });
}

lgx_status lgx_gqa_prefill_attn_i8(lgx_ctx* c, const float* q, const lgx_kv_i8* kv, const int32_t* page_table,
                                   const int32_t* seq_len, const int32_t* n_new, int32_t B, int32_t P, int32_t hq,
                                   int32_t maxp, int32_t max_seq_len, const lgx_attn_opts* opts, float* out,
                                   void* stream) {
    return guarded(__func__, [&] {
        return attn8(c, q, kv, page_table, seq_len, n_new, B, P, hq, maxp, max_seq_len, opts, 1, out, stream);
    });
}

}  // extern "C"
