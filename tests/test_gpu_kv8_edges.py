"""The 8-bit KV cache at the edges of what its calls take, against the definition."""
from fractions import Fraction

import numpy as np
import pytest

import kv8_ref as ref
import logicaffeine_amd as lgx

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24                                     # half a step of binary32


def host(t):
    return t.cpu().numpy()


def upload(ctx, cache):
    return lgx.KvCacheI8(*(ctx.to_device(x) for x in (cache.k, cache.v, cache.ks, cache.vs)))


def i32(ctx, x):
    return ctx.to_device(np.asarray(x, np.int32))


def no_rope(ctx):
    t = ctx.torch
    return lgx.Rope(t.empty((1, 0), device=ctx.dev), t.empty((1, 0), device=ctx.dev))


# ---- append ---------------------------------------------------------------

def nearest(y, scale):
    """The whole number nearest to y / scale, halves away from zero, exactly."""
    r = abs(Fraction(float(y))) / Fraction(float(scale))
    m = (r + Fraction(1, 2)).__floor__()
    return -m if y < 0 else m


def tie_rows(n, d, scale, rng):
    """n rows of d numbers whose quotients by `scale` are halves and their neighbours,
    the first number 127 scale."""
    k = rng.integers(0, 127, (n, d))
    y = ((k + 0.5) * scale).astype(np.float32)
    assert (y.astype(np.float64) == (k + 0.5) * scale).all()
    y[1::3] = np.nextafter(y[1::3], np.float32(0))
    y[2::3] = np.nextafter(y[2::3], np.float32(np.inf))
    y *= rng.choice(np.float32([-1, 1]), y.shape)
    y[0, 0] = 127 * scale
    return y


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("P", [1, 9, 16])
def test_quants_at_exact_ties(ctx, P, d):
    """quant = the nearest integer to value / scale, halves away from zero: also where
    value * (1 / scale) would round to the other side of the half."""
    rng, hkv, hq = np.random.default_rng(P + d), 1, 1
    scales = np.arange(3, 3 + 2 * 200, 2)            # odd numbers: their reciprocals are rounded
    B = len(scales)
    x = np.zeros((B, P, 3, d), np.float32)
    for b, s in enumerate(scales):
        x[b, :, 1], x[b, :, 2] = tie_rows(P, d, s, rng), tie_rows(P, d, s, rng)
    kv = lgx.KvCacheI8.empty(ctx, B, hkv, d)
    ctx.rope_kv_append_i8(ctx.to_device(x.reshape(B * P, 3 * d)), None, no_rope(ctx), i32(ctx, [0] * B),
                          i32(ctx, np.arange(B).reshape(B, 1)), kv, P)
    assert np.array_equal(host(kv.k_scale)[:, 0], scales) and np.array_equal(host(kv.v_scale)[:, 0], scales)
    want = np.array([[[nearest(y, s) for y in row] for row in x[b, :, 1:].reshape(-1, d)] for b, s in enumerate(scales)])
    want = want.reshape(B, P, 2, d)
    assert np.array_equal(host(kv.k)[:, 0, :P], want[:, :, 0])
    assert np.array_equal(host(kv.v)[:, 0, :, :P].transpose(0, 2, 1), want[:, :, 1])


@pytest.mark.parametrize("P", [1, 5])
def test_quants_next_to_a_tie_in_64_bits(ctx, P):
    """bias + row is a binary64 number: 1/2 - 2^-54 is nearer to 0 than to 1."""
    d, hkv = 64, 1
    x = np.zeros((P, 3, d), np.float32)
    x[:, 1:] = np.float32(-2.0 ** -54)
    x[0, 1:, 0] = 126.5
    bias = np.full(3 * d, 0.5, np.float32)
    kv = lgx.KvCacheI8.empty(ctx, 1, hkv, d)
    ctx.rope_kv_append_i8(ctx.to_device(x.reshape(P, 3 * d)), ctx.to_device(bias), no_rope(ctx), i32(ctx, [0]), i32(ctx, [[0]]), kv, P)
    want = np.zeros((P, d), np.int8)
    want[0, 0] = 127
    assert host(kv.k_scale)[0, 0] == 1.0 and host(kv.v_scale)[0, 0] == 1.0
    assert np.array_equal(host(kv.k)[0, 0, :P], want) and np.array_equal(host(kv.v)[0, 0, :, :P].T, want)


@pytest.mark.parametrize("d", [64, 128])
def test_growth_at_every_fill_of_a_page(ctx, d):
    """One row per sequence into pages that hold 1 .. 15 tokens, blocks that double 0 to
    12 times, scales of zero among them."""
    rng, hq, hkv, B = np.random.default_rng(d), 2, 2, 15 * 14
    cache, table = ref.Cache(B, hkv, d, rng), rng.permutation(B).astype(np.int32).reshape(B, 1)
    lens, grow = np.repeat(np.arange(1, 16), 14), np.tile(np.arange(14), 15)
    x = rng.standard_normal((B, 1, (hq + 2 * hkv) * d)).astype(np.float32)
    for b in range(B):
        top = np.abs(x[b]).max() / 127
        cache.ks[table[b, 0]] = cache.vs[table[b, 0]] = 0.0 if grow[b] == 13 else np.float32(top * 1.5 / 2.0 ** grow[b])
    kv = upload(ctx, cache)
    ctx.rope_kv_append_i8(ctx.to_device(x[:, 0]), None, no_rope(ctx), i32(ctx, lens), i32(ctx, table), kv)
    before = [cache.k.copy(), cache.v.copy()]
    cache.append(x, None, *ref.tables(16, 0), False, lens, None, table, hq)
    for got, want in ((kv.k, cache.k), (kv.v, cache.v), (kv.k_scale, cache.ks), (kv.v_scale, cache.vs)):
        assert np.array_equal(host(got), want)
    assert all((a != b).any((1, 2, 3)).all() for a, b in zip(before, (cache.k, cache.v)))


@pytest.mark.parametrize("P", [1, 2, 20])
def test_a_sequence_without_new_rows_touches_nothing(ctx, P):
    """Row counts of zero and below: the page that the length points into keeps its
    scale's bits, whatever they are, and its quants."""
    rng, hq, hkv, d = np.random.default_rng(P), 2, 2, 64
    lens, new = [5, 15, 16, 20, 3], [0, -3, 0, 0, 1]
    B, maxp = len(lens), 4
    cache, table = ref.Cache(B * maxp, hkv, d, rng), rng.permutation(B * maxp).astype(np.int32).reshape(B, maxp)
    for b, v in enumerate((np.inf, -1.0, np.nan, -np.inf)):
        cache.ks[table[b]] = cache.vs[table[b]] = np.float32(v)
    # a number of its own payload, so that a NaN written back in another form would show
    cache.ks.view(np.uint32)[table[2]] = cache.vs.view(np.uint32)[table[2]] = 0x7fc01234
    kv = upload(ctx, cache)
    x = rng.standard_normal((B, P, (hq + 2 * hkv) * d)).astype(np.float32)
    ctx.rope_kv_append_i8(ctx.to_device(x.reshape(B * P, -1)), None, no_rope(ctx), i32(ctx, lens), i32(ctx, table), kv, P,
                          n_new=i32(ctx, new))
    cache.append(x, None, *ref.tables(64, 0), False, lens, new, table, hq)
    for got, want in ((kv.k, cache.k), (kv.v, cache.v), (kv.k_scale, cache.ks), (kv.v_scale, cache.vs)):
        assert host(got).tobytes() == want.tobytes()


@pytest.mark.parametrize("P", [1, 20])
def test_an_idle_row_names_pages_that_others_append_to(ctx, P):
    """Slots of a padded batch that have no sequence any more: their table rows still name
    pages that other sequences of the same call append to, and whose blocks grow."""
    rng, hq, hkv, d, B = np.random.default_rng(P), 2, 2, 64, 32
    maxp = 3
    lens, new = rng.integers(1, 16, B), np.where(np.arange(B) % 2, 0, P)
    cache, table = ref.Cache(B * maxp, hkv, d, rng), rng.permutation(B * maxp).astype(np.int32).reshape(B, maxp)
    table[1::2] = table[0::2]                        # an idle row for each live one, inside the same page
    lens[1::2] = lens[0::2]
    x = (rng.standard_normal((B, P, (hq + 2 * hkv) * d)) * 1e3).astype(np.float32)
    want = ref.Cache(B * maxp, hkv, d)
    want.k, want.v, want.ks, want.vs = (a.copy() for a in (cache.k, cache.v, cache.ks, cache.vs))
    want.append(x, None, *ref.tables(64, 0), False, lens, new, table, hq)
    for _ in range(5):
        kv = upload(ctx, cache)
        ctx.rope_kv_append_i8(ctx.to_device(x.reshape(B * P, -1)), None, no_rope(ctx), i32(ctx, lens), i32(ctx, table), kv, P,
                              n_new=i32(ctx, new))
        for got, w in ((kv.k, want.k), (kv.v, want.v), (kv.k_scale, want.ks), (kv.v_scale, want.vs)):
            assert np.array_equal(host(got), w)


# ---- attention ------------------------------------------------------------

def attend(cache, q, table, seq_len, prefill, scale=None, slopes=None):
    """q [B][P][hq][d] -> (float64 results, bound element by element).

    The bound counts nothing that its weight takes away.  A score that is off by e changes
    the result by at most sum(w e |v|) + sum(w e) sum(w |v|).  e: q to half a step of
    max|q| / 4161536 per product; eight binary32 roundings of the score, four of the
    distance term and of the difference to the maximum.  A weight with its V scale, w vs:
    22 bits, and no better than 2^-34 of the row's largest w vs (the subnormal end of
    binary16); exp2 to one unit; n / 32 + 64 partial sums twice over in binary32."""
    B, P, hq, d = q.shape
    G = hq // cache.hkv
    scale = 1.0 / np.sqrt(d) if scale is None else scale
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(B):
        for j in range(P):
            L = int(seq_len[b]) + j + (1 if prefill else 0)
            k, v = cache.rows(table[b], L)
            pages = np.arange(L) // 16
            back = (L - 1 - np.arange(L)).astype(np.float64)
            for h in range(hq):
                kk, vv, qq = k[:, h // G], v[:, h // G], q[b, j, h].astype(np.float64)
                vs = cache.vs[table[b][pages], h // G].astype(np.float64)
                raw = kk @ qq * scale
                far = slopes[h].astype(np.float64) * back if slopes is not None else 0.0 * back
                s = raw - far
                w = np.exp(s - s.max())
                w /= w.sum()
                out[b, j, h] = w @ vv
                e = np.abs(qq).max() / (127 * 65536) * abs(scale) * np.abs(kk).sum(1) + EPS * (
                    8 * np.abs(raw) + 4 * np.abs(far) + 4 * np.abs(s - s.max()))
                size = w @ np.abs(vv)
                step = 2.0 ** -34 * (w * vs).max() * np.abs(np.divide(vv, vs[:, None], out=np.zeros_like(vv), where=vs[:, None] > 0)).sum(0)
                bound[b, j, h] = (w * e) @ np.abs(vv) + (w @ e) * size + EPS * (8 + 2 * (L / 32 + 64)) * size + step
    return out, bound


def check(got, want, bound, tight):
    """Within the bound, which itself is a small part of each row's largest result."""
    assert (bound.max(-1) <= tight * np.abs(want).max(-1)).all(), (bound.max(-1) / np.abs(want).max(-1)).max()
    worst = np.abs(got - want) - bound
    assert (worst <= 0).all(), (worst.max(), np.unravel_index(worst.argmax(), worst.shape))


def far_scales(rng, d, hkv, pages, kind, ratio):
    """A cache whose heavy pages (weights next to one) and whose large pages are others.
    "faint": the large pages weigh e^-300; "hollow": the heavy pages' V is `ratio`
    times the others' (0: all zero), which weigh about e^-15."""
    cache = ref.Cache(pages, hkv, d, rng)
    heavy = rng.random(pages) < 0.5
    heavy[0], heavy[1] = True, False
    # q is about 1 in every dimension: a score is 8 (or 11.3) times scale and mean quant
    cache.ks[:] = np.float32(0.5)
    gap = {"faint": 300.0, "hollow": 15.0}[kind]
    drop = int(round(gap / (np.sqrt(d) * 0.5)))
    cache.k[:] = rng.integers(18, 23, cache.k.shape)
    cache.k[~heavy] -= np.int8(drop)
    cache.vs[:] = np.float32(0.01)
    cache.vs[~heavy if kind == "faint" else heavy] *= np.float32(ratio)
    return cache


FAR = [("faint", 1e6), ("faint", 1e9), ("faint", 1e15), ("faint", 1e30), ("hollow", 0.0), ("hollow", 1e-20), ("hollow", 1e-6)]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("cols", [16, 32, 128])
@pytest.mark.parametrize("kind,ratio", FAR)
def test_v_scales_do_not_cost_the_pages_that_matter(monkeypatch, d, cols, kind, ratio):
    """V scales count by the weight that meets them, in every kernel, in any order of the
    pages, split among workgroups or not."""
    monkeypatch.setenv("LGX_A8_COLS", str(cols))
    c = lgx.Context(0)
    try:
        rng = np.random.default_rng(d + cols)
        hq, hkv, P, maxp = 4, 2, 40, 30
        cache = far_scales(rng, d, hkv, 2 * maxp, kind, ratio)
        table = np.stack([rng.permutation(2 * maxp)[:maxp] for _ in range(2)]).astype(np.int32)
        q = (1 + 0.02 * rng.standard_normal((2, P, hq, d))).astype(np.float32)
        lens = [maxp * 16 - P, 150]
        kv, tab = upload(c, cache), i32(c, table)
        got = host(c.gqa_prefill_attn_i8(c.to_device(q.reshape(2 * P, hq, d)), kv, tab, i32(c, lens), P, maxp * 16))
        check(got.reshape(q.shape), *attend(cache, q, table, lens, True), tight=1e-3)
        got = host(c.gqa_decode_attn_i8(c.to_device(q[:, 0].copy()), kv, tab, i32(c, lens), maxp * 16))
        want, bound = attend(cache, q[:, :1], table, lens, False)
        check(got, want[:, 0], bound[:, 0], tight=1e-3)
    finally:
        c.close()


@pytest.mark.parametrize("ratio", [1e6, 1e9, 1e20])
@pytest.mark.parametrize("P", [1, 70])
def test_distance_bias_hides_far_pages_of_large_values(ctx, P, ratio):
    """Pages whose distance leaves them no weight, with values far above the near ones'."""
    rng, hq, hkv, d, maxp = np.random.default_rng(P), 4, 2, 64, 40
    cache = ref.Cache(maxp, hkv, d, rng)
    cache.vs[: maxp // 2] *= np.float32(ratio)
    table = np.arange(maxp, dtype=np.int32)[None]
    q = rng.standard_normal((1, P, hq, d)).astype(np.float32)
    lens, slopes = [maxp * 16 - P + (P == 1)], np.float32([2.0, 3.0, 1.5, 2.5])
    opts = lgx.AttnOpts(slopes=ctx.to_device(slopes))
    want, bound = attend(cache, q, table, lens, P > 1, slopes=slopes)
    if P == 1:
        got = ctx.gqa_decode_attn_i8(ctx.to_device(q[:, 0]), upload(ctx, cache), i32(ctx, table), i32(ctx, lens), maxp * 16, opts)
    else:
        got = ctx.gqa_prefill_attn_i8(ctx.to_device(q[0]), upload(ctx, cache), i32(ctx, table), i32(ctx, lens), P, maxp * 16, opts=opts)
    check(host(got).reshape(want.shape), want, bound, tight=1e-3)


def cut_in_groups(cache, q, table, n, g):
    """How much of a row's result the groups of eight products lose at most in the mean,
    relative to it (V of one scale and sign)."""
    k, v = cache.rows(table, n)
    s = k[:, g] @ q.astype(np.float64) / np.sqrt(cache.d)
    vs = float(cache.vs[0, g])
    w, m = np.exp(s - s.max()) * vs, -(-n // 8) * 8
    w, v = np.pad(w, (0, m - n)), np.pad(v[:, g] / vs, ((0, m - n), (0, 0)))
    p = (w[:, None] * v).reshape(-1, 8, cache.d)
    step = 2.0 ** (np.floor(np.log2(p.max(1, keepdims=True))) - 24)
    last = 2.0 ** (np.floor(np.log2(np.maximum(w, 1e-300))) - 10).reshape(-1, 8, 1)
    return (np.where(last >= step, 0.0, np.minimum(p, step / 2)).sum((0, 1)) / p.sum((0, 1))).mean()


@pytest.mark.parametrize("cols", [16, 128])
def test_weights_are_rounded_without_a_bias(monkeypatch, cols):
    """Values of one sign: what the weights' roundings put on a result has no mean.  Each
    row's weights are off by at most 2^-22 in all, to either side, independently of the
    other rows': over 2048 rows the mean deviates by less than 2^-22 / sqrt(3 * 2048) = 3.0e-9
    (cut weights: 7.5e-8).  Five deviations, and the last roundings' of the results (2^-24 /
    sqrt(3 * 2048 * 64), 1e-10), are 1.6e-8.

    Beside this the matrix unit itself: it adds products in groups of eight (a lane's, here
    eight tokens of a page), each cut toward zero at 2^-24 of the binade of the group's largest:
    1 - 1 + 7 * 2^-25 gives 0 there, and 1 - 1 + 7 * 1.9375 * 2^-20 loses what lies below 2^-24
    of each.  `lost` takes half of that step from every product that has bits below it (a
    first part has 11 bits, a quant's are whole numbers), as much as the mean can lose."""
    monkeypatch.setenv("LGX_A8_COLS", str(cols))
    c = lgx.Context(0)
    try:
        rng, hq, hkv, d, B, P = np.random.default_rng(cols), 8, 2, 64, 4, 64
        L, maxp = 100, 11
        cache = ref.Cache(B * maxp, hkv, d, rng)
        cache.v[:] = np.abs(cache.v.astype(np.int16)).clip(1, 127)
        cache.vs[:] = np.float32(0.01)
        table = rng.permutation(B * maxp).astype(np.int32).reshape(B, maxp)
        q = rng.standard_normal((B, P, hq, d)).astype(np.float32)
        got = host(c.gqa_prefill_attn_i8(c.to_device(q.reshape(B * P, hq, d)), upload(c, cache), i32(c, table), i32(c, [L] * B),
                                         P, L + P)).reshape(q.shape)
        want, _ = attend(cache, q, table, [L] * B, True)
        lost = np.mean([cut_in_groups(cache, q[b, j, h], table[b], L + j + 1, h // (hq // hkv))
                        for b in range(B) for j in range(P) for h in range(hq)])
        mean = ((got - want) / want).mean()
        assert -1.6e-8 - lost <= mean <= 1.6e-8, (mean, lost)
    finally:
        c.close()


def test_a_sink_among_many_tokens(monkeypatch):
    """One token with half of the weight before 131072 others, all in one wave: their
    weights' second parts are subnormal, and rounded, not cut.

    In units in which the sink's weight is 2^10 at least theirs are 2^-7 and off by 2^-25
    at most, to either side: 1008 distinct weights of a head that come again and again put
    2^-18 / sqrt(3 * 1008) / 2 on the result, 3.5e-8.  The sums: 63 pages come again 32.5
    times in each of the column's four lanes and in the tiles, and a sum that stays in its
    binade rounds them alike each time, by 2^-24 at most.  The weights' sum: the lane that
    holds the sink 32.5 sqrt(63 / 3) 2^-24 = 8.9e-6, the three others, a quarter of it high,
    2.2e-6 each, of a total of 2: 4.8e-6 on all of a head.  A dimension's sum, up to twice as
    high, 8.9e-6, over a head's 64 dimensions 1.1e-6.  Together 4.9e-6 for a head, 3.1e-7 for
    the mean over 256 of them, where cut weights lack 2^-17 of the others' half, 3.8e-6, and
    sums whose second parts fall below half a step of the first ones' lack 2^-13 of it,
    1.2e-4.  Five deviations are allowed."""
    monkeypatch.setenv("LGX_A8_COLS", "128")
    monkeypatch.setenv("LGX_A8_WGS", "1")
    c = lgx.Context(0)
    try:
        rng, hkv, d, pages, P = np.random.default_rng(3), 256, 64, 64, 2
        n = 131072 // 16
        cache = ref.Cache(pages, hkv, d, rng)
        cache.v[:] = np.abs(cache.v.astype(np.int16)).clip(1, 127)
        cache.vs[:] = np.float32(0.01)
        cache.ks[:] = np.float32(2.0 ** -6)
        cache.k[:] = rng.integers(-20, 21, cache.k.shape)
        # page 0 is the sink's: its token 0 scores ln(131072) more than the others, q = 1
        cache.k[0, :, 0] = int(round(np.log(131072.0) / (2.0 ** -6 * 8)))
        table = np.concatenate([[0], 1 + np.arange(n - 1) % (pages - 1)]).astype(np.int32)[None]
        q = np.ones((1, P, hkv, d), np.float32)
        L = n * 16 - P
        got = host(c.gqa_prefill_attn_i8(c.to_device(q[0]), upload(c, cache), i32(c, table), i32(c, [L]), P, n * 16))
        full = np.bincount(table[0, :-1], minlength=pages).astype(np.float64)
        errs = []
        for j in range(P):
            count = np.repeat(full[:, None], 16, 1)
            count[table[0, -1], :16 - P + j + 1] += 1
            for g in range(hkv):
                s = cache.k[:, g].astype(np.float64).sum(-1) * 2.0 ** -6 / 8
                w = count * np.exp(s - s.max())
                v = cache.v[:, g].astype(np.float64) * float(np.float32(0.01))
                want = np.einsum("pt,pdt->d", w, v) / w.sum()
                errs.append(((got[j, g] - want) / want).mean())
        assert 0.3 < w[0, 0] / w.sum() < 0.7
        assert np.abs(np.mean(errs)) <= 5 * 3.1e-7 and np.abs(errs).max() <= 5 * 4.9e-6, (np.mean(errs), np.abs(errs).max())
    finally:
        c.close()


@pytest.mark.parametrize("P", [1, 2])
def test_equal_weights_over_a_long_context(monkeypatch, P):
    """q = 0: the mean of 65536 values of one sign, by one workgroup.  The sum of the
    weights is exact.  A dimension's sum is rounded once for each of up to 1024 tiles, to
    either side, by at most 2^-24 of what it has reached: sqrt(1024 / 3 / 3) 2^-24 = 6.4e-7
    at the end; within the tiles roundings are 1024 times smaller; the weight itself, the V
    scale, is held to 2^-23.  Six deviations (of 64 dimensions the largest) and that: 4.0e-6.
    (Second parts added one by one to sums of 2^15 of the first are lost: 5e-5 to 1e-4.)"""
    monkeypatch.setenv("LGX_A8_COLS", "16" if P == 1 else "128")
    c = lgx.Context(0)
    try:
        rng, B, d, n = np.random.default_rng(P), 256, 64, 4096
        cache = ref.Cache(n, 1, d, rng)
        cache.v[:] = np.abs(cache.v.astype(np.int16)).clip(1, 127)
        cache.vs[:] = np.float32(0.01)
        table = np.broadcast_to(rng.permutation(n).astype(np.int32), (B, n))
        kv, tab, L = upload(c, cache), i32(c, np.ascontiguousarray(table)), n * 16 - (P > 1) * P
        q = c.torch.zeros((B * P, 1, d), device=c.dev)
        before = c.launch_count
        if P == 1:
            got = host(c.gqa_decode_attn_i8(q, kv, tab, i32(c, [L] * B), n * 16))
        else:
            got = host(c.gqa_prefill_attn_i8(q, kv, tab, i32(c, [L] * B), P, n * 16))
        assert c.launch_count - before == 1          # nothing is split
        _, v = cache.rows(table[0], n * 16)
        for j in range(P):
            want = v[:L + j + (P > 1), 0].mean(0)
            err = np.abs(got.reshape(B, P, d)[:, j] - want) / want
            assert err.max() <= 4.0e-6, (j, err.max())
    finally:
        c.close()


@pytest.mark.parametrize("P", [1, 70])
@pytest.mark.parametrize("small", [1e-20, 1e-25, 1e-28])
def test_tiny_queries_under_large_k_scales(ctx, P, small):
    """Queries down to 2^-93 with keys as large: the scores are ordinary numbers."""
    rng, hq, hkv, d, maxp = np.random.default_rng(P), 4, 2, 64, 10
    cache = ref.Cache(maxp, hkv, d, rng)
    cache.ks = (cache.ks * np.float32(1 / small)).astype(np.float32)
    q = (rng.standard_normal((1, P, hq, d)) * small).astype(np.float32)
    table, lens = np.arange(maxp, dtype=np.int32)[None], [maxp * 16 - P]
    want, bound = attend(cache, q, table, lens, P > 1)
    if P == 1:
        got = ctx.gqa_decode_attn_i8(ctx.to_device(q[:, 0]), upload(ctx, cache), i32(ctx, table), i32(ctx, lens), maxp * 16)
    else:
        got = ctx.gqa_prefill_attn_i8(ctx.to_device(q[0]), upload(ctx, cache), i32(ctx, table), i32(ctx, lens), P, maxp * 16)
    check(host(got).reshape(want.shape), want, bound, tight=1e-3)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("B,P", [(1, 1), (3, 1), (2, 5), (40, 1)])
def test_values_near_the_largest_numbers(ctx, B, P, d):
    """A result lies within its values, also where those are 1e38 and their sum over a
    split's tokens is not a number any more, or 1e-36."""
    rng, hq, hkv, maxp = np.random.default_rng(B + P + d), 4, 2, 320
    cache, table = ref.Cache(maxp, hkv, d, rng), rng.integers(0, maxp, (B, maxp)).astype(np.int32)
    cache.ks[:] = np.float32(0.002)
    cache.vs[:, 0], cache.vs[:, 1] = np.float32(1e38 / 127), np.float32(2e-38)
    lens = rng.integers(3000, maxp * 16 - P, B)
    q = rng.standard_normal((B, P, hq, d)).astype(np.float32)
    want, bound = attend(cache, q, table, lens, P > 1)
    if P == 1:
        got = ctx.gqa_decode_attn_i8(ctx.to_device(q[:, 0]), upload(ctx, cache), i32(ctx, table), i32(ctx, lens), maxp * 16)
    else:
        got = ctx.gqa_prefill_attn_i8(ctx.to_device(q.reshape(B * P, hq, d)), upload(ctx, cache), i32(ctx, table), i32(ctx, lens), P,
                                      maxp * 16)
    check(host(got).reshape(want.shape), want, bound + 2.0 ** -149, tight=1e-3)


# ---- recorded steps -------------------------------------------------------

def test_a_recorded_step_outlives_a_larger_call():
    """A step recorded with a small workspace, then calls on the same context that need a
    larger one, and allocations that could take freed memory: the replays still give the
    eager step's results."""
    c = lgx.Context(0)
    try:
        t, rng = c.torch, np.random.default_rng(21)
        hq, hkv, d, B, maxp = 8, 2, 64, 2, 256
        cache, table = ref.Cache(B * maxp, hkv, d, rng), rng.permutation(B * maxp).astype(np.int32).reshape(B, maxp)
        kv, tab, lens = upload(c, cache), i32(c, table), i32(c, [4000, 900])
        q = c.to_device(rng.standard_normal((B, hq, d)).astype(np.float32))
        out = t.empty_like(q)
        want = c.gqa_decode_attn_i8(q, kv, tab, lens, maxp * 16)
        side, graph = t.cuda.Stream(), t.cuda.CUDAGraph()
        t.cuda.synchronize()
        with t.cuda.graph(graph, stream=side):
            c.gqa_decode_attn_i8(q, kv, tab, lens, maxp * 16, out=out)
        # 27 MB of partial results
        chunks = 400
        big = c.gqa_decode_attn(t.zeros((64, 8, 64), device=c.dev),
                                *(t.zeros((1, 2, 16, 64), dtype=t.float16, device=c.dev) for _ in range(2)),
                                t.zeros((64, chunks * 8), dtype=t.int32, device=c.dev), t.ones(64, dtype=t.int32, device=c.dev),
                                chunks * 128)
        t.cuda.synchronize()
        taken = [t.full((1 << 18,), 7.0, device=c.dev) for _ in range(8)]
        for i in range(4):
            out.zero_()
            graph.replay()
            t.cuda.synchronize()
            assert t.equal(out, want), i
            assert t.equal(c.gqa_decode_attn_i8(q, kv, tab, lens, maxp * 16), want), i
        assert all(bool((x == 7.0).all()) for x in taken) and not bool(big.any())
    finally:
        c.close()
