"""The 8-bit KV cache on the device against tests/kv8_ref.py (numpy float64): the
append's scales and quants to the bit, the attention within the bound derived there."""
import numpy as np
import pytest

import kv8_ref as ref
import logicaffeine_amd as lgx

pytestmark = pytest.mark.gpu


def host(t):
    return t.cpu().numpy()


def upload(ctx, cache):
    return lgx.KvCacheI8(*(ctx.to_device(x) for x in (cache.k, cache.v, cache.ks, cache.vs)))


def same_cache(kv, cache):
    for name, got, want in (("k", kv.k, cache.k), ("v", kv.v, cache.v)):
        assert np.array_equal(host(got), want), name
    for name, got, want in (("k_scale", kv.k_scale, cache.ks), ("v_scale", kv.v_scale, cache.vs)):
        assert np.array_equal(host(got), want, equal_nan=True), name


def i32(ctx, x):
    return ctx.to_device(np.asarray(x, np.int32))


def rope_of(ctx, cos, sin, interleaved=False):
    return lgx.Rope(ctx.to_device(cos), ctx.to_device(sin), interleaved)


def table_of(rng, B, maxp):
    return rng.permutation(B * maxp).astype(np.int32).reshape(B, maxp)


# ---- append ---------------------------------------------------------------

@pytest.mark.parametrize("hq,hkv,d,rot,inter,P,lens,new", [
    (14, 2, 64, 64, False, 1, [0, 1, 15, 16, 17, 40], None),
    (28, 4, 128, 128, False, 1, [0, 31, 100], None),
    (12, 2, 128, 64, True, 1, [7, 16], None),
    (4, 4, 64, 16, False, 5, [0, 13, 14, 33], [5, 0, 1, 4]),
    (12, 2, 128, 128, True, 33, [0, 1, 16, 30], [33, 16, 15, 2]),
    (2, 1, 64, 6, False, 40, [3, 0], None),          # pairs across the threads' elements
    (16, 1, 128, 0, False, 18, [15], None),          # no rotation at all
    (3, 3, 128, 2, True, 2, [14, 15], None),
])
def test_append_is_the_definition(ctx, hq, hkv, d, rot, inter, P, lens, new):
    """Every length around a page's edges, padded rows, part rotations; values that
    make old blocks grow; untouched slots and pages keep their bytes."""
    rng = np.random.default_rng(hq * d + P + rot)
    B, maxp = len(lens), (max(lens) + P) // 16 + 2
    cache = ref.Cache(B * maxp, hkv, d, rng)
    table = table_of(rng, B, maxp)
    cos, sin = ref.tables(max(lens) + P + 1, rot)
    x = (rng.standard_normal((B, P, (hq + 2 * hkv) * d)) * 10.0 ** rng.uniform(-2, 2, (B, P, 1))).astype(np.float32)
    bias = rng.standard_normal((hq + 2 * hkv) * d).astype(np.float32)
    kv = upload(ctx, cache)
    q = ctx.torch.full((B * P, hq, d), 7.0, device=ctx.dev)
    ctx.rope_kv_append_i8(ctx.to_device(x.reshape(B * P, -1)), ctx.to_device(bias), rope_of(ctx, cos, sin, inter),
                          i32(ctx, lens), i32(ctx, table), kv, P, n_new=None if new is None else i32(ctx, new), q_out=q)
    want = cache.append(x, bias, cos, sin, inter, lens, new, table, hq)
    same_cache(kv, cache)
    pad = np.arange(P) >= (np.full(B, P) if new is None else np.asarray(new))[:, None]
    want[pad] = 7.0                                  # padding rows of q are left alone
    assert np.array_equal(host(q).reshape(B, P, hq, d), want)


@pytest.mark.parametrize("hq,hkv,d,rot,inter,P", [(4, 2, 128, 64, False, 21), (3, 1, 64, 64, True, 5), (2, 2, 128, 128, False, 1)])
def test_append_from_rows_that_are_only_4_byte_aligned(ctx, hq, hkv, d, rot, inter, P):
    """The same quants whether rows and tables come in wide loads or number by number."""
    t, rng = ctx.torch, np.random.default_rng(d + P)
    lens, width = [7, 16], (hq + 2 * hkv) * d
    cache, table = ref.Cache(8, hkv, d, rng), table_of(rng, 2, 4)
    cos, sin = ref.tables(64, rot)
    x, bias = rng.standard_normal((2, P, width)).astype(np.float32), rng.standard_normal(width).astype(np.float32)
    kv = upload(ctx, cache)

    def odd(a):
        buf = t.zeros(a.size + 1, device=ctx.dev)[1:].view(a.shape)
        buf.copy_(ctx.to_device(a))
        assert buf.data_ptr() % 16 == 4
        return buf

    rope = lgx.Rope(odd(cos), odd(sin), inter)
    q = ctx.rope_kv_append_i8(odd(x.reshape(2 * P, width)), odd(bias), rope, i32(ctx, lens), i32(ctx, table), kv, P)
    want = cache.append(x, bias, cos, sin, inter, lens, None, table, hq)
    assert np.array_equal(host(q).reshape(want.shape), want)
    same_cache(kv, cache)


@pytest.mark.parametrize("P,new", [(1, [0, 1, 1, 0, 5, -2]), (3, [0, 0, -1, 0, 0, 0]), (20, [0, 20, 1, 16, 99, -7])])
def test_append_of_few_or_no_rows(ctx, P, new):
    """Row counts of zero, negative ones (zero) and too many (P)."""
    rng = np.random.default_rng(P)
    hq, hkv, d, B = 3, 1, 64, 6
    lens = [0, 15, 16, 31, 3, 8]
    cache, table = ref.Cache(B * 4, hkv, d, rng), table_of(rng, B, 4)
    cos, sin = ref.tables(64, d)
    x = rng.standard_normal((B, P, (hq + 2 * hkv) * d)).astype(np.float32)
    kv = upload(ctx, cache)
    q = ctx.torch.full((B * P, hq, d), 7.0, device=ctx.dev)
    ctx.rope_kv_append_i8(ctx.to_device(x.reshape(B * P, -1)), None, rope_of(ctx, cos, sin), i32(ctx, lens), i32(ctx, table), kv, P,
                          n_new=i32(ctx, new), q_out=q)
    want = cache.append(x, None, cos, sin, False, lens, new, table, hq)
    want[np.arange(P) >= np.clip(new, 0, P)[:, None]] = 7.0
    assert np.array_equal(host(q).reshape(want.shape), want)
    same_cache(kv, cache)


def test_append_token_by_token_keeps_old_values_within_a_step(ctx):
    """Tokens that keep growing, one call each: the device follows the definition, and
    no value is ever off by more than one step of its block's scale, nor is the scale
    more than twice what the block needs."""
    rng = np.random.default_rng(3)
    hq, hkv, d, B, n = 2, 2, 64, 3, 37
    maxp = 3
    cache, table = ref.Cache(B * maxp, hkv, d), table_of(rng, 3, 3)
    kv = lgx.KvCacheI8.empty(ctx, B * maxp, hkv, d)
    rope = rope_of(ctx, *ref.tables(64, 2))
    lens = np.array([0, 0, 0], np.int32)
    x = (rng.standard_normal((n, B, 1, (hq + 2 * hkv) * d)) * 1.4 ** np.arange(n)[:, None, None, None]).astype(np.float32)
    x[:, 2] *= 1e-30                                 # one sequence of tiny values
    for t in range(n):
        ctx.rope_kv_append_i8(ctx.to_device(x[t].reshape(B, -1)), None, rope, ctx.to_device(lens), i32(ctx, table), kv)
        cache.append(x[t], None, *ref.tables(64, 2), False, lens, None, table, hq)
        lens += 1
    same_cache(kv, cache)
    for b in range(B):
        _, v = cache.rows(table[b], n)
        true = x[:, b, 0].reshape(n, -1, d)[:, hq + hkv:].astype(np.float64)
        for p in range(0, n, 16):
            step = cache.vs[table[b, p // 16]].astype(np.float64)[:, None]
            assert (np.abs(v[p:p + 16] - true[p:p + 16]) <= step * (1 + 1e-6)).all()
            assert (step[:, 0] <= 2.0001 * np.abs(true[p:p + 16]).max((0, 2)) / 127).all()


def test_append_special_values(ctx):
    """Zero blocks, subnormal ones, the largest numbers, infinities and NaN: what
    becomes of the block's scale, and that a fresh start clears a NaN block."""
    hq, hkv, d, P = 1, 1, 64, 3
    cases = [0.0, 1e-40, 1e-28, 3e38, np.inf, np.nan, -np.inf]
    B, rng = len(cases), np.random.default_rng(5)
    table = np.arange(B, dtype=np.int32).reshape(B, 1)
    x = rng.uniform(-1, 1, (B, P, 3 * d)).astype(np.float32)
    for b, c in enumerate(cases):
        if np.isfinite(c):
            x[b] *= np.float32(c)
        else:
            x[b, 1, 100:170:7] = c
    cos, sin = ref.tables(64, 32)
    rope = rope_of(ctx, cos, sin)
    kv, cache = lgx.KvCacheI8.empty(ctx, B, hkv, d), ref.Cache(B, hkv, d)
    with np.errstate(all="ignore"):
        for lens, finite in (([0] * B, False), ([3] * B, False), ([0] * B, True)):
            x = np.where(np.isfinite(x), x, 1).astype(np.float32) if finite else x
            q = ctx.rope_kv_append_i8(ctx.to_device(x.reshape(B * P, -1)), None, rope, i32(ctx, lens), i32(ctx, table), kv, P)
            want = cache.append(x, None, cos, sin, False, lens, None, table, hq)
            assert np.array_equal(host(q).reshape(want.shape), want, equal_nan=True)
            same_cache(kv, cache)
            assert np.isnan(host(kv.k_scale)).ravel().tolist() == [False] * 4 + [not finite] * 3


def test_append_stays_inside_its_pages(ctx):
    """Lengths and page ids out of range, positions past the tables: nothing outside
    the sequence's own pages is written."""
    rng = np.random.default_rng(11)
    hq, hkv, d, P, maxp = 2, 1, 64, 20, 2
    lens = [-5, 20, 32, 2**31 - 1, 4]
    table = np.array([[0, 1], [2, 3], [4, 5], [6, 7], [-1, 99]], np.int32)
    B = len(lens)
    cache = ref.Cache(10, hkv, d, rng)
    kv = upload(ctx, cache)
    cos, sin = ref.tables(24, d)
    x = rng.standard_normal((B, P, (hq + 2 * hkv) * d)).astype(np.float32)
    q = ctx.rope_kv_append_i8(ctx.to_device(x.reshape(B * P, -1)), None, rope_of(ctx, cos, sin), i32(ctx, lens),
                              i32(ctx, table), kv, P, n_new=i32(ctx, [20, 99, 20, 20, 20]))
    want = cache.append(x, None, cos, sin, False, lens, [20, 20, 20, 20, 20], table, hq)
    assert np.array_equal(host(q).reshape(want.shape), want)
    same_cache(kv, cache)


@pytest.mark.parametrize("d", [64, 128])
def test_read_back(ctx, d):
    """Values from any token on, zeros past the sequence's pages."""
    rng = np.random.default_rng(d)
    hkv, B, maxp, n = 3, 4, 3, 21
    cache, table = ref.Cache(B * maxp, hkv, d, rng), table_of(rng, B, maxp)
    start = [0, 5, 30, 48]
    k, v = ctx.kv_read_i8(upload(ctx, cache), i32(ctx, table), i32(ctx, start), n)
    for b, s in enumerate(start):
        for got, full in zip((host(k)[b], host(v)[b]), cache.rows(table[b], maxp * 16)):
            want = np.zeros((n, hkv, d), np.float32)
            part = full[s:s + n]
            want[:len(part)] = part.astype(np.float32)
            assert np.array_equal(got, want)


# ---- attention ------------------------------------------------------------

def decode(ctx, cache, q, table, lens, max_len, kv=None, **opts):
    if "slopes" in opts:
        opts["slopes"] = ctx.to_device(opts["slopes"])
    return host(ctx.gqa_decode_attn_i8(ctx.to_device(q), kv or upload(ctx, cache), i32(ctx, table), i32(ctx, lens), max_len,
                                       lgx.AttnOpts(**opts) if opts else None))


def check(got, want, bound):
    assert np.isfinite(want).all()
    worst = np.abs(got - want) - bound
    assert (worst <= 0).all(), (worst.max(), np.unravel_index(worst.argmax(), worst.shape))


LENS = [1, 16, 17, 63, 64, 65, 255, 257, 700, 0]
OPTIONS = [dict(), dict(softcap=2.0), dict(window=1), dict(window=100), dict(scale=0.3, softcap=30.0, window=65),
           dict(slopes=True), dict(slopes=True, softcap=5.0, window=300)]


def options(o, hq):
    o = dict(o)
    if o.get("slopes"):
        o["slopes"] = (2.0 ** (-8.0 * np.arange(1, hq + 1) / hq)).astype(np.float32)
    return o


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (2, 1), (6, 2), (14, 2), (8, 1), (11, 1), (16, 1), (28, 4), (5, 5)])
def test_decode_head_layouts(ctx, hq, hkv, d):
    rng = np.random.default_rng(hq * d + hkv)
    B, maxp = len(LENS), -(-max(LENS) // 16)
    cache, table = ref.Cache(B * maxp, hkv, d, rng), table_of(rng, B, maxp)
    q = rng.standard_normal((B, hq, d)).astype(np.float32)
    got = decode(ctx, cache, q, table, LENS, max(LENS))
    want, bound = ref.attend(cache, q[:, None], table, LENS, max(LENS), prefill=False)
    check(got, want[:, 0], bound[:, 0])
    assert np.all(got[-1] == 0.0)                    # an empty sequence


@pytest.mark.parametrize("opts", OPTIONS, ids=str)
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (12, 2, 128)])
def test_decode_options(ctx, hq, hkv, d, opts):
    rng = np.random.default_rng(17)
    B, maxp = len(LENS), -(-max(LENS) // 16)
    cache, table = ref.Cache(B * maxp, hkv, d, rng), table_of(rng, B, maxp)
    q = rng.standard_normal((B, hq, d)).astype(np.float32)
    o = options(opts, hq)
    got = decode(ctx, cache, q, table, LENS, max(LENS), **o)
    want, bound = ref.attend(cache, q[:, None], table, LENS, max(LENS), prefill=False, **o)
    check(got, want[:, 0], bound[:, 0])


@pytest.mark.parametrize("B,L,window", [(1, 5000, 0), (3, 20000, 0), (2, 20000, 3000), (1, 70000, 0)])
def test_decode_long_contexts(ctx, B, L, window):
    """Several workgroups per sequence, their results joined; next to a short one."""
    rng = np.random.default_rng(L)
    hq, hkv, d = 4, 1, 64
    maxp = -(-L // 16)
    lens = ([L, 100, L // 3] * B)[:B]
    cache, table = ref.Cache(B * maxp, hkv, d, rng), table_of(rng, B, maxp)
    q = rng.standard_normal((B, hq, d)).astype(np.float32)
    got = decode(ctx, cache, q, table, lens, L, **(dict(window=window) if window else {}))
    want, bound = ref.attend(cache, q[:, None], table, lens, L, prefill=False, window=window)
    check(got, want[:, 0], bound[:, 0])


@pytest.mark.parametrize("B,window", [(70, 0), (255, 0), (255, 90), (300, 0)])
def test_decode_many_ragged_sequences(ctx, B, window):
    """Batches whose tiles are split by all their lengths (up to 256 sequences and KV
    heads together) and one that is not, empty sequences among them."""
    rng = np.random.default_rng(B + window)
    hq, hkv, d, top = 2, 1, 64, 900
    lens = rng.integers(0, top + 1, B)
    lens[::7] = rng.integers(0, 3, len(lens[::7]))
    lens[B // 2] = top
    maxp = -(-top // 16)
    cache, table = ref.Cache(B * maxp, hkv, d, rng), table_of(rng, B, maxp)
    q = rng.standard_normal((B, hq, d)).astype(np.float32)
    got = decode(ctx, cache, q, table, lens, top, **(dict(window=window) if window else {}))
    want, bound = ref.attend(cache, q[:, None], table, lens, top, prefill=False, window=window)
    check(got, want[:, 0], bound[:, 0])
    assert np.all(got[lens == 0] == 0.0)


def test_decode_when_every_length_is_zero(ctx):
    cache = ref.Cache(200, 2, 128)
    cache.ks[:] = cache.vs[:] = np.nan
    got = decode(ctx, cache, np.ones((2, 4, 128), np.float32), np.arange(200).reshape(2, 100), [0, 0], 1600)
    assert np.all(got == 0.0)


PREFILL = [(14, 2, 64, [0, 37, 500], 40, None), (28, 4, 128, [0, 200], 72, None), (12, 2, 128, [500, 0, 255], 9, [9, 4, 0]),
           (8, 8, 64, [3], 257, None), (8, 1, 128, [1000, 64], 20, [1, 20]), (16, 1, 64, [5, 0], 1, None),
           (7, 1, 128, [2000], 2, None), (4, 2, 64, [0, 1, 63, 64], 130, [130, 129, 65, 64])]


@pytest.mark.parametrize("hq,hkv,d,lens,P,new", PREFILL)
@pytest.mark.parametrize("opts", [OPTIONS[0], OPTIONS[4], OPTIONS[6], dict(window=1)], ids=str)
def test_prefill(ctx, hq, hkv, d, lens, P, new, opts):
    rng = np.random.default_rng(hq * d + P)
    B, top = len(lens), max(lens) + P
    maxp = -(-top // 16)
    cache, table = ref.Cache(B * maxp, hkv, d, rng), table_of(rng, B, maxp)
    q = rng.standard_normal((B, P, hq, d)).astype(np.float32)
    o = options(opts, hq)
    want, bound = ref.attend(cache, q, table, lens, top, n_new=new, **o)
    if "slopes" in o:
        o["slopes"] = ctx.to_device(o["slopes"])
    out = ctx.torch.full((B * P, hq, d), 7.0, device=ctx.dev)
    ctx.gqa_prefill_attn_i8(ctx.to_device(q.reshape(B * P, hq, d)), upload(ctx, cache), i32(ctx, table), i32(ctx, lens), P, top,
                            n_new=None if new is None else i32(ctx, new), opts=lgx.AttnOpts(**o) if o else None, out=out)
    got = host(out).reshape(q.shape)
    pad = np.arange(P) >= (np.full(B, P) if new is None else np.asarray(new))[:, None]
    assert np.all(got[pad] == 7.0)
    want[pad] = 7.0
    check(got, want, bound)


@pytest.mark.parametrize("cols", [16, 32, 128])
@pytest.mark.parametrize("hq,hkv,d,lens,P,new", [PREFILL[i] for i in (0, 2, 4, 7)] + [(28, 4, 128, [700, 3], 33, [33, 20])])
@pytest.mark.parametrize("opts", [OPTIONS[0], OPTIONS[6]], ids=str)
def test_prefill_by_every_number_of_columns(monkeypatch, hq, hkv, d, lens, P, new, opts, cols):
    """16, 32 and 128 (row, head) pairs per workgroup, few and many workgroups."""
    monkeypatch.setenv("LGX_A8_COLS", str(cols))
    monkeypatch.setenv("LGX_A8_WGS", "1" if cols == 32 else "5")
    c = lgx.Context(0)
    try:
        before = c.launch_count
        test_prefill(c, hq, hkv, d, lens, P, new, opts)
        assert c.launch_count - before in (1, 2)
    finally:
        c.close()


def test_a_cache_beyond_4_gib(ctx):
    """Pages whose bytes lie past 2^32: append, read-back, decode and prefill attention
    give what they give near the start of a small cache."""
    t, rng = ctx.torch, np.random.default_rng(9)
    hq, hkv, d, B, P, maxp, big = 16, 8, 128, 2, 20, 40, 290000
    assert (big - 100) * hkv * 16 * d > 2**32
    small = ref.Cache(B * maxp, hkv, d, rng)
    table = table_of(rng, B, maxp)
    far = table + (big - B * maxp)
    kv = lgx.KvCacheI8.empty(ctx, big, hkv, d)
    near = upload(ctx, small)
    for a, b in ((kv.k, near.k), (kv.v, near.v), (kv.k_scale, near.k_scale), (kv.v_scale, near.v_scale)):
        a[big - B * maxp:] = b
    rope = rope_of(ctx, *ref.tables(700, d))
    x = ctx.to_device(rng.standard_normal((B * P, (hq + 2 * hkv) * d)).astype(np.float32))
    lens, got = i32(ctx, [601, 300]), []
    for cache, tab in ((near, i32(ctx, table)), (kv, i32(ctx, far))):
        q = ctx.rope_kv_append_i8(x, None, rope, lens, tab, cache, P)
        out = ctx.gqa_prefill_attn_i8(q, cache, tab, lens, P, maxp * 16)
        one = ctx.gqa_decode_attn_i8(q[:B].contiguous(), cache, tab, lens, maxp * 16)
        got.append((q, out, one) + ctx.kv_read_i8(cache, tab, lens, P))
    for a, b in zip(*got):
        assert t.equal(a, b)
    assert bool((kv.k[:big - B * maxp] == 0).all()) and bool((kv.v_scale[:big - B * maxp] == 0).all())


def test_two_contexts_on_two_streams(ctx):
    """Split attention of two contexts at once: each has its own workspace."""
    t, rng = ctx.torch, np.random.default_rng(12)
    hq, hkv, d, B, L = 8, 2, 128, 2, 9000
    maxp = -(-L // 16)
    cache, table = ref.Cache(B * maxp, hkv, d, rng), table_of(rng, B, maxp)
    kv, tab, lens = upload(ctx, cache), i32(ctx, table), i32(ctx, [L, L - 77])
    qs = [ctx.to_device(rng.standard_normal((B, hq, d)).astype(np.float32)) for _ in range(2)]
    want = [ctx.gqa_decode_attn_i8(q, kv, tab, lens, L) for q in qs]
    other = lgx.Context(0)
    try:
        t.cuda.synchronize()
        streams, outs = [t.cuda.Stream(), t.cuda.Stream()], [[], []]
        for _ in range(20):
            for i, c in enumerate((ctx, other)):
                with t.cuda.stream(streams[i]):
                    outs[i].append(c.gqa_decode_attn_i8(qs[i], kv, tab, lens, L))
        t.cuda.synchronize()
        for i in range(2):
            assert all(t.equal(o, want[i]) for o in outs[i])
    finally:
        other.close()


def test_lengths_are_clamped(ctx):
    rng = np.random.default_rng(2)
    hq, hkv, d, maxp = 6, 2, 64, 10
    cache, table = ref.Cache(3 * maxp, hkv, d, rng), table_of(rng, 3, maxp)
    table[1, 3] = -7                                 # page ids too
    table[0, 1] = 10000
    q = rng.standard_normal((3, hq, d)).astype(np.float32)
    lens = [2**31 - 1, 100, -3]
    got = decode(ctx, cache, q, table, lens, 130)
    want, bound = ref.attend(cache, q[:, None], table, [130, 100, 0], 130, prefill=False)
    check(got, want[:, 0], bound[:, 0])
    q = rng.standard_normal((3, 4, hq, d)).astype(np.float32)
    got = host(ctx.gqa_prefill_attn_i8(ctx.to_device(q.reshape(12, hq, d)), upload(ctx, cache), i32(ctx, table),
                                       i32(ctx, lens), 4, 130)).reshape(q.shape)
    want, bound = ref.attend(cache, q, table, lens, 130)
    check(got, want, bound)


def test_one_token_gives_its_value_and_constant_v_itself(ctx):
    """Closed forms: the weight of a single token is 1; equal V rows come back."""
    rng = np.random.default_rng(8)
    hq, hkv, d, maxp = 8, 2, 128, 8
    cache, table = ref.Cache(2 * maxp, hkv, d, rng), table_of(rng, 2, maxp)
    q = rng.standard_normal((2, hq, d)).astype(np.float32)
    got = decode(ctx, cache, q, table, [1, 1], 128)
    for b in range(2):
        _, v = cache.rows(table[b], 1)
        assert np.allclose(got[b], np.repeat(v[0], 4, axis=0), rtol=2.0 ** -20, atol=0)
    cache.v[:] = rng.integers(-127, 128, (1, hkv, d, 1), dtype=np.int8)
    cache.vs[:] = 0.02
    got = decode(ctx, cache, q, table, [128, 77], 128)
    want = np.repeat(cache.v[0, :, :, 0] * np.float64(np.float32(0.02)), 4, axis=0)
    assert np.allclose(got, want[None], rtol=2.0 ** -18, atol=0)


@pytest.mark.parametrize("d", [64, 128])
def test_what_is_not_seen_does_not_matter(ctx, d):
    """NaN and infinite scales on pages past a sequence's length, out of its window, or
    seen by later rows only; the same page seen gives NaN."""
    rng = np.random.default_rng(d)
    hq, hkv, P, top = 4, 2, 20, 200
    maxp = 16
    cache, table = ref.Cache(maxp, hkv, d, rng), np.arange(maxp, dtype=np.int32)[None]
    q = rng.standard_normal((1, P, hq, d)).astype(np.float32)
    lens = [150]                                     # rows at 150 .. 169
    want, bound = ref.attend(cache, q, table, lens, top)
    for scales in (cache.ks, cache.vs):
        for value in (np.nan, np.inf):
            keep = scales.copy()
            scales[11:] = value                      # tokens from 176 on
            scales[10, 1] = value                    # KV head 1, tokens 160 .. 175: rows 10 .. 19
            got = host(ctx.gqa_prefill_attn_i8(ctx.to_device(q.reshape(P, hq, d)), upload(ctx, cache), i32(ctx, table),
                                               i32(ctx, lens), P, top)).reshape(q.shape)
            check(got[:, :10], want[:, :10], bound[:, :10])
            check(got[:, :, :2], want[:, :, :2], bound[:, :, :2])
            assert np.isnan(got[:, 10:, 2:]).all()
            scales[:] = keep
            scales[:2] = value                       # the first 32 tokens, out of the window
            w2, b2 = ref.attend(cache_without(cache, keep, scales), q, table, lens, top, window=100)
            got = host(ctx.gqa_prefill_attn_i8(ctx.to_device(q.reshape(P, hq, d)), upload(ctx, cache), i32(ctx, table),
                                               i32(ctx, lens), P, top, opts=lgx.AttnOpts(window=100))).reshape(q.shape)
            check(got, w2, b2)
            scales[:] = keep


def cache_without(cache, keep, scales):
    """The cache with the scales it had before."""
    c = ref.Cache(1, cache.hkv, cache.d)
    c.k, c.v = cache.k, cache.v
    c.ks, c.vs = (keep if x is scales else x for x in (cache.ks, cache.vs))
    return c


def test_queries_and_scales_of_extreme_size(ctx):
    """Rows of zeros, tiny and huge queries (the weights become one-hot), V scales that
    span 60 orders between pages; an infinite or NaN query gives NaN for its head alone."""
    rng = np.random.default_rng(1)
    hq, hkv, d, maxp, L = 8, 2, 64, 12, 190
    cache, table = ref.Cache(maxp, hkv, d, rng), np.arange(maxp, dtype=np.int32)[None]
    q = rng.standard_normal((1, hq, d)).astype(np.float32)
    q[0, 0] = 0.0
    q[0, 1] *= np.float32(1e-35)
    q[0, 2] *= np.float32(1e-42)
    q[0, 3] *= np.float32(1e4)
    cache.vs[::3] *= np.float32(1e-30)
    cache.vs[1::3] *= np.float32(1e30)
    got = decode(ctx, cache, q, table, [L], L)
    want, bound = ref.attend(cache, q[:, None], table, [L], L, prefill=False)
    check(got, want[:, 0], bound[:, 0])
    q[0, 5, 3], q[0, 6, 7] = np.inf, np.nan
    bad = decode(ctx, cache, q, table, [L], L)
    assert np.isnan(bad[0, 5:7]).all()
    assert np.array_equal(np.delete(bad[0], [5, 6], 0), np.delete(got[0], [5, 6], 0))


# ---- together -------------------------------------------------------------

@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (6, 1, 128)])
def test_prompt_then_tokens(ctx, hq, hkv, d):
    """As a decode loop runs them: a padded prompt appended and attended to, then
    tokens one by one, everything on the device; against the definition."""
    rng = np.random.default_rng(d)
    B, P, steps, maxp = 3, 37, 20, 5
    rope_np = ref.tables(128, d)
    cache, table = ref.Cache(B * maxp, hkv, d), table_of(rng, B, maxp)
    kv, rope, tab = lgx.KvCacheI8.empty(ctx, B * maxp, hkv, d), rope_of(ctx, *rope_np), i32(ctx, table)
    width = (hq + 2 * hkv) * d
    lens, new = np.zeros(B, np.int32), np.array([37, 5, 16], np.int32)
    dl, dn = ctx.to_device(lens), ctx.to_device(new)
    x = rng.standard_normal((B, P, width)).astype(np.float32)
    q = ctx.rope_kv_append_i8(ctx.to_device(x.reshape(B * P, width)), None, rope, dl, tab, kv, P, n_new=dn)
    got = host(ctx.gqa_prefill_attn_i8(q, kv, tab, dl, P, maxp * 16, n_new=dn)).reshape(B, P, hq, d)
    qn = cache.append(x, None, *rope_np, False, lens, new, table, hq)
    want, bound = ref.attend(cache, qn, table, lens, maxp * 16, n_new=new)
    for b in range(B):
        check(got[b, :new[b]], want[b, :new[b]], bound[b, :new[b]])
    lens = lens + new
    dl = dl + dn
    for _ in range(steps):
        x = rng.standard_normal((B, 1, width)).astype(np.float32)
        q = ctx.rope_kv_append_i8(ctx.to_device(x[:, 0]), None, rope, dl, tab, kv)
        dl = dl + 1
        out = ctx.gqa_decode_attn_i8(q, kv, tab, dl, maxp * 16)
        qn = cache.append(x, None, *rope_np, False, lens, None, table, hq)
        lens = lens + 1
        want, bound = ref.attend(cache, qn, table, lens, maxp * 16, prefill=False)
        check(host(out), want[:, 0], bound[:, 0])
    same_cache(kv, cache)


def test_a_captured_step_replays(ctx):
    """append + decode attention recorded once, replayed with new rows and lengths in
    the same buffers, eager work between the replays."""
    t = ctx.torch
    rng = np.random.default_rng(4)
    hq, hkv, d, B, L0, maxp = 8, 2, 64, 2, 3000, 200
    cache, table = ref.Cache(B * maxp, hkv, d, rng), table_of(rng, B, maxp)
    width = (hq + 2 * hkv) * d
    rope = rope_of(ctx, *ref.tables(3200, d))
    tab, kv, kv2 = i32(ctx, table), upload(ctx, cache), upload(ctx, cache)
    x, lens = t.zeros((B, width), device=ctx.dev), i32(ctx, [L0, 17])
    q, out = t.empty((B, hq, d), device=ctx.dev), t.empty((B, hq, d), device=ctx.dev)

    def step(kv, x, lens, q, out):
        ctx.rope_kv_append_i8(x, None, rope, lens, tab, kv, q_out=q)
        lens += 1
        ctx.gqa_decode_attn_i8(q, kv, tab, lens, maxp * 16, out=out)

    side = t.cuda.Stream()
    with t.cuda.stream(side):
        step(upload(ctx, cache), x, lens.clone(), q, out)      # the workspace grows outside the capture
    t.cuda.synchronize()
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph, stream=side):
        step(kv, x, lens, q, out)
    lens.copy_(i32(ctx, [L0, 17]))
    lens2, q2, out2 = lens.clone(), t.empty_like(q), t.empty_like(out)
    for i in range(4):
        row = ctx.to_device(rng.standard_normal((B, width)).astype(np.float32))
        x.copy_(row)
        graph.replay()
        t.cuda.synchronize()
        step(kv2, row, lens2, q2, out2)
        assert t.equal(out, out2) and t.equal(q, q2) and t.equal(lens, lens2), i
        assert t.equal(kv.k, kv2.k) and t.equal(kv.v, kv2.v) and t.equal(kv.v_scale, kv2.v_scale), i


def test_same_bits_again_and_on_another_stream(ctx):
    t = ctx.torch
    rng = np.random.default_rng(6)
    hq, hkv, d, B, L = 28, 4, 128, 2, 3000
    maxp = -(-L // 16)
    cache, table = ref.Cache(B * maxp, hkv, d, rng), table_of(rng, B, maxp)
    kv, tab = upload(ctx, cache), i32(ctx, table)
    q = ctx.to_device(rng.standard_normal((B * 6, hq, d)).astype(np.float32))
    lens = i32(ctx, [L - 6, 50])
    first = ctx.gqa_prefill_attn_i8(q, kv, tab, lens, 6, L)
    side = t.cuda.Stream()
    side.wait_stream(t.cuda.current_stream())
    with t.cuda.stream(side):
        again = ctx.gqa_prefill_attn_i8(q, kv, tab, lens, 6, L)
    t.cuda.synchronize()
    assert t.equal(first, again)


def test_refusals_on_the_device(ctx):
    t = ctx.torch
    kv = lgx.KvCacheI8.empty(ctx, 4, 2, 64)
    tab, lens = t.zeros((1, 4), dtype=t.int32, device=ctx.dev), t.ones(1, dtype=t.int32, device=ctx.dev)
    q = t.zeros((1, 4, 64), device=ctx.dev)
    for bad, status in ((lambda: ctx.gqa_decode_attn_i8(q, kv, tab, lens, 65), "LGX_OUT_OF_BOUNDS"),
                        (lambda: ctx.gqa_decode_attn_i8(q, kv, tab, lens, 64, lgx.AttnOpts(softcap=-1.0)), "LGX_INVALID_ARGUMENT"),
                        (lambda: ctx.gqa_decode_attn_i8(t.zeros((1, 34, 64), device=ctx.dev), kv, tab, lens, 64), "LGX_UNSUPPORTED"),
                        (lambda: ctx.gqa_decode_attn_i8(t.zeros((1, 3, 64), device=ctx.dev), kv, tab, lens, 64), "LGX_INVALID_ARGUMENT")):
        with pytest.raises(lgx.LgxError) as e:
            bad()
        assert e.value.status_name == status
    for bad in (lambda: ctx.gqa_decode_attn_i8(q.half(), kv, tab, lens, 64),
                lambda: ctx.gqa_decode_attn_i8(q.transpose(1, 2), kv, tab, lens, 64),
                lambda: ctx.gqa_decode_attn_i8(q, kv, tab, lens.long(), 64),
                lambda: ctx.gqa_decode_attn_i8(q, kv, tab.cpu(), lens, 64),
                lambda: ctx.gqa_decode_attn_i8(q, kv, tab, lens, 64, lgx.AttnOpts(slopes=t.zeros(3, device=ctx.dev))),
                lambda: ctx.gqa_prefill_attn_i8(q, kv, tab, lens, 2, 64),
                lambda: lgx.KvCacheI8(kv.k, kv.k, kv.k_scale, kv.v_scale),
                lambda: ctx.rope_kv_append_i8(q, None, None, lens, tab, kv)):
        with pytest.raises(ValueError):
            bad()
