"""The 8-bit KV cache at the edges of what its calls take, against the definition."""
import numpy as np
import pytest

import kv8_ref as ref
import logicaffeine_amd as lgx

pytestmark = pytest.mark.gpu


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
