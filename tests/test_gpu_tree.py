"""Trees of drafted tokens: plan, append to the binary16 cache, the walk over those that
hold, and the rows moved together."""
import numpy as np
import pytest
import torch

import logicaffeine_amd as lgx
import tree_ref as ref_

pytestmark = pytest.mark.gpu
I32 = np.int32


@pytest.mark.parametrize("B,N,span", [(1, 1, 1), (3, 6, 1), (5, 64, 3), (2, 65, 12), (40, 100, 30), (3, 256, 1), (4, 256, 255)])
@pytest.mark.parametrize("padded", [False, True])
def test_plan(ctx, B, N, span, padded):
    rng = np.random.default_rng(N)
    parent = ref_.random_trees(rng, B, N, span)
    n = rng.integers(0, N + 1, B).astype(I32) if padded else None
    depth, mask = ctx.tree_plan(ctx.to_device(parent), ctx.to_device(n) if padded else None)
    for b in range(B):
        sees, want = ref_.ancestors(parent[b])
        k = n[b] if padded else N
        assert np.array_equal(depth[b, :k].cpu().numpy(), want[:k]) and not depth[b, k:].any()
        assert np.array_equal(mask[b, :k].cpu().numpy(), ref_.words(sees)[:k]) and not mask[b, k:].any()


def test_plan_takes_other_parents_for_roots(ctx):
    parent = np.array([[5, 0, 2, -7, 4, 2**31 - 1, -2**31, 6]], I32)
    depth, mask = ctx.tree_plan(ctx.to_device(parent))
    assert depth[0].tolist() == [0, 1, 0, 0, 0, 0, 0, 1]
    assert mask[0, :, 0].tolist() == [1, 3, 4, 8, 16, 32, 64, 192]


@pytest.mark.parametrize("B,N", [(1, 1), (7, 6), (20, 64), (9, 130), (3, 256)])
def test_accept(ctx, B, N):
    """Few different tokens: long paths, and siblings with the same token."""
    rng = np.random.default_rng(B)
    for vocab in (1, 2, 5):
        parent = ref_.random_trees(rng, B, N)
        tokens, picked = (rng.integers(0, vocab, (B, N)).astype(I32) for _ in range(2))
        n, lens = rng.integers(0, N + 1, B).astype(I32), rng.integers(0, 1000, B).astype(I32)
        n[0] = N
        dev = [ctx.to_device(x) for x in (tokens, parent, picked)]
        before = torch.full((B,), -9, dtype=torch.int32, device=ctx.dev)
        path, count, token, new = ctx.tree_accept(*dev, ctx.to_device(lens), ctx.to_device(n), next_tokens=before)
        for b in range(B):
            want, last = ref_.accept(tokens[b], parent[b], picked[b], n[b])
            assert path[b].tolist() == want + [-1] * (N - len(want)) and int(count[b]) == len(want)
            assert int(token[b]) == (-9 if last is None else last) and int(new[b]) == lens[b] + len(want)
        path2, count2, _, none = ctx.tree_accept(*dev)
        assert none is None and int(count2[0]) == int(count[0]) and torch.equal(path2[0], path[0])


def cache(ctx, rng, B, maxp, hkv, d, extra=3, bits=False):
    """Random pages and a table of distinct ones."""
    pages = B * maxp + extra
    k, v = (torch.as_tensor(rng.standard_normal((pages, hkv, 16, d)).astype(np.float16)).to(ctx.dev) for _ in range(2))
    table = rng.permutation(pages)[:B * maxp].reshape(B, maxp).astype(I32)
    kv = lgx.KvCacheF16(k.view(torch.int16), v.view(torch.int16)) if bits else lgx.KvCacheF16(k, v)
    return kv, table


@pytest.mark.parametrize("hkv,d", [(1, 64), (2, 128), (5, 64), (4, 128)])
@pytest.mark.parametrize("N", [1, 6, 40, 300])
def test_keep(ctx, hkv, d, N):
    """Rows moved in place in the caches of 67 layers, more than a launch takes, at
    any start; other rows and pages keep their bits."""
    rng = np.random.default_rng(N + d)
    B, maxp, layers = 4, N // 16 + 5, 67 if N == 6 else 2
    caches, host = [], []
    _, table = cache(ctx, rng, B, maxp, hkv, d)
    for _ in range(layers):
        kv, _ = cache(ctx, rng, B, maxp, hkv, d)
        caches.append(kv)
        host.append([kv.k.cpu().numpy().copy(), kv.v.cpu().numpy().copy()])
    start = rng.integers(0, 16 * maxp - N + 1, B).astype(I32)
    keep, count = np.full((B, N), -1, I32), rng.integers(0, N + 1, B).astype(I32)
    count[0] = N                                      # every row stays
    for b in range(B):
        keep[b, :count[b]] = np.sort(rng.permutation(N)[:count[b]])
        for pair in host:
            for x in pair:
                ref_.keep_rows(x, table[b], start[b], keep[b, :count[b]])
    ctx.kv_keep(caches, *(ctx.to_device(x) for x in (table, start, keep, count)))
    for kv, (k, v) in zip(caches, host):
        assert np.array_equal(kv.k.cpu().numpy(), k) and np.array_equal(kv.v.cpu().numpy(), v)


def test_keep_leaves_what_is_outside(ctx):
    """Rows past the table, on bad pages or negative, counts outside [0, N], sequences that
    keep nothing: not touched, and the rest is."""
    rng = np.random.default_rng(2)
    kv, table = cache(ctx, rng, 4, 3, 2, 64)
    before = kv.k.cpu().numpy().copy()
    table[1, 2], table[2, 0] = 10**6, -1
    start = np.array([44, 20, 0, -5], I32)
    keep = np.array([[0, 3, 6, 9], [2, 5, 12, 13], [3, 17, 18, 20], [-1, 2, 3, 4]], I32)
    ctx.kv_keep([kv], *(ctx.to_device(x) for x in (table, start, keep, np.array([9, 4, 3, 4], I32))))
    row = lambda b, t: before[table[b, t // 16], :, t % 16].copy()  # noqa: E731
    want = before.copy()
    want[table[0, 2], :, 13] = row(0, 47)                       # 47 -> 45; 50 and 53 are no rows
    want[table[1, 1], :, 4], want[table[1, 1], :, 5] = row(1, 22), row(1, 25)
    for i, t in ((1, 2), (2, 3), (3, 4)):                       # a start below 0 counts as 0
        want[table[3, 0], :, i] = row(3, t)
    got = kv.k.cpu().numpy()
    # sequence 2: rows 0 .. on the missing page, 17 and 18 would go to 1 and 2 of it
    assert np.array_equal(got, want)
    ctx.kv_keep([kv], *(ctx.to_device(x) for x in (table, start, keep, np.array([0, -4, 0, 0], I32))))
    assert np.array_equal(kv.k.cpu().numpy(), want)


@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (28, 4, 128), (1, 1, 128), (3, 3, 64)])
@pytest.mark.parametrize("bits", [False, True])
def test_append_of_a_run_is_the_single_rows(ctx, hq, hkv, d, bits):
    """Without depths: the bits of lgx_rope_kv_append row by row."""
    rng = np.random.default_rng(d)
    B, N, maxp = 5, 21, 4
    kv, table = cache(ctx, rng, B, maxp, hkv, d, bits=bits)
    other = [kv.k.clone(), kv.v.clone()]
    lens = np.array([0, 1, 15, 30, 40], I32)
    x = torch.randn(B * N, (hq + 2 * hkv) * d, device=ctx.dev) * 3
    bias = torch.randn((hq + 2 * hkv) * d, device=ctx.dev)
    rope = lgx.Rope.tables(ctx, 64, d)
    dt, dl = ctx.to_device(table), ctx.to_device(lens)
    q = ctx.rope_kv_append_rows(x, bias, rope, dl, dt, kv, N)
    for j in range(N):
        rows = x.view(B, N, -1)[:, j].contiguous()
        one = ctx.rope_kv_append(rows, bias, rope.cos, rope.sin, dl + j, dt, other[0].view(torch.int16),
                                 other[1].view(torch.int16), hq, 64)
        assert torch.equal(one, q.view(B, N, hq, d)[:, j])
    assert torch.equal(kv.k, other[0]) and torch.equal(kv.v, other[1])


def rotated(x, pos, cos, sin, rot, inter):
    """[rows][heads][d] in 64 bits."""
    c, s = cos.astype(np.float64)[pos][:, None], sin.astype(np.float64)[pos][:, None]
    y = x.astype(np.float64).copy()
    lo, hi = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = x[..., lo].astype(np.float64), x[..., hi].astype(np.float64)
    y[..., lo], y[..., hi] = a * c - b * s, b * c + a * s
    return y


@pytest.mark.parametrize("d,rot", [(64, 64), (64, 32), (64, 10), (64, 0), (128, 128), (128, 64), (128, 72), (128, 2)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("shift", [0, 1])
def test_append_of_trees(ctx, d, rot, inter, shift):
    """Positions by depth, slots by number, padding left alone; rows 16-byte aligned or not.
    x + bias, two products and their sum round by 2^-24 each of at most |x0| + |x1| +
    |b0| + |b1|: q within 2^-22 of that; K and V by half a step of binary16 more."""
    rng = np.random.default_rng(rot)
    B, N, hq, hkv, maxp = 6, 19, 6, 2, 5
    kv, table = cache(ctx, rng, B, maxp, hkv, d)
    k0, v0 = kv.k.cpu().numpy().copy(), kv.v.cpu().numpy().copy()
    parent = ref_.random_trees(rng, B, N)
    n, lens = rng.integers(0, N + 1, B).astype(I32), rng.integers(0, 16 * maxp - N, B).astype(I32)
    depth, _ = ctx.tree_plan(ctx.to_device(parent))
    width = (hq + 2 * hkv) * d
    store = torch.randn(B * N * width + shift, device=ctx.dev)
    x, bias = store[shift:].view(B * N, width), torch.randn(width, device=ctx.dev)
    rope = lgx.Rope.tables(ctx, 90, rot, interleaved=inter) if rot else \
        lgx.Rope(torch.zeros(1, 0, device=ctx.dev), torch.zeros(1, 0, device=ctx.dev))
    q0 = torch.full((B * N, hq, d), 7.0, device=ctx.dev)
    q = ctx.rope_kv_append_rows(x, bias, rope, ctx.to_device(lens), ctx.to_device(table), kv, N, depth=depth,
                                n_new=ctx.to_device(n), q_out=q0).cpu().numpy().reshape(B, N, hq, d)
    xs, bs = x.cpu().numpy().reshape(B, N, -1, d), bias.cpu().numpy().reshape(-1, d)
    k, v = kv.k.cpu().numpy(), kv.v.cpu().numpy()
    cos, sin = rope.cos.cpu().numpy(), rope.sin.cpu().numpy()
    for b in range(B):
        pos = lens[b] + depth[b].cpu().numpy()
        whole = xs[b].astype(np.float64) + bs
        mag = np.abs(whole).max(-1, keepdims=True) * 2.0 ** -21 if rot else np.abs(whole) * 2.0 ** -23
        y = rotated(whole, pos, cos, sin, rot, inter) if rot else whole
        m = n[b]
        assert (np.abs(q[b, :m] - y[:m, :hq]) <= mag[:m, :hq]).all() and (q[b, m:] == 7.0).all()
        for j in range(m):
            t = lens[b] + j
            page = table[b, t // 16]
            for got, want, tol in ((k, y[j, hq:hq + hkv], mag[j, hq:hq + hkv]), (v, whole[j, hq + hkv:], mag[j, hq + hkv:])):
                assert (np.abs(got[page, :, t % 16] - want) <= tol + np.abs(want) * 2.0 ** -11 + 2.0 ** -25).all()
            k[page, :, t % 16], v[page, :, t % 16] = k0[page, :, t % 16], v0[page, :, t % 16]
    assert np.array_equal(k, k0) and np.array_equal(v, v0)


def test_append_at_the_edges(ctx):
    """Slots past the table, pages outside the cache, lengths and positions out of range:
    q is written, keys and values are not, positions clamp to the tables."""
    rng = np.random.default_rng(0)
    kv, table = cache(ctx, rng, 4, 2, 1, 64)
    table[1, 1], table[2, 0] = kv.num_pages, -1
    lens = np.array([30, 15, -4, 2**31 - 1], I32)
    depth = np.array([[0, 1, 2], [0, 100, -100], [0, 1, 2], [2**31 - 1, 0, 0]], I32)
    k0 = kv.k.clone()
    x = torch.randn(12, 3 * 64, device=ctx.dev)
    rope = lgx.Rope.tables(ctx, 40, 64)
    q = ctx.rope_kv_append_rows(x, None, rope, ctx.to_device(lens), ctx.to_device(table), kv, 3, depth=ctx.to_device(depth))
    pos = np.array([30, 31, 32, 15, 39, 0, 0, 1, 2, 39, 32, 32])
    want = rotated(x.cpu().numpy().reshape(12, 3, 64), pos, rope.cos.cpu().numpy(), rope.sin.cpu().numpy(), 64, False)
    assert np.abs(q.cpu().numpy()[:, 0] - want[:, 0]).max() <= 2.0 ** -21 * np.abs(want).max()
    changed = (kv.k != k0).any(-1).any(1).nonzero().tolist()
    assert sorted(map(tuple, changed)) == sorted([(int(table[0, 1]), 14), (int(table[0, 1]), 15), (int(table[1, 0]), 15)])


def test_argument_checks(ctx):
    rng = np.random.default_rng(0)
    kv, table = cache(ctx, rng, 2, 2, 1, 64)
    t, lens = ctx.to_device(table), torch.zeros(2, dtype=torch.int32, device=ctx.dev)
    two = torch.zeros(2, 4, dtype=torch.int32, device=ctx.dev)
    x, rope = torch.zeros(8, 192, device=ctx.dev), lgx.Rope.tables(ctx, 8, 64)
    for bad in (lambda: lgx.KvCacheF16(kv.k.float(), kv.v.float()), lambda: lgx.KvCacheF16(kv.k, kv.v.view(torch.int16)),
                lambda: lgx.KvCacheF16(kv.k[:, :, :8], kv.v), lambda: ctx.tree_plan(two[0]), lambda: ctx.tree_plan(two.long()),
                lambda: ctx.tree_accept(two, two, two[:, :3]), lambda: ctx.tree_accept(two, two, two, lens[:1]),
                lambda: ctx.kv_keep([], t, lens, two, lens), lambda: ctx.kv_keep([kv], t, lens, two[:1], lens),
                lambda: ctx.rope_kv_append_rows(x, None, rope, lens, t, kv, 3),
                lambda: ctx.rope_kv_append_rows(x, None, rope, lens, t, kv, 4, depth=two[:, :2]),
                lambda: ctx.rope_kv_append_rows(x.t(), None, rope, lens, t, kv, 4)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(lgx.LgxError):
        ctx.tree_plan(torch.zeros(1, 257, dtype=torch.int32, device=ctx.dev))
    other, _ = cache(ctx, rng, 2, 2, 2, 64)
    with pytest.raises(lgx.LgxError):
        ctx.kv_keep([kv, other], t, lens, two, lens)
