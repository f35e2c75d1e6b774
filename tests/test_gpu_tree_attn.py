"""Attention of draft trees over the binary16 cache against the definition in 64 bits."""
import numpy as np
import pytest
import torch

import logicaffeine_amd as lgx
import tree_ref as ref_

pytestmark = pytest.mark.gpu
I32 = np.int32


def reference(q, k, v, table, sl, n, sees, depth, scale=None, cap=0.0, window=0, slopes=None):
    """[n][hq][d] of one sequence and the bound of each result: q, k, v in 64 bits, tokens by
    the table; sees [N][N], depth [N].

    Bound.  A score's error is at most A (2^-21 + (2 d / 8 + 8) 2^-24), A = scale sum |q k|:
    q's two parts leave 2^-22, the matrix unit rounds after groups of eight products of
    both, scaling and distances add a few roundings of the score.  A weight is off by that,
    by the rounding of its exponent (|score| 2^-24, within 8 A 2^-24 but for a distance's share,
    added below), by 2^-22 of exp2 and 2^-22 of its two parts, and sums of hundreds of tiles
    by less than 2^-19.  A result, a mean of values by weights, is off by twice a
    weight's error times the largest value that the row sees, and has one more rounding."""
    hq, hkv, d = q.shape[1], k.shape[1], q.shape[2]
    T = sl + n
    rows = [table[t // 16] for t in range(T)], [t % 16 for t in range(T)]
    K, V = k[rows[0], :, rows[1]].astype(np.float64), v[rows[0], :, rows[1]].astype(np.float64)   # [T][hkv][d]
    pos = np.concatenate([np.arange(sl), sl + depth[:n]])
    out, tol = np.zeros((n, hq, d)), np.zeros((n, hq))
    scale = 1 / np.sqrt(d) if scale is None else scale
    for j in range(n):
        back = sl + depth[j] - pos
        on = np.concatenate([np.ones(sl, bool), sees[j, :n]])
        if window:
            on &= back < window
        if not on.any():
            continue
        for h in range(hq):
            g = h // (hq // hkv)
            x = q[j, h].astype(np.float64)
            with np.errstate(all="ignore"):
                s = K[on][:, g] @ x * scale
                A = np.abs(scale) * (np.abs(K[on][:, g]) @ np.abs(x)).max()
                s = cap * np.tanh(s / cap) if cap else s
                if slopes is not None:
                    s = s - float(slopes[h]) * back[on]
                    A = A + 4 * np.abs(slopes[h] * back[on]).max()
                w = np.exp(s - s.max())
                out[j, h] = (w[:, None] * V[on][:, g]).sum(0) / w.sum()
            tol[j, h] = np.abs(V[on][:, g]).max() * (2 * A * (2.0 ** -21 + (d / 4 + 16) * 2.0 ** -24) + 2.0 ** -18)
    return out, tol


def make(ctx, rng, B, N, hq, hkv, d, lens, n=None, span=4, spare=1, dtype=torch.float16):
    """A case on both sides: a cache of random pages, of which those that no sequence
    names, and slots behind the last node, hold NaN."""
    lens = np.asarray(lens, I32)
    maxp = -(-(int(lens.max()) + N) // 16) + spare
    pages = B * maxp + 2
    k, v = (rng.standard_normal((pages, hkv, 16, d)).astype(np.float16) for _ in range(2))
    table = rng.permutation(pages)[:B * maxp].reshape(B, maxp).astype(I32)
    nodes = np.full(B, N, I32) if n is None else np.asarray(n, I32)
    used = np.zeros((pages, 16), bool)
    for b in range(B):
        for t in range(lens[b] + min(max(nodes[b], 0), N)):
            used[table[b, t // 16], t % 16] = True
    k.transpose(0, 2, 1, 3)[~used] = np.nan
    v.transpose(0, 2, 1, 3)[~used] = np.nan
    parent = ref_.random_trees(rng, B, N, span)
    q = rng.standard_normal((B * N, hq, d)).astype(np.float32)
    kv = lgx.KvCacheF16(*(torch.as_tensor(x).to(ctx.dev).view(dtype) for x in (k, v)))
    return dict(q=q, k=k, v=v, table=table, lens=lens, n=nodes, parent=parent, kv=kv, B=B, N=N, hq=hq, d=d, given=n is not None)


def run(ctx, s, opts=None, top=None, plan=True, mask=None):
    depth, bits = ctx.tree_plan(ctx.to_device(s["parent"])) if plan else (None, mask)
    out = torch.full((s["B"] * s["N"], s["hq"], s["d"]), 7.0, device=ctx.dev)
    got = ctx.gqa_tree_attn(ctx.to_device(s["q"]), s["kv"], ctx.to_device(s["table"]), ctx.to_device(s["lens"]), s["N"],
                            int(s["lens"].max()) if top is None else top, mask=bits, depth=depth,
                            n_nodes=ctx.to_device(s["n"]) if s["given"] else None, opts=opts, out=out)
    assert got is out
    return out.cpu().numpy().reshape(s["B"], s["N"], s["hq"], s["d"])


def check(s, got, sees=None, depth=None, only=None, **more):
    err = norm = 0.0
    for b in range(s["B"]) if only is None else only:
        n = min(max(s["n"][b], 0), s["N"])
        a, dep = ref_.ancestors(s["parent"][b])
        a, dep = (a if sees is None else sees[b]), (dep if depth is None else depth)
        want, tol = reference(s["q"].reshape(s["B"], s["N"], s["hq"], s["d"])[b, :n], s["k"], s["v"], s["table"][b], int(s["lens"][b]), n,
                              a, dep, **more)
        assert np.isfinite(got[b, :n]).all(), b
        off = np.abs(got[b, :n] - want)
        assert (off <= tol[..., None]).all(), (b, (off / np.maximum(tol[..., None], 1e-30)).max())
        assert (got[b, n:] == 7.0).all()
        err, norm = err + (off ** 2).sum(), norm + (want ** 2).sum()
    # random inputs: as documented
    assert err <= (1e-6) ** 2 * norm or not norm


SHAPES = [(14, 2, 64), (28, 4, 128), (12, 2, 128), (3, 3, 64), (16, 1, 64), (16, 1, 128), (2, 1, 128)]


@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("N", [1, 2, 5, 17, 64, 70])
def test_trees_behind_short_contexts(ctx, hq, hkv, d, N):
    """Lengths around pages and tiles, padding, nothing cached at all."""
    rng = np.random.default_rng(N * d + hq)
    lens = [0, 1, 15, 16, 63, 64, 65, 130]
    s = make(ctx, rng, 8, N, hq, hkv, d, lens)
    check(s, run(ctx, s))
    s = make(ctx, rng, 8, N, hq, hkv, d, lens, n=np.minimum(rng.integers(-1, N + 2, 8), 2 * N))
    check(s, run(ctx, s))


@pytest.mark.parametrize("wgs", [1, 5])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("opts", [False, True])
def test_other_splits(wgs, d, opts, monkeypatch):
    """Runs of tiles for fewer and for more workgroups than there are by default."""
    monkeypatch.setenv("LGX_TREE_WGS", str(wgs))
    ctx = lgx.Context(0)
    rng = np.random.default_rng(wgs)
    o, more = (lgx.AttnOpts(softcap=20.0, window=150), dict(cap=20.0, window=150)) if opts else (None, {})
    for hq, hkv, N, lens in ((4, 2, 1, [300, 5]), (14, 2, 13, [200, 700, 64]), (7, 1, 40, [1000]), (2, 1, 2, [5000, 90])):
        s = make(ctx, rng, len(lens), N, hq, hkv, d, lens, n=[N] + [max(1, N - 3)] * (len(lens) - 1))
        check(s, run(ctx, s, o), **more)
    ctx.close()


@pytest.mark.parametrize("lens", [[330] * 140, [330, 290] * 70, [400, 1] * 70, [400] + [30] * 139, [1000] * 100 + [0] * 40])
def test_batches_that_fill_the_device(ctx, lens):
    """Sequences of about one length are not split, others are."""
    rng = np.random.default_rng(sum(lens))
    s = make(ctx, rng, 140, 2, 4, 2, 64, lens, n=rng.integers(0, 3, 140))
    check(s, run(ctx, s), only=[0, 1, 2, 57, 99, 100, 138, 139])


@pytest.mark.parametrize("hq,hkv,d", SHAPES[:3])
@pytest.mark.parametrize("B,N,L", [(1, 6, 3000), (3, 12, 1000), (2, 64, 2100), (1, 256, 700), (5, 1, 2500), (40, 3, 300)])
def test_long_contexts(ctx, hq, hkv, d, B, N, L):
    """Splits over the tiles, ragged lengths, one far shorter than max_seq_len says."""
    rng = np.random.default_rng(L)
    lens = rng.integers(0, L + 1, B)
    lens[0] = L
    s = make(ctx, rng, B, N, hq, hkv, d, lens, n=rng.integers(1, N + 1, B), span=9, spare=L // 32)
    got = run(ctx, s)
    check(s, got, only=range(min(B, 4)))
    # a larger bound splits otherwise: each result within its own error of the same value
    wide = run(ctx, s, top=L + (L // 32 - 1) * 16)
    check(s, wide, only=range(min(B, 4)))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("opts", [dict(cap=5.0), dict(window=1), dict(window=40), dict(window=700), dict(slopes=True),
                                  dict(scale=0.3), dict(scale=-0.1), dict(cap=30.0, window=129, slopes=True, scale=0.2)])
def test_options(ctx, d, opts):
    rng = np.random.default_rng(5)
    hq, hkv = 6, 2
    more = dict(opts)
    slopes = (2.0 ** -np.arange(1, hq + 1)).astype(np.float32) if opts.get("slopes") else None
    more["slopes"] = slopes
    o = lgx.AttnOpts(scale=opts.get("scale", 0.0), softcap=opts.get("cap", 0.0), window=opts.get("window", 0),
                     slopes=None if slopes is None else ctx.to_device(slopes))
    for N, lens in ((1, [50, 0, 900]), (20, [0, 33, 64, 500]), (90, [10, 300])):
        s = make(ctx, rng, len(lens), N, hq, hkv, d, lens, n=[N] * (len(lens) - 1) + [max(1, N // 2)])
        check(s, run(ctx, s, o), **more)


@pytest.mark.parametrize("d", [64, 128])
def test_any_mask_and_no_mask(ctx, d):
    """Masks that are no trees, rows that see nothing (nor is anything cached), bits past the
    last node; without mask and depths a causal run."""
    rng = np.random.default_rng(6)
    for N, lens in ((3, [0, 0, 20]), (66, [0, 5, 128, 200]), (130, [61, 0])):
        B = len(lens)
        s = make(ctx, rng, B, N, 10, 2, d, lens, n=[N] * (B - 1) + [N - 1])
        sees = rng.random((B, N, N)) < 0.3
        sees[:, ::5] = False
        bits = ref_.words(sees) | (np.int64(-1) << np.int64(N % 64) if N % 64 else np.int64(0)) * (np.arange(-(-N // 64)) == N // 64)
        got = run(ctx, s, plan=False, mask=ctx.to_device(np.ascontiguousarray(bits)))
        check(s, got, sees=sees, depth=np.arange(N))
        for b in range(B):
            if lens[b] == 0:
                assert not got[b, :s["n"][b]][~sees[b, :s["n"][b], :s["n"][b]].any(1)].any()
        causal = np.broadcast_to(np.tril(np.ones((N, N), bool)), (B, N, N))
        check(s, run(ctx, s, plan=False), sees=causal, depth=np.arange(N))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window", [0, 30])
def test_infinities_and_nan_where_a_row_does_not_see(ctx, d, window):
    """Nodes whose keys and values are not finite leave their siblings' rows as they are;
    cached ones outside the window too.  Rows that see them are not finite."""
    rng = np.random.default_rng(7)
    B, N, hq, hkv = 3, 24, 14, 2
    s = make(ctx, rng, B, N, hq, hkv, d, [100, 3, 61], span=3)
    o, more = (lgx.AttnOpts(window=window), dict(window=window)) if window else (None, {})
    clean = run(ctx, s, o)
    check(s, clean, **more)
    bad = [7, 20]
    for b in range(B):
        for i, (x, val) in zip(bad, ((s["v"], np.inf), (s["k"], np.nan))):
            t = s["lens"][b] + i
            x[s["table"][b, t // 16], :, t % 16, ::3] = val
    if window:
        s["v"][s["table"][0, 1], :, 3] = -np.inf
        s["k"][s["table"][0, 0], :, 5] = np.nan
    s["kv"] = lgx.KvCacheF16(*(torch.as_tensor(s[x]).to(ctx.dev) for x in "kv"))
    got = run(ctx, s, o)
    for b in range(B):
        sees, _ = ref_.ancestors(s["parent"][b])
        hit = sees[:, bad].any(1)
        assert hit.any() and not hit.all()
        want, tol = reference(s["q"].reshape(B, N, hq, d)[b], np.nan_to_num(s["k"], posinf=0, neginf=0), np.nan_to_num(s["v"], posinf=0, neginf=0),
                              s["table"][b], int(s["lens"][b]), N, *ref_.ancestors(s["parent"][b]), **more)
        assert np.isfinite(got[b][~hit]).all()
        assert (np.abs(got[b] - want)[~hit] <= tol[~hit][..., None]).all()
        assert (~np.isfinite(got[b][hit][..., ::3])).all()
        only_v = sees[:, 7] & ~sees[:, 20]
        assert np.isposinf(got[b][only_v][..., ::3]).all() and np.isfinite(got[b][only_v][..., 1::3]).all()


def spoil(s, b, tokens, step=1):
    """Infinities and NaN in the keys and values of a sequence's tokens; the cache on the device anew."""
    for i, t in enumerate(tokens):
        at = s["table"][b, t // 16], slice(None), t % 16, slice(None, None, step)
        s["k"][at] = (np.nan, np.inf, -np.inf)[i % 3]
        s["v"][at] = (np.inf, np.nan, -np.inf)[i % 3]
    s["kv"] = lgx.KvCacheF16(*(torch.as_tensor(s[x]).to(s["kv"].device) for x in "kv"))


def check_unseen(s, got, sees, depth, bad, **more):
    """Rows that see no bad token equal the definition's over finite ones (those that see nothing
    at all are zeros); bad: tokens by sequence."""
    B, N, hq, d = got.shape
    finite = [np.nan_to_num(s[x], nan=0, posinf=0, neginf=0) for x in "kv"]
    for b in range(B):
        n, sl = min(max(s["n"][b], 0), N), int(s["lens"][b])
        pos = np.concatenate([np.arange(sl), sl + depth[b][:n]])
        on = np.concatenate([np.ones((n, sl), bool), sees[b][:n, :n]], 1)
        if more.get("window"):
            on &= sl + depth[b][:n, None] - pos < more["window"]
        clean = ~on[:, [t for t in bad[b] if t < sl + n]].any(1)
        assert clean.any(), b
        want, tol = reference(s["q"].reshape(B, N, hq, d)[b, :n], *finite, s["table"][b], sl, n, sees[b], depth[b], **more)
        off = np.abs(got[b, :n] - want)
        assert np.isfinite(got[b, :n][clean]).all(), (b, np.flatnonzero(clean & ~np.isfinite(got[b, :n]).all((1, 2))))
        assert (off <= tol[..., None])[clean].all(), b
        assert not got[b, :n][~on.any(1)].any()


@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (8, 2, 128), (6, 6, 128)])
@pytest.mark.parametrize("N,lens", [(24, [250]), (100, [448]), (24, [250, 1000, 63]), (100, [448, 30, 2000]), (256, [700])])
@pytest.mark.parametrize("window", [0, 60])
def test_bad_drafts_behind_a_split(ctx, hq, hkv, d, N, lens, window):
    """A context of more than four tiles is split: of the last run, with later nodes alone, the
    first nodes see nothing, whatever stands there."""
    rng = np.random.default_rng(N + len(lens))
    s = make(ctx, rng, len(lens), N, hq, hkv, d, lens, span=5)
    s["parent"][:, 3] = 0                         # node 2 is no one's parent
    for j in range(4, N):
        s["parent"][:, j] = np.where(s["parent"][:, j] == 2, 1, s["parent"][:, j])
    bad = [[int(L) + i for i in (2, N - 3, N - 2, N - 1)] for L in lens]
    for b in range(len(lens)):
        spoil(s, b, bad[b], step=3)
    o, more = (lgx.AttnOpts(window=window), dict(window=window)) if window else (None, {})
    tree = [ref_.ancestors(p) for p in s["parent"]]
    check_unseen(s, run(ctx, s, o), [t[0] for t in tree], [t[1] for t in tree], bad, **more)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens", [[0, 0, 0], [0, 900, 1], [300, 0, 64]])
def test_rows_that_see_nothing_over_bad_slots(ctx, d, lens):
    """Empty masks, nothing cached, every slot of the nodes an infinity or a NaN: zeros; and
    rows that see a few finite nodes only."""
    rng = np.random.default_rng(d + sum(lens))
    B, N = 3, 70
    s = make(ctx, rng, B, N, 10, 2, d, lens, n=[N, N - 1, N - 5])
    sees = np.zeros((B, N, N), bool)
    finite = np.arange(N) % 9 == 4
    sees[:, 1::2] = finite
    bad = [[int(lens[b]) + i for i in range(N) if not finite[i]] for b in range(B)]
    for b in range(B):
        spoil(s, b, bad[b])
    got = run(ctx, s, plan=False, mask=ctx.to_device(ref_.words(sees)))
    check_unseen(s, got, sees, [np.arange(N)] * B, bad)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window", [400, 900])
def test_bad_tokens_ahead_of_the_windows_of_deep_nodes(ctx, d, window):
    """The first runs of tiles lie in the windows of the shallow nodes alone."""
    rng = np.random.default_rng(window)
    N, L = 20, 1500
    s = make(ctx, rng, 1, N, 4, 2, d, [L])
    depth = np.where(np.arange(N) < 5, 0, 350 + 3 * np.arange(N))
    sees = np.tril(np.ones((1, N, N), bool))
    bad = [list(range(L - window + 1, L - window + 300, 7))]
    spoil(s, 0, bad[0])
    out = torch.full((N, 4, d), 7.0, device=ctx.dev)
    ctx.gqa_tree_attn(ctx.to_device(s["q"]), s["kv"], ctx.to_device(s["table"]), ctx.to_device(s["lens"]), N, L,
                      depth=ctx.to_device(depth[None].astype(I32)), opts=lgx.AttnOpts(window=window), out=out)
    check_unseen(s, out.cpu().numpy().reshape(1, N, 4, d), sees, [depth], bad, window=window)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window", [0, 50, 2**31 - 1])
def test_depths_up_to_the_last_position(ctx, d, window):
    """Positions end at 2^31 - 1: nodes that would stand behind it stand there, with the
    distances and the window of that position."""
    rng = np.random.default_rng(d)
    B, N, hq, lens = 3, 9, 4, [400, 70, 0]
    s = make(ctx, rng, B, N, hq, 2, d, lens)
    most = 2**31 - 1
    depth = np.array([0, 1, most, 2**30, most - 399, most - 400, most - 10, 2**31 - 70, -5])
    slopes = (2.0 ** -np.arange(29, 29 + hq)).astype(np.float32)
    sees = np.tril(np.ones((N, N), bool))
    out = torch.full((B * N, hq, d), 7.0, device=ctx.dev)
    ctx.gqa_tree_attn(ctx.to_device(s["q"]), s["kv"], ctx.to_device(s["table"]), ctx.to_device(s["lens"]), N, 400,
                      depth=ctx.to_device(np.tile(depth.astype(I32), (B, 1))),
                      opts=lgx.AttnOpts(window=window, slopes=ctx.to_device(slopes)), out=out)
    # each sequence by itself: the last position is as far behind its length as that leaves
    got = out.cpu().numpy().reshape(B, N, hq, d)
    for b in range(B):
        check(s, got, sees=[sees] * B, depth=np.clip(depth, 0, most - lens[b]), only=[b], window=window, slopes=slopes)


def test_bad_queries_and_far_scales(ctx):
    """NaN or infinite query rows give NaN and nothing else does; rows of 2^-60 and 2^40 keep
    their bits; scores of thousands."""
    rng = np.random.default_rng(9)
    s = make(ctx, rng, 2, 5, 4, 2, 64, [70, 200])
    q = s["q"].reshape(2, 5, 4, 64)
    q[0, 1, 2, 5], q[1, 3, 0, 0] = np.nan, np.inf
    q[0, 0] *= 2.0 ** -60
    q[1, 0] *= 500.0
    q[1, 1] = 0.0
    got = run(ctx, s)
    assert np.isnan(got[0, 1, 2]).all() and np.isnan(got[1, 3, 0]).all()
    q[0, 1, 2], q[1, 3, 0] = 0, 0
    for b in range(2):
        want, tol = reference(q[b], s["k"], s["v"], s["table"][b], int(s["lens"][b]), 5, *ref_.ancestors(s["parent"][b]))
        off = np.abs(got[b] - want)
        off[1 if b == 0 else 3, 2 if b == 0 else 0] = 0
        assert (off <= tol[..., None]).all()


def test_queries_far_above_one(ctx):
    """Rows of 2^40 and 2^100 beside ordinary ones, and rows of 2^-60, with scales that leave
    moderate scores."""
    rng = np.random.default_rng(15)
    for d in (64, 128):
        for up in (40, 100, -60):
            s = make(ctx, rng, 2, 5, 4, 2, d, [70, 300])
            s["q"].reshape(2, 5, -1)[:, ::2 if up > 0 else 1] *= 2.0 ** up
            scale = 2.0 ** (-3 - up)
            for more in (dict(), dict(cap=10.0), dict(window=33)):
                o = lgx.AttnOpts(scale=scale, softcap=more.get("cap", 0.0), window=more.get("window", 0))
                check(s, run(ctx, s, o), scale=scale, **more)


def test_constant_values_and_one_token(ctx):
    """Weights sum to one: constant V comes out as it is, one seen token as its V row."""
    rng = np.random.default_rng(10)
    s = make(ctx, rng, 2, 9, 14, 2, 128, [500, 0])
    s["v"][np.isfinite(s["v"])] = 1.5
    s["kv"] = lgx.KvCacheF16(*(torch.as_tensor(s[x]).to(ctx.dev) for x in "kv"))
    assert np.abs(run(ctx, s) - 1.5).max() <= 1.5 * 2.0 ** -20
    s = make(ctx, rng, 1, 1, 14, 2, 128, [0])
    got = run(ctx, s)
    v = s["v"][s["table"][0, 0], :, 0].astype(np.float32)
    assert np.abs(got[0, 0] - np.repeat(v, 7, axis=0)).max() <= np.abs(v).max() * 2.0 ** -20


def test_lengths_and_pages_out_of_range(ctx):
    """Lengths clamp to [0, max_seq_len] and pages to the cache, as the other attentions' do."""
    rng = np.random.default_rng(11)
    s = make(ctx, rng, 3, 4, 4, 2, 64, [100, 100, 40], spare=2)
    s["k"], s["v"] = (np.nan_to_num(s[x], nan=0.5) for x in "kv")
    s["kv"] = lgx.KvCacheF16(*(torch.as_tensor(s[x]).to(ctx.dev) for x in "kv"))
    s["table"][2, 1], s["table"][2, 0] = 10**6, -3
    true = s["lens"].copy()
    s["lens"] = np.array([2**31 - 1, 100, 40], I32)
    got = run(ctx, s, top=100)
    s["lens"] = true
    s["table"][2, 1], s["table"][2, 0] = len(s["k"]) - 1, 0
    check(s, got)
    s["lens"] = np.array([-5, 0, 0], I32)
    a = run(ctx, s, top=0)
    s["lens"] = np.array([0, 0, 0], I32)
    check(s, a)


def test_same_bits_again_in_a_graph_and_on_another_stream(ctx):
    """A step's attention recorded twice, two graphs that share the workspace, replayed in
    turn with lengths that change; each replay equals the call made then and there."""
    rng = np.random.default_rng(12)
    cases = [make(ctx, rng, 2, 8, 28, 4, 128, [3000, 1100]), make(ctx, rng, 1, 30, 14, 2, 64, [2000])]
    held = []
    for s in cases:
        depth, mask = ctx.tree_plan(ctx.to_device(s["parent"]))
        lens, q = ctx.to_device(s["lens"]), ctx.to_device(s["q"])
        args = (s["kv"], ctx.to_device(s["table"]), lens, s["N"], int(s["lens"].max()))
        out = torch.zeros_like(q)
        ctx.gqa_tree_attn(q, *args, mask=mask, depth=depth, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ctx.gqa_tree_attn(q, *args, mask=mask, depth=depth, out=out)
        held.append((graph, q, args, mask, depth, out, lens))
    for turn in range(3):
        for graph, q, args, mask, depth, out, lens in held:
            q.mul_(-0.9)
            lens.sub_(17 * turn)
            graph.replay()
            torch.cuda.synchronize()
            want = ctx.gqa_tree_attn(q, *args, mask=mask, depth=depth)
            assert torch.equal(out, want) and torch.isfinite(out).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ctx.gqa_tree_attn(q, *args, mask=mask, depth=depth)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, want)


@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (28, 4, 128)])
def test_a_decode_step_agrees_with_the_exact_one(ctx, hq, hkv, d):
    """N = 1 without mask: lgx_gqa_decode_attn over the token and those before it, both within
    binary32's error of the definition."""
    rng = np.random.default_rng(13)
    s = make(ctx, rng, 4, 1, hq, hkv, d, [0, 30, 255, 900], dtype=torch.int16)
    for x in "kv":
        s[x] = np.nan_to_num(s[x])
    s["kv"] = lgx.KvCacheF16(*(torch.as_tensor(s[x]).to(ctx.dev).view(torch.int16) for x in "kv"))
    got = run(ctx, s, plan=False)
    exact = ctx.gqa_decode_attn(ctx.to_device(s["q"]), s["kv"].k, s["kv"].v, ctx.to_device(s["table"]),
                                ctx.to_device(s["lens"] + 1), 901).cpu().numpy()
    check(s, got)
    check(s, exact.reshape(got.shape))


def test_far_pages(ctx):
    """Pages past 2^32 bytes of K."""
    hkv, d, pages = 8, 128, 140000                     # 32 KiB of K per page
    k, v = (torch.empty(pages, hkv, 16, d, dtype=torch.float16, device=ctx.dev) for _ in range(2))
    rng = np.random.default_rng(14)
    table = np.array([[139999, 3, 131073, 65536, 138000, 70000]], I32)
    small = [rng.standard_normal((6, hkv, 16, d)).astype(np.float16) for _ in range(2)]
    for x, y in ((k, small[0]), (v, small[1])):
        x[torch.as_tensor(table[0].astype(np.int64)).to(ctx.dev)] = torch.as_tensor(y).to(ctx.dev)
    s = dict(q=rng.standard_normal((7, 16, d)).astype(np.float32), k=small[0], v=small[1], table=table, lens=np.array([80], I32),
             n=np.array([7], I32), parent=ref_.random_trees(rng, 1, 7), kv=lgx.KvCacheF16(k, v), B=1, N=7, hq=16, d=d, given=False)
    got = run(ctx, s)
    s["table"] = np.arange(6, dtype=I32)[None]
    check(s, got)
    # rows moved and appended there
    s["table"] = table
    t, lens = ctx.to_device(table), ctx.to_device(s["lens"])
    ctx.kv_keep([s["kv"]], t, lens, ctx.to_device(np.array([[0, 3, 6]], I32)), ctx.to_device(np.array([3], I32)))
    assert torch.equal(k[70000, :, 1].cpu(), torch.as_tensor(small[0][5, :, 3])) and \
        torch.equal(v[70000, :, 2].cpu(), torch.as_tensor(small[1][5, :, 6]))
    x = torch.randn(1, (16 + 2 * hkv) * d, device=ctx.dev)
    ctx.rope_kv_append_rows(x, None, lgx.Rope(torch.zeros(1, 0, device=ctx.dev), torch.zeros(1, 0, device=ctx.dev)), lens + 9, t, s["kv"])
    assert torch.equal(v[70000, :, 9], x.view(-1, d)[16 + hkv:].half())


def test_argument_checks(ctx):
    rng = np.random.default_rng(0)
    s = make(ctx, rng, 2, 4, 4, 2, 64, [20, 10])
    q, t, lens = ctx.to_device(s["q"]), ctx.to_device(s["table"]), ctx.to_device(s["lens"])
    depth, mask = ctx.tree_plan(ctx.to_device(s["parent"]))
    call = lambda **k: ctx.gqa_tree_attn(**{**dict(q=q, kv=s["kv"], page_table=t, seq_len=lens, N=4, max_seq_len=20), **k})  # noqa: E731
    call()
    for k in (dict(N=3), dict(mask=mask[:, :3]), dict(mask=mask.int()), dict(depth=depth.long()), dict(n_nodes=lens[:1]),
              dict(q=q.double()), dict(q=q[:, :, :32]), dict(out=q[:4]), dict(seq_len=lens.cpu()), dict(page_table=t.t()),
              dict(opts=lgx.AttnOpts(slopes=torch.zeros(3, device=ctx.dev)))):
        with pytest.raises(ValueError):
            call(**k)
    for k in (dict(max_seq_len=16 * t.shape[1] - 3), dict(max_seq_len=-1), dict(opts=lgx.AttnOpts(softcap=-1.0)),
              dict(opts=lgx.AttnOpts(window=-1)), dict(opts=lgx.AttnOpts(scale=float("nan")))):
        with pytest.raises(lgx.LgxError):
            call(**k)
