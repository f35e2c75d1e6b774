"""Sampling with per-row settings against the definition in 64 bits."""
import itertools

import numpy as np
import pytest
import torch

import tree_ref as ref_

pytestmark = pytest.mark.gpu


def check(ctx, logits, u, T=None, k=None, p=None, mp=None):
    """Tokens equal the definition's; probabilities are one binary32 rounding (2^-24) and
    sums in units of 2^-42 (1e-12) off.  A row whose draw or share stands within 1e-9 of a
    border would say nothing; there is none in these tests but where sums are exact."""
    m = len(logits)
    f = lambda x, t: None if x is None else torch.as_tensor(np.broadcast_to(np.asarray(x, t), (m,)).copy()).to(ctx.dev)  # noqa: E731
    x = logits if isinstance(logits, torch.Tensor) else torch.as_tensor(np.asarray(logits, np.float32)).to(ctx.dev)
    out, prob = ctx.sample_filtered(x, f(u, np.float32), f(T, np.float32), f(k, np.int32), f(p, np.float32), f(mp, np.float32))
    out, prob = out.cpu().numpy(), prob.cpu().numpy()
    rows = x.cpu().numpy()
    at = lambda v, i, d, t: t(d if v is None else np.broadcast_to(np.asarray(v, t), (m,))[i])  # noqa: E731
    for i in range(m):
        want, share = ref_.choose(rows[i], at(u, i, 0, np.float32), at(T, i, 1, np.float32), int(at(k, i, 0, np.int32)),
                                  at(p, i, 1, np.float32), at(mp, i, 0, np.float32))
        assert out[i] == want, (i, out[i], want)
        assert abs(prob[i] - share) <= 2.0 ** -24 * share + 1e-12, (i, prob[i], share)
    return out


def peaked(rng, m, V):
    x = 2.0 * rng.standard_normal((m, V))
    for row in x:
        row[rng.integers(0, V, max(1, min(V // 4, 40)))] += 12 + 3 * rng.standard_normal()
    return x.astype(np.float32)


@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 1000, 4096, 4097, 32003, 151936])
def test_every_mix_of_settings(ctx, V):
    rng = np.random.default_rng(V)
    sets = list(itertools.product((0.0, 0.5, 1.0), (0, 1, 7, 50), (1.0, 0.9, 0.3), (0.0, 0.05)))
    x = peaked(rng, len(sets), V)
    T, k, p, mp = (np.array(c) for c in zip(*sets))
    check(ctx, x, rng.random(len(sets), dtype=np.float32), T, k, p, mp)


@pytest.mark.parametrize("V", [1500, 32003, 152064])
@pytest.mark.parametrize("scale", [1e-3, 0.1, 1.0])
def test_flat_rows_keep_most_of_the_vocabulary(ctx, V, scale):
    """More tokens than the list in LDS holds."""
    rng = np.random.default_rng(V)
    sets = [(1.0, 0, 0.95, 0.0), (0.7, 0, 1.0, 0.3), (1.3, V // 2, 1.0, 0.0), (1.0, V - 1, 0.5, 0.0), (1.0, 4097, 0.9, 0.01),
            (1.0, 0, 1.0, 0.0), (2.0, 0, 0.02, 0.0)]
    x = (scale * rng.standard_normal((len(sets), V))).astype(np.float32)
    T, k, p, mp = (np.array(c) for c in zip(*sets))
    check(ctx, x, rng.random(len(sets), dtype=np.float32), T, k, p, mp)


def test_equal_logits_count_by_index(ctx):
    """Exact shares: of V equal tokens top_k keeps the first k, top_p the first ceil(p V),
    and u takes the floor(u n)-th."""
    for V in (8, 1000, 6000, 40000):
        x = torch.zeros(6, V, device=ctx.dev)
        x[:, ::2] = -0.0
        u = [0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 0.125]
        assert check(ctx, x, u).tolist() == [0, V // 4, V // 2, 3 * V // 4, V - 1, V // 8]
        assert check(ctx, x, u, p=0.5).tolist() == [0, V // 8, V // 4, 3 * V // 8, V // 2 - 1, V // 16]
        assert check(ctx, x, u, k=V // 2).tolist() == [0, V // 8, V // 4, 3 * V // 8, V // 2 - 1, V // 16]
        assert check(ctx, x, u, k=V // 2, p=0.5, mp=1.0).tolist() == [0, V // 16, V // 8, 3 * V // 16, V // 4 - 1, V // 32]
        assert check(ctx, x, u, T=0.0).tolist() == [0] * 6


def test_ties_at_the_border(ctx):
    """Tokens of one logit straddle top_k and top_p: the lower indexes stay."""
    rng = np.random.default_rng(3)
    for V, levels in ((300, 5), (20000, 9), (152064, 40)):
        x = np.log(2.0) * rng.integers(0, levels, (24, V)).astype(np.float32)
        k = rng.integers(1, V, 24)
        check(ctx, x, rng.random(24, dtype=np.float32), k=k)
        check(ctx, x, rng.random(24, dtype=np.float32), k=k, p=0.6)
        check(ctx, x, rng.random(24, dtype=np.float32), p=rng.random(24, dtype=np.float32))
        check(ctx, x, rng.random(24, dtype=np.float32), mp=0.2, p=0.99)


def test_tails_of_weights_near_the_unit(ctx):
    """Half a million tokens that weigh about as much as a weight is rounded to, 2^-43 (those
    below it weigh nothing).  A sum over n of them is off by e = n 2^-43 at most, and by 2^-41 of
    it for exp and for binary64.  So a token is right if the definition's draw falls within 2 e
    of its interval; with top-p, whose cut may be 2 e off as well, which moves both ends and
    the draw by up to 4 e, within 6 e."""
    V = 1 << 19
    rng = np.random.default_rng(19)
    u = np.array([0.0, 2.0 ** -30, 2.0 ** -25, 2.0 ** -24, 1.5 * 2.0 ** -24, 2.0 ** -23, 2.0 ** -22, 0.5], np.float32)
    m = len(u)
    for tail in (np.full(V, np.log(1.49 * 2.0 ** -42)), np.full(V, np.log(0.49 * 2.0 ** -42)),
                 rng.uniform(np.log(2.0 ** -45), np.log(2.0 ** -40), V)):
        row = tail.astype(np.float32)
        row[V - 1] = 0.0
        x = torch.as_tensor(row).to(ctx.dev).expand(m, V).contiguous()
        w = np.exp(row.astype(np.longdouble))
        for k, p in ((V - 1, 1.0), (300000, 1.0), (0, 1 - 2.0 ** -24), (0, 1 - 2.0 ** -23), (V - 1, 1 - 2.0 ** -24)):
            f = lambda v, t: torch.full((m,), v, dtype=t, device=ctx.dev)  # noqa: E731
            out, prob = (y.cpu().numpy() for y in ctx.sample_filtered(x, torch.as_tensor(u).to(ctx.dev), top_k=f(k, torch.int32),
                                                                      top_p=f(p, torch.float32)))
            order = np.argsort(-row, kind="stable")[:k or V]
            up = np.cumsum(w[order])
            e = len(order) * 2.0 ** -43 + up[-1] * 2.0 ** -41
            room = 2 * e if p >= 1 else 6 * e
            cut = len(order) if p >= 1 else int((up - w[order] < np.longdouble(np.float32(p)) * up[-1] + 2 * e).sum())
            kept = np.sort(order[:cut])
            c = np.cumsum(w[kept])
            for i in range(m):
                at = int(np.searchsorted(kept, out[i]))
                assert at < cut and kept[at] == out[i], (k, p, u[i], out[i])
                t = np.longdouble(u[i]) * c[-1]
                assert c[at] - w[out[i]] - room <= t <= c[at] + room, (k, p, u[i], out[i])
                assert abs(prob[i] - w[out[i]] / c[-1]) <= 2.0 ** -24 * prob[i] + room + 2.0 ** -43


def test_infinities_nan_and_masked_rows(ctx):
    inf, nan = np.inf, np.nan
    rng = np.random.default_rng(1)
    V = 5000
    x = rng.standard_normal((12, V)).astype(np.float32)
    x[0] = nan
    x[1] = -inf
    x[2, ::2], x[2, 1::2] = nan, -inf
    x[3, 1:] = -inf                                   # one token left
    x[4, :4900] = nan
    x[5, [7, 4000]] = inf
    x[6, 11:] = -inf
    x[7] = -3e38
    x[7, 9] = 3e38
    x[8, ::3] = nan
    x[9] = np.float32(1e-45)
    x[10, 100:200] = inf
    x[10, 300] = nan
    u = np.linspace(0, 0.999, 12).astype(np.float32)
    for T, k, p, mp in ((1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 20, 1.0, 0.0), (0.8, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.1),
                        (1.5, 3000, 0.7, 0.001), (1e-30, 0, 0.5, 0.0)):
        check(ctx, x, u, T, k, p, mp)


def test_settings_outside_their_ranges(ctx):
    """As documented: none, the first token, or the nearest in range."""
    rng = np.random.default_rng(8)
    x = peaked(rng, 9, 3000)
    nan, inf = np.nan, np.inf
    check(ctx, x, 0.4, k=[-5, 0, 3000, 3001, 2**31 - 1, -2**31, 1, 2999, 2])
    check(ctx, x, 0.4, p=[0.0, -1.0, 1.0, 2.0, nan, inf, -inf, 1e-30, 0.999999])
    check(ctx, x, 0.4, mp=[0.0, -1.0, 1.0, 2.0, nan, inf, -inf, 1e-30, 0.999999])
    check(ctx, x, 0.4, T=[0.0, -1.0, -0.0, nan, -inf, 1e-20, 1e3, 100.0, 5.0])
    for p in (None, 0.9):
        check(ctx, x, [0.0, -1.0, 1.0, 2.0, nan, inf, -inf, 1 - 2.0 ** -24, 2.0 ** -149], p=p)


def test_rows_of_a_wider_tensor_and_settings_left_out(ctx):
    rng = np.random.default_rng(4)
    for V, ld, off in ((1000, 1003, 1), (32000, 32004, 0), (4095, 5000, 3)):
        wide = torch.as_tensor(rng.standard_normal((7, ld)).astype(np.float32)).to(ctx.dev)
        wide[:, V + off:] = 99.0
        check(ctx, wide[:, off:off + V], rng.random(7, dtype=np.float32), k=40, p=0.9)
        check(ctx, wide[:, off:off + V], rng.random(7, dtype=np.float32))


def test_a_rows_token_does_not_depend_on_its_batch(ctx):
    x = torch.randn(200, 20000, device=ctx.dev) * 3
    u = torch.rand(200, device=ctx.dev)
    p = torch.full((200,), 0.9, device=ctx.dev)
    all_, prob = ctx.sample_filtered(x, u, top_p=p)
    for i in (0, 7, 199):
        one, q = ctx.sample_filtered(x[i:i + 1], u[i:i + 1], top_p=p[i:i + 1])
        assert int(one) == int(all_[i]) and float(q) == float(prob[i])


def test_frequencies_follow_the_filtered_distribution(ctx):
    """200000 evenly spaced numbers: each token's count is its share, up to one at each end
    of its interval."""
    m = 50000
    x = torch.tensor([[1.0, 3.0, 2.0, -1.0, 2.5, 0.0, 3.0, -4.0]], device=ctx.dev).repeat(m, 1)
    u = ((torch.arange(m, device=ctx.dev, dtype=torch.float64) + 0.5) / m).float()
    out, _ = ctx.sample_filtered(x, u, top_k=torch.full((m,), 6, dtype=torch.int32, device=ctx.dev),
                                 top_p=torch.full((m,), 0.93, device=ctx.dev))
    w = np.exp(x[0].double().cpu().numpy())
    order = np.argsort(-w, kind="stable")[:6]
    c = np.cumsum(w[order])
    kept = order[:int((c - w[order] < float(np.float32(0.93)) * c[-1]).sum())]
    count = np.bincount(out.cpu().numpy(), minlength=8)
    share = np.where(np.isin(np.arange(8), kept), w, 0) / w[kept].sum()
    assert np.abs(count - m * share).max() <= 2


def test_in_a_graph_and_on_another_stream(ctx):
    x, u = torch.randn(40, 30000, device=ctx.dev), torch.rand(40, device=ctx.dev)
    p = torch.rand(40, device=ctx.dev)
    out, prob = torch.zeros(40, dtype=torch.int32, device=ctx.dev), torch.zeros(40, device=ctx.dev)
    ctx.sample_filtered(x, u, top_p=p, out=out, prob=prob)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.sample_filtered(x, u, top_p=p, out=out, prob=prob)
    for seed in range(3):
        torch.manual_seed(seed)
        x.normal_()
        u.uniform_()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want, _ = ctx.sample_filtered(x, u, top_p=p)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)


def test_argument_checks(ctx):
    x, u = torch.zeros(2, 10, device=ctx.dev), torch.zeros(2, device=ctx.dev)
    import logicaffeine_amd as lgx
    for bad in (lambda: ctx.sample_filtered(x.double(), u), lambda: ctx.sample_filtered(x.t(), u), lambda: ctx.sample_filtered(x[0], u),
                lambda: ctx.sample_filtered(x, u[:1]), lambda: ctx.sample_filtered(x, u, top_k=u), lambda: ctx.sample_filtered(x.cpu(), u),
                lambda: ctx.sample_filtered(x, u, out=u), lambda: ctx.sample_filtered(x, None)):
        with pytest.raises((ValueError, AttributeError)):
            bad()
    with pytest.raises(lgx.LgxError):
        ctx.sample_filtered(x[:1].expand(2, 10), u)


@pytest.mark.parametrize("V", [20000, 151936])
def test_many_wide_rows_among_others(ctx, V):
    """Rows whose kept tokens are more than one workgroup lists, by top-p, min-p and both, with
    ties at the border, beside rows of every other kind."""
    rng = np.random.default_rng(V)
    sets = list(itertools.product((1.0, 1.7, 0.0), (0, 40), (1.0, 0.9, 0.5, 0.99), (0.0, 0.3, 0.02)))
    x = (0.5 * rng.standard_normal((len(sets), V))).astype(np.float32)
    T, k, p, mp = (np.array(c) for c in zip(*sets))
    check(ctx, x, rng.random(len(sets), dtype=np.float32), T, k, p, mp)
    check(ctx, np.round(x, 1), rng.random(len(sets), dtype=np.float32), T, k, p, mp)
    one = np.where(rng.random(x.shape) < 0.9, np.float32(0.25), x)     # most of a row in one logit
    check(ctx, one, rng.random(len(sets), dtype=np.float32), T, k, p, mp)


def test_more_wide_rows_than_there_is_room_for(ctx):
    """Bins of 64 MiB hold some 1300 rows of 100000 logits."""
    m, V = 1500, 100000
    x = torch.randn(1, V, device=ctx.dev) * 0.2
    wide = x.expand(m, V).contiguous()
    p = torch.full((m,), 0.9, device=ctx.dev)
    u = torch.linspace(0, 0.9999, m, device=ctx.dev)
    out, prob = ctx.sample_filtered(wide, u, top_p=p)
    row = x[0].cpu().numpy()
    for i in (0, 1, 700, 1299, 1300, 1420, 1499):
        want, share = ref_.choose(row, float(u[i]), p=np.float32(0.9))
        assert int(out[i]) == want and abs(float(prob[i]) - share) <= 2.0 ** -24 * share + 1e-12
    assert (out[1:] >= out[:-1]).all()


@pytest.mark.parametrize("m,V,scale", [(7, 151937, 0.1), (96, 152064, 0.1), (64, 4097, 0.01), (200, 60000, 1.0)])
def test_wide_rows_give_the_same_again(ctx, m, V, scale):
    """Which workgroup goes on with a wide row depends on their order, its token does not:
    again and again, with another call's values in the workspace between, and alone."""
    g = torch.Generator(device="cuda").manual_seed(m)
    x, other = (scale * torch.randn(m, V, device="cuda", generator=g) for _ in range(2))
    u, p, mp = (torch.rand(m, device="cuda", generator=g) for _ in range(3))
    p, mp = 0.5 + 0.5 * p, 0.2 * mp
    first = [y.clone() for y in ctx.sample_filtered(x, u, top_p=p, min_p=mp)]
    for i in range(30):
        if i % 2:
            ctx.sample_filtered(other, u, top_p=p, min_p=mp)
        for a, b in zip(first, ctx.sample_filtered(x, u, top_p=p, min_p=mp)):
            assert torch.equal(a, b)
    for i in range(0, m, 7):
        one = slice(i, i + 1)
        for a, b in zip(first, ctx.sample_filtered(x[one], u[one], top_p=p[one], min_p=mp[one])):
            assert torch.equal(a[one], b)
