"""Drafts, sampling and a cache's pages together, as a server uses them: sequences of a
small network go on by trees of drafts, share pages where one forks from another, and
yield the tokens that they would yield one at a time."""
import numpy as np
import pytest
import torch

import logicaffeine_amd as lgx
import tree_ref as R

pytestmark = pytest.mark.gpu

LAYERS, HQ, HKV, D, VOCAB, PAGE, MAXP = 2, 6, 2, 64, 300, 16, 12
H = HQ * D


class Net:
    """Token embedding, LAYERS of attention, logits; in 64 bits on the host for one
    sequence, by the library for a batch's trees of drafts."""

    def __init__(self, ctx, rng):
        self.ctx = ctx
        self.emb = rng.standard_normal((VOCAB, H)).astype(np.float32)
        self.wqkv = [(rng.standard_normal((H, (HQ + 2 * HKV) * D)) * H ** -0.5).astype(np.float32) for _ in range(LAYERS)]
        self.out = (rng.standard_normal((H, VOCAB)) * 2 * H ** -0.5).astype(np.float32)
        self.gpu = {k: [torch.tensor(x, device="cuda") for x in v] if isinstance(v, list) else torch.tensor(v, device="cuda")
                    for k, v in (("emb", self.emb), ("wqkv", self.wqkv), ("out", self.out))}
        self.rope = lgx.Rope.tables(ctx, MAXP * PAGE, D, theta=1e4)
        ang = np.arange(MAXP * PAGE)[:, None] * 1e4 ** (-2.0 * np.arange(D // 2) / D)
        self.cos, self.sin = np.cos(ang)[:, None], np.sin(ang)[:, None]

    def turn(self, x, first):
        a, b, n = x[..., :D // 2], x[..., D // 2:], len(x)
        c, s = self.cos[first:first + n], self.sin[first:first + n]
        return np.concatenate([a * c - b * s, a * s + b * c], -1)

    def logits(self, tokens):
        """Behind the last of the tokens."""
        x = self.emb[tokens].astype(np.float64)
        for w in self.wqkv:
            qkv = (x @ w).reshape(len(x), HQ + 2 * HKV, D)
            q = self.turn(qkv[:, :HQ], 0)
            k, v = (y.astype(np.float16).astype(np.float64) for y in (self.turn(qkv[:, HQ:HQ + HKV], 0), qkv[:, HQ + HKV:]))
            s = np.einsum("ighd,jgd->ghij", q.reshape(-1, HKV, HQ // HKV, D), k) / np.sqrt(D)
            s = np.where(np.tri(len(x), dtype=bool), s, -np.inf)
            p = np.exp(s - s.max(-1, keepdims=True))
            x = x + np.einsum("ghij,jgd->ighd", p / p.sum(-1, keepdims=True), v).reshape(len(x), H)
        return x[-1] @ self.out

    def step(self, tokens, N, lens, table, caches, depth, mask, n, top):
        """Logits [B*N][VOCAB] behind every node."""
        x = self.gpu["emb"][tokens.reshape(-1).long()]
        for w, kv in zip(self.gpu["wqkv"], caches):
            q = self.ctx.rope_kv_append_rows(x @ w, None, self.rope, lens, table, kv, N, depth, n)
            o = torch.zeros_like(q)               # rows that are no nodes are left as they are
            self.ctx.gqa_tree_attn(q, kv, table, lens, N, top, mask, depth, n, out=o)
            x = x + o.reshape(-1, H)
        return x @ self.gpu["out"]


class Server:
    """State on the device of S sequences; one round checks a tree of N drafts of each."""

    def __init__(self, net, S, N, pages):
        ctx = self.ctx = net.ctx
        self.net, self.S, self.N = net, S, N
        self.caches = [lgx.KvCacheF16.empty(ctx, pages, HKV, D) for _ in range(LAYERS)]
        for kv in self.caches:
            kv.k.fill_(float("nan"))              # what nothing wrote, nothing may read
            kv.v.fill_(float("nan"))
        self.pool = lgx.PagePool.empty(ctx, pages)
        self.planes = lgx.PagePlanes([x for kv in self.caches for x in (kv.k, kv.v)])
        i32 = dict(dtype=torch.int32, device="cuda")
        self.table = torch.full((S, MAXP), -1, **i32)
        self.lens, self.n, self.last = torch.zeros(S, **i32), torch.zeros(S, **i32), torch.zeros(S, **i32)
        self.tokens, self.parent = torch.zeros((S, N), **i32), torch.full((S, N), -1, **i32)
        self.room = (torch.zeros((S, 2), **i32), torch.zeros(1, **i32), torch.zeros(1, **i32))
        self.u = torch.zeros(S * N, device="cuda")
        self.settings = {}

    def round(self):
        ctx, N = self.ctx, self.N
        copies, n_copies, _ = ctx.pages_reserve(self.pool, self.table, self.lens, self.n, out=self.room)
        ctx.pages_copy(self.planes, copies, n_copies)
        depth, mask = ctx.tree_plan(self.parent, self.n)
        logits = self.net.step(self.tokens, N, self.lens, self.table, self.caches, depth, mask, self.n, MAXP * PAGE - N)
        picked, _ = ctx.sample_filtered(logits, self.u, **self.settings)
        path, count, _, new = ctx.tree_accept(self.tokens, self.parent, picked.view(self.S, N), self.lens, self.n, self.last)
        ctx.kv_keep(self.caches, self.table, self.lens, path, count)
        self.lens.copy_(new)
        ctx.pages_free(self.pool, self.table, self.lens)
        self.path, self.count, self.picked = path, count, picked


@pytest.fixture(scope="module")
def ctx():
    c = lgx.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("S,N,settings", [
    (3, 1, {}), (2, 5, dict(temperature=0.0)), (4, 7, dict(temperature=1.0)), (4, 12, dict(temperature=0.8, top_k=20)),
    (3, 70, dict(temperature=1.0, top_p=0.9, min_p=0.01))])
def test_drafts_yield_the_tokens_of_single_steps(ctx, S, N, settings, captured):
    """Every sequence's tokens are those of the 64-bit network and the definition's choice,
    one at a time.  The random number of a choice belongs to the sequence and the position.
    Both sides round keys and values to binary16, and a key that 32 and 64 bits round to
    either side changes a logit by some 1e-4: random numbers are such that logits off by
    1e-3 give the same choice."""
    rng = np.random.default_rng(100 * S + N)
    net, total = Net(ctx, rng), 60
    u = rng.random((S, total + N + 2)).astype(np.float32)
    prompt = rng.integers(0, VOCAB, 21)
    T, k, p, mp = (settings.get(x, y) for x, y in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0)))

    def choice(seq, s):
        logits = net.logits(seq)
        for _ in range(100):
            x = u[s, len(seq) - 1]
            token = R.choose(logits, x, T, k, p, mp)[0]
            if all(R.choose(logits + rng.uniform(-1e-3, 1e-3, VOCAB), y, T, k, p, mp)[0] == token
                   for y in (x, x, max(x - 1e-3, 0), x + 1e-3)):
                return token
            u[s, len(seq) - 1] = rng.random()
        raise AssertionError("no choice is clear")

    want = []
    for s in range(S):                            # sequence 0's first tokens, then each its own way
        seq = list(prompt) if s == 0 else want[0][:30]
        while len(seq) < total:
            seq.append(choice(seq, s))
        want.append(seq)

    srv = Server(net, S, N, pages=S * -(-(total + N) // PAGE) + 1)
    for name, x in settings.items():
        srv.settings[name] = torch.full((S * N,), x, device="cuda", dtype=torch.int32 if name == "top_k" else torch.float32)
    graph = None

    def drafts(s, at):
        """A tree whose node 0 is token `at` of the sequence: the tokens to come among others."""
        n = int(rng.integers(1, N + 1))
        tok, par, dep = rng.integers(0, VOCAB, N), np.full(N, -1), np.zeros(N, int)
        tok[0], right = want[s][at], 0            # `right`: the last node of the true path
        for j in range(1, n):
            par[j] = right if rng.random() < 0.7 else rng.integers(0, j)
            dep[j] = dep[par[j]] + 1
            nxt = at + dep[j]
            if par[j] == right and rng.random() < 0.8 and nxt < total:
                tok[j], right = want[s][nxt], j
        return tok, par, dep, n

    def fill(live):
        tokens, parent, n = np.zeros((S, N), np.int32), np.full((S, N), -1, np.int32), np.zeros(S, np.int32)
        us = np.zeros((S, N), np.float32)
        for s in live:
            tokens[s], parent[s], dep, n[s] = drafts(s, len(have[s]) - 1)
            us[s] = u[s, np.minimum(len(have[s]) - 1 + dep, u.shape[1] - 1)]
        srv.tokens.copy_(torch.tensor(tokens))
        srv.parent.copy_(torch.tensor(parent))
        srv.n.copy_(torch.tensor(n))
        srv.u.copy_(torch.tensor(us.reshape(-1)))

    def go():
        nonlocal graph
        if not captured:
            return srv.round()
        if graph is None:
            saved = [x.clone() for x in (srv.pool.ref, srv.table, srv.lens, srv.last)]
            planes = [x.clone() for x in srv.planes.tensors]
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):         # libraries set up, workspaces grow
                srv.round()
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                srv.round()
            for x, y in zip((srv.pool.ref, srv.table, srv.lens, srv.last, *srv.planes.tensors), saved + planes):
                x.copy_(y)
        graph.replay()

    # the prompt but its last token, as a run of new tokens in pieces of N
    have = {0: list(prompt)}
    for i in range(0, len(prompt) - 1, N):
        part = prompt[i:min(i + N, len(prompt) - 1)]
        one = torch.zeros((S, N), dtype=torch.int32, device="cuda")
        one[0, :len(part)] = torch.tensor(part, device="cuda")
        n = torch.tensor([len(part)] + [0] * (S - 1), dtype=torch.int32, device="cuda")
        ctx.pages_reserve(srv.pool, srv.table, srv.lens, n, out=srv.room)
        net.step(one, N, srv.lens, srv.table, srv.caches, None, None, n, MAXP * PAGE - N)
        srv.lens += n
    rounds = 0
    while any(len(x) < total for x in have.values()):
        live = [s for s in have if len(have[s]) < total]
        fill(live)
        go()
        count, path, last = (x.cpu().numpy() for x in (srv.count, srv.path, srv.last))
        tokens, lens = srv.tokens.cpu().numpy(), srv.lens.cpu().numpy()
        assert int(srv.room[2]) == 0
        for s in live:
            new = [int(tokens[s, j]) for j in path[s, 1:count[s]]] + [int(last[s])]
            have[s] += new
            assert count[s] >= 1 and have[s][:total] == want[s][:len(have[s])], (s, rounds)
            assert lens[s] == len(have[s]) - 1
        if len(have) == 1 and len(have[0]) >= 32:
            # the others fork from the first, back to 29 cached tokens, amid a page
            dst = torch.arange(1, S, dtype=torch.int32, device="cuda")
            ctx.pages_fork(srv.pool, srv.table, srv.lens, torch.zeros_like(dst), dst)
            srv.lens[1:] = 29
            ctx.pages_free(srv.pool, srv.table, srv.lens)
            assert int(srv.pool.ref.max()) == S
            have.update({s: want[0][:30] for s in range(1, S)})
        rounds += 1
    # every holder accounted for, and all pages come back
    table = srv.table.cpu().numpy()
    assert np.array_equal(np.bincount(table[table >= 0], minlength=srv.pool.num_pages), srv.pool.ref.cpu().numpy())
    ctx.pages_free(srv.pool, srv.table, torch.zeros_like(srv.lens))
    assert int(srv.pool.ref.abs().sum()) == 0 and bool((srv.table == -1).all())
    if N > 1:
        assert rounds < total - len(prompt)       # drafts held


def test_two_graphs_share_a_workspace_that_grows(ctx):
    """Split attention, wide rows of logits and a reservation, whose intermediates all lie in
    the context's workspace, in two graphs replayed in turn; between the replays other inputs and
    an eager call that needs a larger workspace."""
    own = lgx.Context(0)
    rng = np.random.default_rng(8)
    B, N, hq, hkv, d, L = 2, 5, 4, 2, 64, 900
    maxp = -(-(L + N) // PAGE)
    kv = lgx.KvCacheF16(*(torch.tensor(rng.standard_normal((B * maxp, hkv, PAGE, d)), dtype=torch.float16, device="cuda")
                          for _ in range(2)))
    table = torch.arange(B * maxp, dtype=torch.int32, device="cuda").view(B, maxp)
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    q = torch.zeros((B * N, hq, d), device="cuda")
    logits, u = torch.zeros((3, 30000), device="cuda"), torch.zeros(3, device="cuda")
    top_p = torch.tensor([0.9, 0.5, 0.99], device="cuda")
    ref = torch.zeros(50, dtype=torch.int32, device="cuda")
    rows, held, need = (torch.full(s, v, dtype=torch.int32, device="cuda") for s, v in (((4, 9), -1), ((4,), 0), ((4,), 0)))

    def fill(i):
        r = np.random.default_rng(100 + i)
        lens.copy_(torch.tensor(r.integers(0, L + 1, B)))
        q.copy_(torch.tensor(r.standard_normal(q.shape)))
        logits.copy_(torch.tensor(0.2 * r.standard_normal(logits.shape)))
        u.copy_(torch.tensor(r.random(3)))
        need.copy_(torch.tensor(r.integers(0, 100, 4)))
        ref.zero_()
        rows.fill_(-1)

    def work(c):
        out = c.gqa_tree_attn(q, kv, table, lens, N, L)
        token, prob = c.sample_filtered(logits, u, top_p=top_p)
        more = c.pages_reserve(lgx.PagePool(ref), rows, held, need)
        return [out, token, prob, *more, rows, ref]

    fill(0)
    work(own)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            result = work(own)
        graphs.append((g, result))
    for i in range(8):
        g, result = graphs[i % 2]
        fill(i)
        g.replay()
        got = [x.clone() for x in result]
        fill(i)
        for x, y in zip(got, work(ctx)):
            assert torch.equal(x, y)
        if i == 3:                                # outgrows the workspace that the graphs go on using
            many = torch.randn((400, 40000), device="cuda")
            own.sample_filtered(many, torch.rand(400, device="cuda"), top_p=torch.full((400,), 0.9, device="cuda"))
    del graphs, g, result
    torch.cuda.synchronize()
    own.close()


@pytest.mark.parametrize("captured", [False, True])
def test_a_round_where_pages_run_out(ctx, captured):
    """Three sequences share a partly filled page, and the pool lacks a page for their drafts: a
    round that takes its numbers of nodes times (lacking == 0) changes nothing, however often
    it runs; once a page is free it goes on, each sequence in a page of its own.  Rows of
    padding stay zeros."""
    S, N, pages, held, hq, hkv, d, vocab = 3, 5, 4, 21, 28, 4, 128, 64
    rng = np.random.default_rng(21)
    i32 = dict(dtype=torch.int32, device="cuda")
    layers = [lgx.KvCacheF16.empty(ctx, pages, hkv, d) for _ in range(28)]
    planes = lgx.PagePlanes([x for kv in layers for x in (kv.k, kv.v)])
    pool = lgx.PagePool.empty(ctx, pages)
    q, out = (torch.zeros(S * N, hq, d, device="cuda") for _ in range(2))
    qkv = torch.tensor(rng.standard_normal((S * N, (hq + 2 * hkv) * d)), dtype=torch.float32, device="cuda")
    logits = torch.tensor(rng.standard_normal((S * N, vocab)), dtype=torch.float32, device="cuda")
    u, rope = torch.full((S * N,), 0.5, device="cuda"), lgx.Rope.tables(ctx, 4 * PAGE, d)
    tokens, parent = torch.zeros((S, N), **i32), torch.arange(-1, N - 1, **i32).repeat(S, 1)
    n, none = torch.tensor([N, N - 2, N], **i32), torch.zeros(1, **i32)
    table, lens = torch.full((S, 4), -1, **i32), torch.full((S,), held, **i32)
    table[:, :2] = torch.tensor([2, 0])
    pool.ref.copy_(torch.tensor([S, 0, S, 1]))    # page 3 is held elsewhere
    for x in planes.tensors:
        x.copy_(torch.tensor(rng.standard_normal(x.shape), dtype=x.dtype))

    def work():
        copies, n_copies, lacking = ctx.pages_reserve(pool, table, lens, n)
        live = n * (lacking == 0)
        ctx.pages_copy(planes, copies, n_copies)
        depth, mask = ctx.tree_plan(parent, live)
        for kv in layers:
            ctx.rope_kv_append_rows(qkv, None, rope, lens, table, kv, N, depth, live, q_out=q)
            ctx.gqa_tree_attn(q, kv, table, lens, N, 4 * PAGE - N, mask, depth, live, out=out)
        picked, _ = ctx.sample_filtered(logits, u)
        path, count, _, new = ctx.tree_accept(tokens, parent, picked.view(S, N), lens, live)
        ctx.kv_keep(layers, table, lens, path, count)
        lens.copy_(new)
        ctx.pages_free(pool, table, lens)
        ctx.pages_fork(pool, table, lens, none, none)     # onto itself: left out
        return lacking, count

    def state():
        return [x.clone() for x in (table, lens, pool.ref, *planes.tensors)]

    before = state()
    if captured:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            work()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            result = work()

    def go():
        if not captured:
            return work()
        graph.replay()
        return result

    for _ in range(3):
        lacking, count = go()
        assert int(lacking) == 1 and not count.any() and not q.any() and not out.any()
        for x, y in zip(before, state()):
            assert torch.equal(x, y)
    pool.ref[3] = 0
    lacking, count = go()
    assert int(lacking) == 0
    rows = table[:, 1].cpu().numpy()
    assert sorted(rows) == [0, 1, 3] and (table[:, 0] == 2).all() and pool.ref.tolist() == [1, 1, S, 1]
    assert (count >= 1).all() and torch.equal(lens, held + count)
    v = qkv.view(S, N, hq + 2 * hkv, d)[:, 0, hq + hkv:].half()
    for kv, old in zip(layers, before[3:][1::2]):
        for s in range(S):
            at = held % PAGE                      # what the page held, then node 0's row
            assert torch.equal(kv.v[rows[s], :, :at], old[0, :, :at]) and torch.equal(kv.v[rows[s], :, at], v[s])
    for x in (q, out):
        assert x.view(S, N, -1).any(-1).tolist() == [[True] * N, [True] * (N - 2) + [False] * 2, [True] * N]
