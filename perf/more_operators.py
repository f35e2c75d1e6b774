"""The operators of drafted tokens and of a cache's pages as cases that can be timed
and compared: appending the rows of a draft tree to the paged binary16 cache,
attention of such a tree over it, sampling with per-row settings from given random
numbers, accepting drafts and closing the cache's rows up behind them, and forking,
reserving, copying and freeing pages.  Shapes are those of the library's own
configurations (the 0.5B-, 1.5B- and 7B-shaped models), and `draw` gives others of
the same ranges.

`own` false: the plain form, elementary torch operations; true: the library's
calls.  `exact` states the definitions once more in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

# (query heads, KV heads, head dim, layers) of the 0.5B-, 1.5B- and 7B-shaped models
HEADS = {"0.5b": (14, 2, 64, 24), "1.5b": (12, 2, 128, 28), "7b": (28, 4, 128, 28)}
PAGE = 16
THETA = 1e6

_ctx = None


def _context():
    """One library context for the process, as a serving program keeps it."""
    global _ctx
    import logicaffeine_amd as lgx

    if _ctx is None:
        _ctx = lgx.Context(torch.cuda.current_device())
    return _ctx


# N: drafted nodes of a sequence; span: a node's parent is one of the `span` nodes
# before it (1: a chain)
def _append(name, shape, B, N, L, span=4, rot=0, pairs="half", ragged=True, padded=False):
    return dict(name=name, kind="append", shape=shape, B=B, N=N, L=L, span=span, rot=rot or HEADS[shape][2],
                pairs=pairs, ragged=ragged, padded=padded)


def _attn(name, shape, B, N, L, span=4, ragged=False, padded=False, cap=0.0, window=0, slopes=False):
    return dict(name=name, kind="attn", shape=shape, B=B, N=N, L=L, span=span, ragged=ragged, padded=padded, cap=cap,
                window=window, slopes=slopes)


def _sample(name, m, vocab, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mixed=False, flat=False):
    return dict(name=name, kind="sample", m=m, vocab=vocab, temperature=temperature, top_k=top_k, top_p=top_p,
                min_p=min_p, mixed=mixed, flat=flat)


def _commit(name, shape, B, N, L, span=4):
    return dict(name=name, kind="commit", shape=shape, B=B, N=N, L=L, span=span, ragged=True, padded=False)


def _pages(name, shape, S, L, need, cache="f16"):
    return dict(name=name, kind="pages", shape=shape, S=S, L=L, need=need, cache=cache)


def listed() -> list:
    return [
        # one user of the small model with a chain of five drafts
        _append("append-0.5b-b1-n6", "0.5b", 1, 6, 200, span=1),
        # a full batch's draft trees at the ragged positions that a server sees
        _append("append-7b-b64-n33", "7b", 64, 33, 4000, padded=True),
        # one user at the start of a conversation, a chain of drafts
        _attn("attn-0.5b-b1-n6-l200", "0.5b", 1, 6, 200, span=1),
        # one user far into a long context, a wide tree
        _attn("attn-7b-b1-n64-l8000", "7b", 1, 64, 8000, span=12),
        # a batch of ragged sequences with a small tree each
        _attn("attn-7b-b32-n16-l4096", "7b", 32, 16, 4096, ragged=True),
        # trees of differing odd sizes, capped scores over a sliding window
        _attn("attn-1.5b-b9-n201-l1500-cap", "1.5b", 9, 201, 1500, span=30, padded=True, cap=30.0, window=1000),
        # one user's next token
        _sample("sample-m1-v151936", 1, 151936, temperature=0.7, top_k=50, top_p=0.95),
        # every node of a batch's trees, each request with settings of its own
        _sample("sample-m512-v152064-mixed", 512, 152064, mixed=True),
        # the accepted drafts of one user, a small tree, all layers of the small model
        _commit("commit-0.5b-b1-n6", "0.5b", 1, 6, 200, span=3),
        # those of a batch, all layers of the large model
        _commit("commit-7b-b32-n24", "7b", 32, 24, 300),
        # one sequence forked, both go on; the 8-bit cache
        _pages("pages-0.5b-s2-i8", "0.5b", 2, 200, 6, cache="i8"),
        # a batch forked, room for trees of drafts in both halves
        _pages("pages-7b-s96", "7b", 96, 250, 24),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    """An integer of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["append", "attn", "attn", "sample", "sample", "commit", "pages"])
    shape = rng.choice(sorted(HEADS))
    hq, hkv, d, layers = HEADS[shape]
    span = rng.choice([1, 2, 4, 12])
    if kind == "append":
        B = _log_int(rng, 1, 64)
        case = _append("", shape, B, min(_log_int(rng, 1, 200), 64 * 33 // B), _log_int(rng, 1, 4000), span,
                       rng.choice([d, d, d // 2]), rng.choice(["half", "even"]), rng.random() < 0.7, rng.random() < 0.4)
    elif kind == "attn":
        # rows x heads x tokens up to that of the listed batch
        B, N, top = _log_int(rng, 1, 64), _log_int(rng, 1, 200), 32 * 16 * 28 * 4096
        while B * N * N * hq > top:
            B, N = max(1, B // 2), max(1, N // 2)
        L = min(_log_int(rng, 1, 12000), top // (B * N * hq), 32 * 4096 * 2 * 128 // (B * hkv * d))
        case = _attn("", shape, B, N, L, span, rng.random() < 0.6, rng.random() < 0.4, rng.choice([0.0, 0.0, 0.0, 25.0]),
                     rng.choice([0, 0, 0, _log_int(rng, 1, 4000)]), rng.random() < 0.2)
    elif kind == "sample":
        vocab = rng.choice([151936, 152064, _log_int(rng, 500, 150000), _log_int(rng, 500, 150000)])
        case = _sample("", _log_int(rng, 1, 512), vocab, rng.choice([1.0, 1.0, rng.uniform(0.4, 1.5), 0.0]),
                       rng.choice([0, 0, _log_int(rng, 1, 200)]), rng.choice([1.0, rng.uniform(0.7, 0.99)]),
                       rng.choice([0.0, 0.0, rng.uniform(0.01, 0.2)]), rng.random() < 0.4, rng.random() < 0.15)
    elif kind == "commit":
        case = _commit("", shape, _log_int(rng, 1, 32), _log_int(rng, 2, 24), _log_int(rng, 1, 300), span)
    else:
        case = _pages("", shape, 2 * _log_int(rng, 1, 48), _log_int(rng, 1, 250), _log_int(rng, 1, 24), rng.choice(["f16", "i8"]))
    del case["name"]
    return case


# ---- inputs ---------------------------------------------------------------

def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _lens(case, seed):
    """Committed tokens and drafted nodes of each sequence."""
    B, L, N = case["B"], case["L"], case["N"]
    cpu = torch.Generator().manual_seed(seed)
    n = torch.full((B,), L, dtype=torch.int32)
    if case["ragged"]:
        n = torch.randint(L // 8, L + 1, (B,), generator=cpu, dtype=torch.int32)
        n[0] = L
    new = torch.full((B,), N, dtype=torch.int32)
    if case["padded"]:
        new = torch.randint(1, N + 1, (B,), generator=cpu, dtype=torch.int32)
        new[0] = N
    return n, new


def _trees(case, seed):
    """Each node's parent, its depth, and the nodes that it sees as bits of 64-bit
    words: itself and its ancestors."""
    B, N = case["B"], case["N"]
    cpu = torch.Generator().manual_seed(seed + 1)
    back = torch.rand(B, N, generator=cpu)
    parent = torch.full((B, N), -1, dtype=torch.int64)
    depth = torch.zeros(B, N, dtype=torch.int64)
    sees = torch.zeros(B, N, N, dtype=torch.bool)
    at = torch.arange(B)
    for j in range(N):
        if j:
            p = j - 1 - (back[:, j] * min(j, case["span"])).long()
            parent[:, j], depth[:, j], sees[:, j] = p, depth[at, p] + 1, sees[at, p]
        sees[:, j, j] = True
    words = -(-N // 64)
    bits = torch.zeros(B, N, words, dtype=torch.int64)
    for j in range(N):
        bit = 1 << (j % 64)
        bits[:, :, j // 64] |= sees[:, :, j].long() * (bit - (1 << 64) if j % 64 == 63 else bit)
    return dict(parent=parent.int().cuda(), depth=depth.int().cuda(), mask=bits.cuda())


def _maxp(case) -> int:
    return -(-(case["L"] + case["N"]) // PAGE)


def _cache(case, g, layers=1):
    """Pages of normal keys and values [layers][2][pages][hkv][16][d] and the page table."""
    _, hkv, d, _ = HEADS[case["shape"]]
    B, maxp = case["B"], _maxp(case)
    kv = torch.empty(layers, 2, B * maxp, hkv, PAGE, d, dtype=torch.float16, device="cuda")
    for i in range(layers):
        for j in range(2):
            kv[i, j] = torch.randn(kv.shape[2:], device="cuda", generator=g, dtype=torch.float16)
    table = torch.randperm(B * maxp, device="cuda", generator=g).to(torch.int32).view(B, maxp)
    return kv, table


def _tables(case):
    """cos / sin of every position's angles, rounded once from 64 bits."""
    pos = torch.arange(case["L"] + case["N"] + 1, dtype=torch.float64, device="cuda")
    i = torch.arange(case["rot"] // 2, dtype=torch.float64, device="cuda")
    ang = pos[:, None] * THETA ** (-2.0 * i / case["rot"])
    return ang.cos().float(), ang.sin().float()


def _sample_inputs(case, g):
    m, V = case["m"], case["vocab"]
    logits = torch.empty(m, V, device="cuda")
    for lo in range(0, m, 64):
        x = torch.randn(logits[lo:lo + 64].shape, device="cuda", generator=g)
        if case["flat"]:
            logits[lo:lo + 64] = 0.1 * x
        else:
            # most of the vocabulary far below a few dozen likely tokens
            likely = torch.randint(0, V, (len(x), 40), device="cuda", generator=g)
            x = (2.0 * x).scatter_add_(1, likely, 12.0 + 3.0 * torch.randn(likely.shape, device="cuda", generator=g))
            logits[lo:lo + 64] = x
    pick = lambda *values: torch.tensor(values, device="cuda")[torch.randint(0, len(values), (m,), device="cuda", generator=g)]  # noqa: E731
    if case["mixed"]:
        more = dict(temperature=pick(0.0, 0.6, 0.8, 1.0, 1.0, 1.3), top_k=pick(0, 0, 20, 40, 100).int(), top_p=pick(1.0, 0.8, 0.9, 0.95),
                    min_p=pick(0.0, 0.0, 0.05, 0.1))
    else:
        more = {k: torch.full((m,), case[k], dtype=torch.int32 if k == "top_k" else torch.float32, device="cuda")
                for k in ("temperature", "top_k", "top_p", "min_p")}
    return dict(logits=logits, u=torch.rand(m, device="cuda", generator=g), **more)


def _commit_inputs(case, seed, g):
    """Draft trees of which a path holds: the token picked behind a node of the path
    is its child's, behind the others any."""
    B, N, layers = case["B"], case["N"], HEADS[case["shape"]][3]
    s = _trees(case, seed)
    s["kv"], s["table"] = _cache(case, g, layers)
    cpu = torch.Generator().manual_seed(seed + 2)
    tokens = torch.randint(0, 150000, (B, N), generator=cpu, dtype=torch.int32)
    picked = torch.randint(0, 150000, (B, N), generator=cpu, dtype=torch.int32)
    leaf = torch.randint(0, N, (B,), generator=cpu).tolist()
    parent = s["parent"].tolist()
    for b in range(B):
        j = leaf[b]
        while j > 0:
            picked[b, parent[b][j]] = tokens[b, j]
            j = parent[b][j]
    return dict(s, tokens=tokens.cuda(), picked=picked.cuda())


def _pages_inputs(case, seed, g):
    """The first half of S sequences hold pages, the second none; pages of every
    layer's cache."""
    _, hkv, d, layers = HEADS[case["shape"]]
    S, L, need = case["S"], case["L"], case["need"]
    maxp = -(-(L + need) // PAGE)
    cpu = torch.Generator().manual_seed(seed)
    lens = torch.zeros(S, dtype=torch.int32)
    lens[:S // 2] = torch.randint(max(1, L // 2), L + 1, (S // 2,), generator=cpu, dtype=torch.int32)
    num = S * maxp
    held = (lens + PAGE - 1) // PAGE
    order = torch.randperm(num, generator=cpu, dtype=torch.int64).to(torch.int32)
    col = torch.arange(maxp)
    own_page = col < held[:, None]
    table = torch.full((S, maxp), -1, dtype=torch.int32)
    table[own_page] = order[:int(own_page.sum())]
    ref = torch.zeros(num, dtype=torch.int32)
    ref[table[own_page].long()] = 1
    if case["cache"] == "f16":
        planes = [torch.randint(-2 ** 15, 2 ** 15, (layers, 2, num, hkv * PAGE * d), device="cuda", generator=g, dtype=torch.int16)]
    else:
        planes = [torch.randint(-127, 128, (layers, 2, num, hkv * PAGE * d), device="cuda", generator=g, dtype=torch.int8),
                  torch.randint(0, 2 ** 30, (layers, 2, num, hkv), device="cuda", generator=g, dtype=torch.int32)]
    half = torch.arange(S // 2, dtype=torch.int32)
    keep = torch.where(torch.arange(S) < S // 2, lens, 0)
    return dict(planes=planes, table=table.cuda(), ref=ref.cuda(), lens=lens.cuda(), src=half.cuda(), dst=(half + S // 2).cuda(),
                need=torch.full((S,), need, dtype=torch.int32, device="cuda"), keep=keep.int().cuda(),
                copies=torch.zeros(S, 2, dtype=torch.int32, device="cuda"), n_copies=torch.zeros(1, dtype=torch.int32, device="cuda"),
                lacking=torch.zeros(1, dtype=torch.int32, device="cuda"))


def _inputs(case, seed):
    g = _gen(seed)
    if case["kind"] == "sample":
        return dict(case=case, **_sample_inputs(case, g))
    if case["kind"] == "pages":
        return dict(case=case, **_pages_inputs(case, seed, g))
    hq, hkv, d, _ = HEADS[case["shape"]]
    n, new = _lens(case, seed)
    s = dict(case=case, lens=n.cuda(), new=new.cuda())
    if case["kind"] == "commit":
        return dict(s, **_commit_inputs(case, seed, g))
    s.update(_trees(case, seed))
    s["kv"], s["table"] = _cache(case, g)
    rows = case["B"] * case["N"]
    if case["kind"] == "append":
        s["x"] = torch.randn(rows, (hq + 2 * hkv) * d, device="cuda", generator=g)
        s["bias"] = 0.02 * torch.randn((hq + 2 * hkv) * d, device="cuda", generator=g)
        s["cos"], s["sin"] = _tables(case)
    else:
        s["q"] = torch.randn(rows, hq, d, device="cuda", generator=g)
        s["slopes"] = torch.pow(2.0, -8.0 * torch.arange(1, hq + 1, device="cuda", dtype=torch.float64) / hq).float() if case["slopes"] else None
    return s


def prepare(case, seed):
    state = _inputs(case, seed)
    kind = case["kind"]
    if kind in ("append", "attn"):
        hq, _, d, _ = HEADS[case["shape"]]
        # padding rows are left as they are: the buffer starts with zeros
        state["out"] = torch.zeros(case["B"] * case["N"], hq, d, device="cuda")
    if own:
        import logicaffeine_amd as lgx

        state["ctx"] = _context()
        if kind in ("append", "attn", "commit"):
            state["caches"] = [lgx.KvCacheF16(k, v) for k, v in state["kv"]]
        if kind == "append":
            state["rope"] = lgx.Rope(state["cos"], state["sin"], interleaved=case["pairs"] == "even")
        if kind == "attn":
            state["opts"] = lgx.AttnOpts(softcap=case["cap"], window=case["window"], slopes=state["slopes"])
        if kind == "pages":
            state["pool"] = lgx.PagePool(state["ref"])
            state["set"] = lgx.PagePlanes([plane for both in zip(*(p.flatten(0, 1) for p in state["planes"])) for plane in both])
    return state


# ---- the plain form -------------------------------------------------------

def _plain_append(s):
    case, table = s["case"], s["table"].long()
    hq, hkv, d, _ = HEADS[case["shape"]]
    B, N, rot = case["B"], case["N"], case["rot"]
    x = (s["x"] + s["bias"]).view(B, N, hq + 2 * hkv, d)
    pos = s["lens"].long()[:, None] + s["depth"].long()
    c, sn = s["cos"][pos][:, :, None], s["sin"][pos][:, :, None]
    z = x[:, :, :hq + hkv, :rot]
    if case["pairs"] == "half":
        a, b = z[..., :rot // 2], z[..., rot // 2:]
        turned = torch.cat([a * c - b * sn, b * c + a * sn], -1)
    else:
        a, b = z[..., 0::2], z[..., 1::2]
        turned = torch.stack([a * c - b * sn, b * c + a * sn], -1).flatten(-2)
    qk = torch.cat([turned, x[:, :, :hq + hkv, rot:]], -1)
    real = torch.arange(N, device="cuda") < s["new"].long()[:, None]
    q = s["out"].view(B, N, hq, d)
    q.copy_(torch.where(real[:, :, None, None], qk[:, :, :hq], q))
    slot = s["lens"].long()[:, None] + torch.arange(N, device="cuda")
    page, slot = table.gather(1, slot // PAGE)[real], (slot % PAGE)[real]
    k, v = s["kv"][0]
    k[page, :, slot] = qk[:, :, hq:][real].half()
    v[page, :, slot] = x[:, :, hq + hkv:][real].half()
    return dict(q=q.view(B * N, hq, d), k=k, v=v)


def _bits(mask, N):
    """[..., words] 64-bit words as truth values [..., N]."""
    j = torch.arange(N, device=mask.device)
    return ((mask[..., j // 64] >> (j % 64)) & 1) != 0


def _plain_attn(s):
    case = s["case"]
    hq, hkv, d, _ = HEADS[case["shape"]]
    B, N, G = case["B"], case["N"], hq // hkv
    T = s["table"].shape[1] * PAGE
    page = s["table"].long()
    k, v = (x[page].transpose(1, 2).reshape(B, hkv, T, d).float() for x in s["kv"][0])
    q = s["q"].view(B, N, hkv, G, d).transpose(1, 2).reshape(B, hkv, N * G, d)
    w = torch.matmul(q, k.transpose(2, 3).contiguous()).view(B, hkv, N, G, T)
    w *= 1.0 / math.sqrt(d)
    if case["cap"]:
        w = case["cap"] * torch.tanh(w / case["cap"])
    t = torch.arange(T, device="cuda")
    node = t - s["lens"].long()[:, None]                                # [B][T]: the node in a slot
    drafted = (node >= 0) & (node < s["new"].long()[:, None])
    at = node.clamp(0, N - 1)
    here = torch.where(drafted, s["lens"].long()[:, None] + s["depth"].long().gather(1, at), t)
    back = (s["lens"].long()[:, None] + s["depth"].long())[:, :, None] - here[:, None]   # [B][N][T]
    seen = _bits(s["mask"], N).gather(2, at[:, None].expand(-1, N, -1)) & drafted[:, None] | (node < 0)[:, None]
    if case["window"]:
        seen = seen & (back < case["window"])
    if s["slopes"] is not None:
        w -= s["slopes"].view(1, hkv, 1, G, 1) * back[:, None, :, None]
    w.masked_fill_(~seen[:, None, :, None], -math.inf)
    w = torch.exp(w.sub_(w.amax(-1, keepdim=True).clamp_(min=-3e38)))
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w.view(B, hkv, N * G, T), v).view(B, hkv, N, G, d) / torch.where(total > 0, total, 1.0)
    o = o.permute(0, 2, 1, 3, 4).reshape(B, N, hq, d)
    real = torch.arange(N, device="cuda") < s["new"].long()[:, None]
    out = s["out"].view(B, N, hq, d)
    out.copy_(torch.where(real[:, :, None, None], o, out))
    return out.view(B * N, hq, d)


def _plain_sample(s):
    """64 bits from the differences of the logits on: a draw next to a border does
    not depend on the order of the sums."""
    V = s["case"]["vocab"]
    temperature = s["temperature"].double()[:, None]
    greedy = temperature == 0
    best, order = torch.sort(s["logits"], dim=1, descending=True, stable=True)
    w = torch.exp((best.double() - best[:, :1].double()) / torch.where(greedy, 1.0, temperature))
    k = s["top_k"].long()[:, None]
    kept = torch.arange(V, device="cuda") < torch.where(k > 0, k, V)
    c = torch.cumsum(torch.where(kept, w, 0.0), 1)
    top_p = s["top_p"].double()[:, None]
    kept &= (c - w < top_p * c[:, -1:]) | (top_p >= 1)
    kept &= w >= s["min_p"].double()[:, None]
    w = torch.zeros_like(w).scatter_(1, order, torch.where(kept, w, 0.0))
    c = torch.cumsum(w, 1)
    token = (c <= s["u"].double()[:, None] * c[:, -1:]).sum(1, keepdim=True).clamp_(max=V - 1)
    token = torch.where(greedy, order[:, :1], token)
    prob = torch.where(greedy, 1.0, w.gather(1, token) / c[:, -1:])
    return dict(token=token[:, 0].int(), prob=prob[:, 0].float())


def _plain_commit(s):
    case = s["case"]
    B, N = case["B"], case["N"]
    tokens, parent, node = s["tokens"], s["parent"].long(), torch.arange(N, device="cuda")
    real = node < s["new"].long()[:, None]
    # a draft that the model picked, the first of its siblings with that token
    holds = (tokens == s["picked"].gather(1, parent.clamp(min=0))) & (parent >= 0) & real
    twin = (tokens[:, :, None] == tokens[:, None]) & (parent[:, :, None] == parent[:, None]) & (node[None, :] < node[:, None])
    holds &= ~(twin & real[:, None]).any(2)
    holds |= (node == 0) & real
    kept = (~_bits(s["mask"], N) | holds[:, None]).all(2) & (_bits(s["mask"], N)[:, :, 0]) & real
    count = kept.sum(1)
    path = torch.where(node < count[:, None], torch.argsort((~kept).int(), dim=1, stable=True), -1)
    last = path.gather(1, (count - 1).clamp(min=0)[:, None])
    token = s["picked"].gather(1, last.clamp(min=0))[:, 0]
    move = path >= 0
    src, dst = s["lens"].long()[:, None] + path, s["lens"].long()[:, None] + node
    table, kv = s["table"].long(), s["kv"]
    page = lambda t: table.gather(1, (t // PAGE).clamp(min=0))[move]  # noqa: E731
    kv[:, :, page(dst), :, (dst % PAGE)[move]] = kv[:, :, page(src), :, (src % PAGE)[move]]
    return dict(path=path.int(), count=count.int(), token=token, lens=(s["lens"] + count).int(), kv=kv.view(torch.int16))


def _plain_pages(s):
    table, ref, lens = s["table"], s["ref"], s["lens"]
    S, maxp = table.shape
    col = torch.arange(maxp, device="cuda")
    one = torch.ones((), dtype=torch.int32, device="cuda")
    # fork: the pages that hold a source's tokens, one more holder each
    src, dst = s["src"].long(), s["dst"].long()
    rows = torch.where(col < -(-lens[src].long() // PAGE)[:, None], table[src], -1)
    ref.index_put_((rows[rows >= 0].long(),), one, accumulate=True)
    table[dst] = rows
    lens[dst] = lens[src]
    # reserve: entries without a page, and a shared page that is partly filled
    # unless all its other holders have left it before
    first, end = lens.long() // PAGE, -(-(lens + s["need"]).long() // PAGE)
    take = (col >= first[:, None]) & (col < end[:, None]) & (table < 0)
    page = table.gather(1, first.clamp(max=maxp - 1)[:, None])[:, 0].long()
    shared = (lens % PAGE != 0) & (s["need"] > 0) & (ref[page] > 1)
    b = torch.arange(S, device="cuda")
    before = ((page[:, None] == page) & shared & (b < b[:, None])).sum(1)
    leave = shared & (before < ref[page] - 1)
    take |= leave[:, None] & (col == first[:, None])
    got = torch.nonzero(ref == 0)[:, 0][:int(take.sum())].int()
    old = page[leave]
    ref.index_put_((old,), -one, accumulate=True)
    table[take] = got
    ref[got.long()] = 1
    n = leave.sum()
    s["n_copies"].copy_(n.view(1))
    new = table.gather(1, first.clamp(max=maxp - 1)[:, None])[:, 0].long()[leave]
    s["copies"][:len(old)] = torch.stack([old, new], 1).int()
    # the copies, and what is not kept given back
    for p in s["planes"]:
        p[:, :, new] = p[:, :, old]
    gone = (col >= -(-s["keep"].long() // PAGE)[:, None]) & (table >= 0)
    ref.index_put_((table[gone].long(),), -one, accumulate=True)
    table.masked_fill_(gone, -1)
    return dict(table=table, ref=ref, lens=lens, copies=s["copies"], n_copies=s["n_copies"], lacking=s["lacking"], planes=s["planes"])


# ---- the calls ------------------------------------------------------------

def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        return dict(append=_plain_append, attn=_plain_attn, sample=_plain_sample, commit=_plain_commit, pages=_plain_pages)[kind](state)
    ctx = state["ctx"]
    if kind == "append":
        new = state["new"] if case["padded"] else None
        q = ctx.rope_kv_append_rows(state["x"], state["bias"], state["rope"], state["lens"], state["table"], state["caches"][0],
                                    case["N"], depth=state["depth"], n_new=new, q_out=state["out"])
        k, v = state["kv"][0]
        return dict(q=q, k=k, v=v)
    if kind == "attn":
        new = state["new"] if case["padded"] else None
        return ctx.gqa_tree_attn(state["q"], state["caches"][0], state["table"], state["lens"], case["N"], case["L"],
                                 mask=state["mask"], depth=state["depth"], n_nodes=new, opts=state["opts"], out=state["out"])
    if kind == "sample":
        token, prob = ctx.sample_filtered(state["logits"], state["u"], state["temperature"], state["top_k"], state["top_p"], state["min_p"])
        return dict(token=token, prob=prob)
    if kind == "commit":
        path, count, token, lens = ctx.tree_accept(state["tokens"], state["parent"], state["picked"], state["lens"])
        ctx.kv_keep(state["caches"], state["table"], state["lens"], path, count)
        return dict(path=path, count=count, token=token, lens=lens, kv=state["kv"].view(torch.int16))
    pool, table, lens = state["pool"], state["table"], state["lens"]
    ctx.pages_fork(pool, table, lens, state["src"], state["dst"])
    ctx.pages_reserve(pool, table, lens, state["need"], out=(state["copies"], state["n_copies"], state["lacking"]))
    ctx.pages_copy(state["set"], state["copies"], state["n_copies"])
    ctx.pages_free(pool, table, state["keep"])
    return dict(table=table, ref=state["ref"], lens=lens, copies=state["copies"], n_copies=state["n_copies"],
                lacking=state["lacking"], planes=state["planes"])


# ---- what a pass cannot do without ----------------------------------------

def work(case) -> dict:
    kind = case["kind"]
    if kind == "sample":
        # the logits once; a comparison, a difference and an exponential for each
        return dict(bytes=4 * case["m"] * case["vocab"], flops=3 * case["m"] * case["vocab"])
    hq, hkv, d, layers = HEADS[case["shape"]]
    if kind == "pages":
        # the last pages of half the sequences copied in all layers (one in 16 is
        # full), every entry of the table and every count
        S, held = case["S"], -(-0.75 * case["L"] // PAGE)
        page = 2 * layers * hkv * (PAGE * d * 2 if case["cache"] == "f16" else PAGE * d + 4)
        return dict(bytes=int(S / 2 * 15 / 16 * 2 * page + 8 * S * held + 4 * S * held), flops=0)
    B, N, L = case["B"], case["N"], case["L"]
    rows = B * ((N + 1) / 2 if case["padded"] else N)
    cached = (L // 8 + L) / 2 if case["ragged"] else L
    if kind == "append":
        return dict(bytes=int(rows * (4 * (hq + 2 * hkv) * d + 4 * hq * d + 4 * hkv * d + 4 * case["rot"])),
                    flops=int(rows * 6 * (hq + hkv) * case["rot"] / 2))
    if kind == "commit":
        # accepted rows behind the root that change their place, read and written
        moved = B * min((N - 1) / 2, max(0.0, 2 * (N - 1) / (case["span"] + 1) / 2 if case["span"] > 1 else 0.0))
        return dict(bytes=int(moved * 8 * hkv * d * layers + 16 * B * N), flops=0)
    seen = min(cached, case["window"] or cached)
    return dict(bytes=int(B * (min(cached, seen + N) + rows / B) * hkv * 4 * d + 8 * rows * hq * d),
                flops=int(4 * d * hq * rows * (seen + 1)))


# ---- the same in 64 bits --------------------------------------------------

def _exact_append(case, seed):
    s = _inputs(case, seed)
    hq, hkv, d, _ = HEADS[case["shape"]]
    B, N, rot = case["B"], case["N"], case["rot"]
    heads = (s["x"].double() + s["bias"].double()).view(B, N, -1, d)
    pos = (s["lens"][:, None] + s["depth"]).long()
    unit = torch.complex(s["cos"].double(), s["sin"].double())[pos][:, :, None]
    z = heads[:, :, :hq + hkv, :rot]
    lo, hi = (z[..., :rot // 2], z[..., rot // 2:]) if case["pairs"] == "half" else (z[..., 0::2], z[..., 1::2])
    w = torch.complex(lo.contiguous(), hi.contiguous()) * unit
    heads = heads.clone()
    heads[:, :, :hq + hkv, :rot] = torch.cat([w.real, w.imag], -1) if case["pairs"] == "half" else torch.view_as_real(w).flatten(-2)
    q = torch.zeros(B, N, hq, d, dtype=torch.float64, device="cuda")
    k, v = s["kv"][0].double()
    for b, (n, new) in enumerate(zip(s["lens"].tolist(), s["new"].tolist())):
        q[b, :new] = heads[b, :new, :hq]
        for j in range(new):
            page, slot = int(s["table"][b, (n + j) // PAGE]), (n + j) % PAGE
            k[page, :, slot] = heads[b, j, hq:hq + hkv]
            v[page, :, slot] = heads[b, j, hq + hkv:]
    return dict(q=q.view(B * N, hq, d), k=k, v=v)


def _exact_attn(case, seed):
    s = _inputs(case, seed)
    hq, hkv, d, _ = HEADS[case["shape"]]
    B, N = case["B"], case["N"]
    out = torch.zeros(B, N, hq, d, dtype=torch.float64, device="cuda")
    parent = s["parent"].tolist()
    for b, (n, new) in enumerate(zip(s["lens"].tolist(), s["new"].tolist())):
        pages = s["table"][b, :-(-(n + new) // PAGE)].long()
        k, v = (x[pages].double().permute(0, 2, 1, 3).reshape(-1, hkv, d)[:n + new] for x in s["kv"][0])
        # every node walks up to the root
        sees = torch.zeros(new, new, dtype=torch.bool)
        for j in range(new):
            i = j
            while i >= 0:
                sees[j, i] = True
                i = parent[b][i]
        depth = sees.sum(1).cuda() - 1
        at = n + depth
        where = torch.cat([torch.arange(n, device="cuda"), at])
        back = (at[:, None] - where).double()
        hidden = torch.cat([torch.zeros(new, n, dtype=torch.bool), ~sees], 1).cuda()
        if case["window"]:
            hidden = hidden | (back >= case["window"])
        for h in range(hq):
            g = h // (hq // hkv)
            z = s["q"].view(B, N, hq, d)[b, :new, h].double() @ k[:, g].T / math.sqrt(d)
            z = case["cap"] * torch.tanh(z / case["cap"]) if case["cap"] else z
            z = z - s["slopes"][h].double() * back if case["slopes"] else z
            out[b, :new, h] = torch.softmax(z.masked_fill(hidden, -math.inf), -1) @ v[:, g]
    return out.view(B * N, hq, d)


def _exact_sample(case, seed):
    s = _inputs(case, seed)
    prob = []
    for row, T, k, p, low, u in zip(s["logits"], *(s[n].tolist() for n in ("temperature", "top_k", "top_p", "min_p", "u"))):
        if T == 0:
            prob.append(torch.ones((), dtype=torch.float64, device="cuda"))
            continue
        z = row.double() / T
        w = torch.exp(z - z.max())
        order = torch.argsort(row, descending=True, stable=True)[:k or None]
        c = torch.cumsum(w[order], 0)
        if p < 1:
            order = order[:int(torch.searchsorted(c, p * c[-1:])) + 1]
        kept = torch.sort(order[w[order] >= low]).values
        c = torch.cumsum(w[kept], 0)
        i = torch.searchsorted(c, u * c[-1:], right=True).clamp(max=len(kept) - 1)
        prob.append(w[kept[i]][0] / c[-1])
    return dict(token=None, prob=torch.stack(prob))


def exact(case, seed):
    f = dict(append=_exact_append, attn=_exact_attn, sample=_exact_sample).get(case["kind"])
    return f(case, seed) if f else None
