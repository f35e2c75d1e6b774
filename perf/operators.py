"""The operators of the 8-bit KV cache as cases that can be timed and compared:
appending rotated keys and values to a paged int8 cache with a scale per page and
KV head, decode attention over it, and the causal attention of several new rows.
Shapes are those of the library's own configurations (the 0.5B-, 1.5B- and
7B-shaped models), and `draw` gives others of the same ranges.

`own` false: the plain form, elementary torch operations; true: the library's
calls.  `exact` states the definitions once more in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

# (query heads, KV heads, head dim) of the 0.5B-, 1.5B- and 7B-shaped models
HEADS = {"0.5b": (14, 2, 64), "1.5b": (12, 2, 128), "7b": (28, 4, 128)}
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


def _append(name, shape, B, P, L, rot, pairs="half", factor=1.0, ragged=True, padded=False):
    return dict(name=name, kind="append", shape=shape, B=B, P=P, L=L, rot=rot, pairs=pairs,
                factor=factor, ragged=ragged, padded=padded)


def _attn(name, shape, B, L, P=0, ragged=False, padded=False, cap=0.0, window=0, slopes=False):
    return dict(name=name, kind="prefill" if P else "decode", shape=shape, B=B, P=max(P, 1), L=L,
                ragged=ragged, padded=padded, cap=cap, window=window, slopes=slopes)


def listed() -> list:
    return [
        # one user's next token in the small model: nothing but latency
        _append("append-0.5b-b1-p1", "0.5b", 1, 1, 200, 64),
        # a full decode batch at the ragged positions that a server sees
        _append("append-7b-b64-p1", "7b", 64, 1, 4096, 128),
        # prompts of differing lengths in one padded chunk, half of each head
        # rotated in neighbouring pairs
        _append("append-1.5b-b16-p193", "1.5b", 16, 193, 700, 64, pairs="even", padded=True),
        # whole prompts of odd length, positions scaled for a longer context
        _append("append-7b-b8-p2047", "7b", 8, 2047, 0, 128, factor=4.0, ragged=False),
        # one user at the start of a conversation
        _attn("decode-0.5b-b1-l17", "0.5b", 1, 17),
        # one user far into a long context
        _attn("decode-7b-b1-l8191", "7b", 1, 8191),
        # a full batch with ragged lengths
        _attn("decode-7b-b64-l4096", "7b", 64, 4096, ragged=True),
        # long contexts, the largest cache
        _attn("decode-1.5b-b16-l32768", "1.5b", 16, 32768),
        # capped scores over a sliding window
        _attn("decode-0.5b-b32-l2048-cap", "0.5b", 32, 2048, ragged=True, cap=30.0, window=1000),
        # a few proposed tokens checked against a long context
        _attn("prefill-7b-b1-p5-l8000", "7b", 1, 8000, P=5),
        # padded chunks of short prompts with a bias that depends on distance
        _attn("prefill-0.5b-b6-p99-l500", "0.5b", 6, 500, P=99, ragged=True, padded=True, slopes=True),
        # the chunk of a prompt batch attending to what is cached
        _attn("prefill-7b-b8-p512-l4000", "7b", 8, 4000, P=512),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    """An integer of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["append", "append", "decode", "decode", "prefill"])
    shape = rng.choice(sorted(HEADS))
    hq, hkv, d = HEADS[shape]
    ragged, padded = rng.random() < 0.5, rng.random() < 0.4
    if kind == "append":
        B = _log_int(rng, 1, 64)
        P = 1 if rng.random() < 0.4 else _log_int(rng, 2, max(2, min(2047, 8 * 2047 // B)))
        case = _append("", shape, B, P, _log_int(rng, 1, 8192), rng.choice([d, d, d // 2, d // 4]),
                       rng.choice(["half", "even"]), rng.choice([1.0, 1.0, 2.0, 4.0]), ragged, padded and P > 1)
    else:
        more = dict(cap=rng.choice([0.0, 0.0, 20.0, 50.0]), slopes=rng.random() < 0.25,
                    window=rng.choice([0, 0, _log_int(rng, 1, 4096)]))
        if kind == "decode":
            B = _log_int(rng, 1, 64)
            case = _attn("", shape, B, min(_log_int(rng, 1, 32768), 16 * 32768 * 2 * 128 // (B * hkv * d)),
                         ragged=ragged, **more)
        else:
            # rows x heads x tokens up to that of the listed chunk
            B, P, top = _log_int(rng, 1, 16), _log_int(rng, 2, 512), 8 * 512 * 28 * 4000
            while B * P * P * hq > top:
                B, P = max(1, B // 2), max(2, P // 2)
            L = min(max(P, _log_int(rng, P, 8000)), top // (B * P * hq))
            case = _attn("", shape, B, L, P=P, ragged=ragged, padded=padded, **more)
    del case["name"]
    return case


# ---- inputs ---------------------------------------------------------------

def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _lens(case, seed):
    """Tokens of each sequence: for decode with the row's own, for the others
    those cached before the new rows; and the new rows of each sequence."""
    B, L, P = case["B"], case["L"], case["P"]
    cpu = torch.Generator().manual_seed(seed)
    top = L - P if case["kind"] == "prefill" else L
    n = torch.full((B,), top, dtype=torch.int32)
    if case["ragged"]:
        n = torch.randint(top // 16, top + 1, (B,), generator=cpu, dtype=torch.int32)
        if case["kind"] == "decode":
            n[0] = top
    new = torch.full((B,), P, dtype=torch.int32)
    if case["padded"]:
        new = torch.randint(1, P + 1, (B,), generator=cpu, dtype=torch.int32)
        new[0] = P
    return n, new


def _blocks(case) -> int:
    """Pages that P new rows of a sequence can touch."""
    return (case["P"] + PAGE - 2) // PAGE + 1


def _cache(case, g):
    """Pages of quantised normal keys and values with their scales, K token by
    token and V dimension by dimension, and the page table."""
    _, hkv, d = HEADS[case["shape"]]
    B = case["B"]
    maxp = -(-case["L"] // PAGE) if case["kind"] != "append" else case["L"] // PAGE + _blocks(case)
    quants, scales = [], []
    for rows in ((PAGE, d), (d, PAGE)):
        q = torch.empty(B * maxp, hkv, *rows, dtype=torch.int8, device="cuda")
        s = torch.empty(B * maxp, hkv, dtype=torch.float32, device="cuda")
        for lo in range(0, B * maxp, 8192):
            x = torch.randn(min(8192, B * maxp - lo), hkv, *rows, device="cuda", generator=g)
            s[lo:lo + 8192] = x.abs().amax((2, 3)) / 127
            q[lo:lo + 8192] = (x / s[lo:lo + 8192, :, None, None]).round_().to(torch.int8)
        quants.append(q)
        scales.append(s)
    table = torch.randperm(B * maxp, device="cuda", generator=g).to(torch.int32).view(B, maxp)
    return quants[0], quants[1], scales[0], scales[1], table


def _tables(case):
    """cos / sin of every position's angles, rounded once from 64 bits."""
    pos = torch.arange(case["L"] + case["P"] + 1, dtype=torch.float64, device="cuda") / case["factor"]
    i = torch.arange(case["rot"] // 2, dtype=torch.float64, device="cuda")
    ang = pos[:, None] * THETA ** (-2.0 * i / case["rot"])
    return ang.cos().float(), ang.sin().float()


def _slopes(hq: int):
    return torch.pow(2.0, -8.0 * torch.arange(1, hq + 1, device="cuda", dtype=torch.float64) / hq).float()


def _inputs(case, seed):
    hq, hkv, d = HEADS[case["shape"]]
    g = _gen(seed)
    n, new = _lens(case, seed)
    s = dict(case=case, lens=n.cuda(), new=new.cuda())
    s["kq"], s["vq"], s["ks"], s["vs"], s["table"] = _cache(case, g)
    rows = case["B"] * case["P"]
    if case["kind"] == "append":
        s["x"] = torch.randn(rows, (hq + 2 * hkv) * d, device="cuda", generator=g)
        s["bias"] = 0.02 * torch.randn((hq + 2 * hkv) * d, device="cuda", generator=g)
        s["cos"], s["sin"] = _tables(case)
        s["start"] = s["lens"] // PAGE * PAGE
    else:
        s["q"] = torch.randn(rows, hq, d, device="cuda", generator=g)
        s["slopes"] = _slopes(hq) if case["slopes"] else None
    return s


def prepare(case, seed):
    state = _inputs(case, seed)
    hq, _, d = HEADS[case["shape"]]
    # padding rows are left as they are: the buffer starts with zeros
    state["out"] = torch.zeros(case["B"] * case["P"], hq, d, device="cuda")
    if own:
        import logicaffeine_amd as lgx

        state["ctx"] = _context()
        state["kv"] = lgx.KvCacheI8(state["kq"], state["vq"], state["ks"], state["vs"])
        if case["kind"] == "append":
            state["rope"] = lgx.Rope(state["cos"], state["sin"], interleaved=case["pairs"] == "even")
        else:
            state["opts"] = lgx.AttnOpts(softcap=case["cap"], window=case["window"], slopes=state["slopes"])
    return state


# ---- the plain form -------------------------------------------------------

def _plain_append(s):
    """64 bits throughout: a quant next to a rounding border does not depend on
    the order of the operations."""
    case, table = s["case"], s["table"].long()
    hq, hkv, d = HEADS[case["shape"]]
    B, P, rot = case["B"], case["P"], case["rot"]
    x = (s["x"].double() + s["bias"].double()).view(B, P, hq + 2 * hkv, d)
    pos = s["lens"].long()[:, None] + torch.arange(P, device="cuda")
    c, sn = s["cos"].double()[pos][:, :, None], s["sin"].double()[pos][:, :, None]
    z = x[:, :, :hq + hkv, :rot]
    if case["pairs"] == "half":
        a, b = z[..., :rot // 2], z[..., rot // 2:]
        turned = torch.cat([a * c - b * sn, b * c + a * sn], -1)
    else:
        a, b = z[..., 0::2], z[..., 1::2]
        turned = torch.stack([a * c - b * sn, b * c + a * sn], -1).flatten(-2)
    qk = torch.cat([turned, x[:, :, :hq + hkv, rot:]], -1)
    real = torch.arange(P, device="cuda") < s["new"].long()[:, None]
    q = s["out"].view(B, P, hq, d)
    q.copy_(torch.where(real[:, :, None, None], qk[:, :, :hq].float(), q))
    # the touched pages of each sequence as [B][blocks][hkv][16][d]
    n = _blocks(case)
    first = s["lens"].long() // PAGE
    blk = first[:, None] + torch.arange(n, device="cuda")
    page = table.gather(1, blk)
    slot = blk[:, :, None] * PAGE + torch.arange(PAGE, device="cuda")     # token of each slot
    row = slot - s["lens"].long()[:, None, None]
    is_new = (row >= 0) & (row < s["new"].long()[:, None, None])
    held = (slot < s["lens"].long()[:, None, None])
    at = row.clamp(0, P - 1).view(B, -1)
    back = []
    for y, quants, scales, flip in ((qk[:, :, hq:], s["kq"], s["ks"], False), (x[:, :, hq + hkv:], s["vq"], s["vs"], True)):
        new = y.gather(1, at[:, :, None, None].expand(-1, -1, hkv, d)).view(B, n, PAGE, hkv, d).transpose(2, 3)
        mask = is_new[:, :, None, :, None]
        new = torch.where(mask, new, 0.0)
        need = (new.abs().amax((3, 4)) / 127).float()
        old_s = scales[page]
        some_old = held.any(-1)[:, :, None]
        steps = torch.ceil(torch.log2(need.double() / old_s.double())).clamp(min=0)
        # the logarithm only proposes the power: the scales decide
        grown = old_s.double() * torch.pow(2.0, steps)
        steps = torch.where(grown < need, steps + 1, torch.where((steps > 0) & (grown / 2 >= need), steps - 1, steps))
        keep = some_old & (old_s > 0)
        steps = torch.where(keep, steps, 0.0)
        scale = torch.where(keep, (old_s.double() * torch.pow(2.0, steps)).float(), need)
        touched = is_new.any(-1)[:, :, None]
        scale = torch.where(touched, scale, old_s)
        inv = torch.where(scale > 0, 1.0 / scale.double(), 0.0)[..., None, None]
        fresh = ((new.abs() * inv + 0.5).floor().clamp(max=127) * new.sign())
        old = quants[page].double()
        old = old.transpose(3, 4) if flip else old
        less = torch.pow(2.0, -torch.where(touched, steps, 0.0))[..., None, None]
        old_q = (old.abs() * less + 0.5).floor() * old.sign()
        old_q = torch.where(held[:, :, None, :, None], old_q, old)
        got = torch.where(mask, fresh, old_q)
        packed = (got.transpose(3, 4) if flip else got).to(torch.int8)
        quants[page.view(-1)] = packed.reshape(B * n, *packed.shape[2:])
        scales[page.view(-1)] = scale.view(B * n, hkv)
        values = got.float() * scale[..., None, None]
        back.append(values.transpose(2, 3).reshape(B, n * PAGE, hkv, d))
    return dict(q=q.view(B * P, hq, d), k=back[0], v=back[1])


def _plain_attn(s):
    case = s["case"]
    hq, hkv, d = HEADS[case["shape"]]
    B, P, G = case["B"], case["P"], hq // hkv
    T = s["table"].shape[1] * PAGE
    page = s["table"].long()
    k = (s["kq"][page].float() * s["ks"][page][..., None, None]).transpose(1, 2).reshape(B, hkv, T, d)
    v = (s["vq"][page].float() * s["vs"][page][..., None, None]).transpose(3, 4).transpose(1, 2).reshape(B, hkv, T, d)
    q = s["q"].view(B, P, hkv, G, d).transpose(1, 2).reshape(B, hkv, P * G, d)
    w = torch.matmul(q, k.transpose(2, 3).contiguous()).view(B, hkv, P, G, T)
    w *= 1.0 / math.sqrt(d)
    if case["cap"]:
        w = case["cap"] * torch.tanh(w / case["cap"])
    # position of row j of sequence b
    at = s["lens"].long()[:, None] + (torch.arange(P, device="cuda") if case["kind"] == "prefill" else -1)
    back = at[:, None, :, None, None] - torch.arange(T, device="cuda")
    if s["slopes"] is not None:
        w -= s["slopes"].view(1, hkv, 1, G, 1) * back
    seen = back >= 0
    if case["window"]:
        seen = seen & (back < case["window"])
    w.masked_fill_(~seen, -math.inf)
    top = w.amax(-1, keepdim=True).clamp_(min=-3e38)
    w = torch.exp(w.sub_(top))
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w.view(B, hkv, P * G, T), v).view(B, hkv, P, G, d) / torch.where(total > 0, total, 1.0)
    o = o.permute(0, 2, 1, 3, 4).reshape(B, P, hq, d)
    real = torch.arange(P, device="cuda") < s["new"].long()[:, None]
    out = s["out"].view(B, P, hq, d)
    out.copy_(torch.where(real[:, :, None, None], o, out))
    return out.view(B * P, hq, d)


# ---- the calls ------------------------------------------------------------

def run(state):
    case = state["case"]
    if not own:
        return _plain_append(state) if case["kind"] == "append" else _plain_attn(state)
    ctx, kv = state["ctx"], state["kv"]
    new = state["new"] if case["padded"] else None
    if case["kind"] == "append":
        q = ctx.rope_kv_append_i8(state["x"], state["bias"], state["rope"], state["lens"], state["table"], kv,
                                  case["P"], n_new=new, q_out=state["out"])
        k, v = ctx.kv_read_i8(kv, state["table"], state["start"], _blocks(case) * PAGE)
        return dict(q=q, k=k, v=v)
    if case["kind"] == "decode":
        return ctx.gqa_decode_attn_i8(state["q"], kv, state["table"], state["lens"], case["L"], opts=state["opts"],
                                      out=state["out"])
    return ctx.gqa_prefill_attn_i8(state["q"], kv, state["table"], state["lens"], case["P"], case["L"], n_new=new,
                                   opts=state["opts"], out=state["out"])


# ---- what a pass cannot do without ----------------------------------------

def work(case) -> dict:
    hq, hkv, d = HEADS[case["shape"]]
    B, P, L = case["B"], case["P"], case["L"]
    rows = B * ((P + 1) / 2 if case["padded"] else P)
    if case["kind"] == "append":
        # the rows in, the turned queries and the quants out; then the touched
        # pages of quants in and their values out
        read = B * _blocks(case) * PAGE * hkv * d
        return dict(bytes=int(rows * (4 * (hq + 2 * hkv) * d + 4 * hq * d + 2 * hkv * d + 4 * case["rot"]) + 10 * read),
                    flops=int(rows * (6 * (hq + hkv) * case["rot"] / 2 + 6 * hkv * d)))
    top = L - P if case["kind"] == "prefill" else L
    cached = (top // 16 + top) / 2 if case["ragged"] else top
    if case["kind"] == "decode":
        attended = tokens = min(cached, case["window"] or cached)
    else:
        new = rows / B
        tokens = cached + new
        attended = cached + (new + 1) / 2
        if case["window"]:
            attended, tokens = min(attended, case["window"]), min(tokens, case["window"] + new)
    return dict(bytes=int(B * tokens * hkv * (2 * d + 0.5) + 8 * rows * hq * d), flops=int(4 * d * hq * rows * attended))


# ---- the same in 64 bits --------------------------------------------------

def _half_up(x):
    """Nearest whole number, halves away from zero."""
    return torch.trunc(x + torch.copysign(torch.full_like(x, 0.5), x))


def _exact_append(case, seed):
    s = _inputs(case, seed)
    hq, hkv, d = HEADS[case["shape"]]
    B, P, rot, n = case["B"], case["P"], case["rot"], _blocks(case)
    heads = (s["x"].double() + s["bias"].double()).view(B * P, -1, d).clone()
    lens, new = s["lens"].tolist(), s["new"].tolist()
    pos = torch.tensor([m + j for m in lens for j in range(P)], device="cuda")
    unit = torch.complex(s["cos"].double(), s["sin"].double())[pos][:, None]
    z = heads[:, :hq + hkv, :rot]
    lo, hi = (z[..., :rot // 2], z[..., rot // 2:]) if case["pairs"] == "half" else (z[..., 0::2], z[..., 1::2])
    w = torch.complex(lo.contiguous(), hi.contiguous()) * unit
    heads[:, :hq + hkv, :rot] = torch.cat([w.real, w.imag], -1) if case["pairs"] == "half" else torch.view_as_real(w).flatten(-2)
    heads = heads.view(B, P, -1, d)
    q = torch.zeros(B, P, hq, d, dtype=torch.float64, device="cuda")
    out = torch.empty(2, B, n * PAGE, hkv, d, dtype=torch.float64, device="cuda")
    for b in range(B):
        q[b, :new[b]] = heads[b, :new[b], :hq]
        for i in range(n):
            at = (lens[b] // PAGE + i) * PAGE
            page = int(s["table"][b, at // PAGE])
            lo, hi = max(at, lens[b]), min(at + PAGE, lens[b] + new[b])
            for which, (quants, scales) in enumerate(((s["kq"], s["ks"]), (s["vq"], s["vs"]))):
                block = quants[page].double()                            # [hkv][16][d]
                block = block.transpose(1, 2).clone() if which else block
                step = scales[page].double()
                if hi > lo:
                    y = heads[b, lo - lens[b]:hi - lens[b], hq + which * hkv:hq + (which + 1) * hkv].transpose(0, 1)
                    need = (y.abs().amax((1, 2)) / 127).float().double()
                    if lo > at:
                        first = step.clone()
                        for _ in range(300):
                            step = torch.where((step < need) & (step > 0), step * 2, step)
                        old = _half_up(block[:, :lo - at] * (first / step)[:, None, None])
                        block[:, :lo - at] = torch.where((step > 0)[:, None, None], old, block[:, :lo - at])
                        step = torch.where(step > 0, step, need)
                    else:
                        step = need
                    block[:, lo - at:hi - at] = _half_up(y / torch.where(step > 0, step, 1.0)[:, None, None]).clamp(-127, 127)
                out[which, b, i * PAGE:(i + 1) * PAGE] = (block * step[:, None, None]).transpose(0, 1)
    return dict(q=q.view(B * P, hq, d), k=out[0], v=out[1])


def _exact_attn(case, seed):
    s = _inputs(case, seed)
    hq, hkv, d = HEADS[case["shape"]]
    B, P = case["B"], case["P"]
    out = torch.zeros(B, P, hq, d, dtype=torch.float64, device="cuda")
    decode = case["kind"] == "decode"
    for b, (n, new) in enumerate(zip(s["lens"].tolist(), s["new"].tolist())):
        T = n if decode else n + new
        if T == 0:
            continue
        pages = s["table"][b, :-(-T // PAGE)].long()
        # token by token: [T][hkv][d]
        k = (s["kq"][pages].double() * s["ks"][pages].double()[..., None, None]).permute(0, 2, 1, 3).reshape(-1, hkv, d)[:T]
        v = (s["vq"][pages].double() * s["vs"][pages].double()[..., None, None]).permute(0, 3, 1, 2).reshape(-1, hkv, d)[:T]
        at = torch.arange(n, n + new, device="cuda") if not decode else torch.tensor([n - 1], device="cuda")
        back = (at[:, None] - torch.arange(T, device="cuda")).double()
        for h in range(hq):
            g = h // (hq // hkv)
            q = s["q"].view(B, P, hq, d)[b, :len(at), h].double()
            z = q @ k[:, g].T / math.sqrt(d)
            z = case["cap"] * torch.tanh(z / case["cap"]) if case["cap"] else z
            z = z - s["slopes"][h].double() * back if case["slopes"] else z
            hidden = (back < 0) | (back >= case["window"]) if case["window"] else back < 0
            out[b, :len(at), h] = torch.softmax(z.masked_fill(hidden, -math.inf), -1) @ v[:, g]
    return out.view(B * P, hq, d)


def exact(case, seed):
    return _exact_append(case, seed) if case["kind"] == "append" else _exact_attn(case, seed)
