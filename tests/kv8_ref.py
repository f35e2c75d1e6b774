"""The 8-bit KV cache and its attention stated once more in numpy float64, block
by block and row by row."""
import numpy as np

PAGE = 16


def half_up(x):
    """Nearest integer, halves away from zero."""
    return np.trunc(x + np.copysign(0.5, x))


def tables(max_pos, rot, theta=1e4):
    ang = np.arange(max_pos)[:, None] * theta ** (-2.0 * np.arange(rot // 2) / max(rot, 1))
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def rotate(x, c, s, interleaved):
    """x [..., d] float64 turned on its first 2 len(c) dimensions."""
    y, h = x.copy(), len(c)
    a, b = (x[..., 0:2 * h:2], x[..., 1:2 * h:2]) if interleaved else (x[..., :h], x[..., h:2 * h])
    u, v = a * c - b * s, b * c + a * s
    if interleaved:
        y[..., 0:2 * h:2], y[..., 1:2 * h:2] = u, v
    else:
        y[..., :h], y[..., h:2 * h] = u, v
    return y


class Cache:
    """k [pages][hkv][16][d], v [pages][hkv][d][16] int8; ks, vs [pages][hkv] float32."""

    def __init__(self, pages, hkv, d, rng=None):
        self.k, self.v = np.zeros((pages, hkv, PAGE, d), np.int8), np.zeros((pages, hkv, d, PAGE), np.int8)
        self.ks, self.vs = np.zeros((pages, hkv), np.float32), np.zeros((pages, hkv), np.float32)
        self.hkv, self.d = hkv, d
        if rng is not None:                      # quants of every value, scales over two decades
            self.k = rng.integers(-127, 128, self.k.shape, dtype=np.int8)
            self.v = rng.integers(-127, 128, self.v.shape, dtype=np.int8)
            self.ks = (10.0 ** rng.uniform(-3, -1, self.ks.shape)).astype(np.float32)
            self.vs = (10.0 ** rng.uniform(-3, -1, self.vs.shape)).astype(np.float32)

    def append_block(self, quants, scales, page, g, s0, new):
        """new [n][d] into slots s0 ..; quants as [16][d] views."""
        a = np.abs(new).max() if np.isfinite(new).all() else np.nan
        need = np.float32(0.0) if a < 2.0 ** -119 else np.float32(a / 127.0)
        old, grow = (scales[page, g] if s0 else np.float32(0.0)), 0
        if np.isnan(need) or not np.isfinite(old) or old < 0:
            scale = np.float32(np.nan)
        elif old > 0:
            scale = old
            while scale < need:
                scale, grow = np.float32(scale * np.float32(2.0)), grow + 1
        else:
            scale = need
        if grow:
            quants[:s0] = half_up(quants[:s0] / 2.0 ** grow).astype(np.int8)
        q = np.zeros(new.shape)
        if scale > 0 and not np.isnan(need):
            q = np.clip(half_up(new * (1.0 / np.float64(scale))), -127, 127)
        quants[s0:s0 + len(new)] = q.astype(np.int8)
        scales[page, g] = scale

    def append(self, x, bias, cos, sin, interleaved, seq_len, n_new, table, hq):
        """x [B][P][(hq + 2 hkv) d] float32; returns q [B][P][hq][d] float32 (zeros in padding rows)."""
        B, P = x.shape[:2]
        hkv, d, maxp = self.hkv, self.d, table.shape[1]
        heads = x.astype(np.float64).reshape(B, P, -1, d)
        if bias is not None:
            heads = heads + bias.astype(np.float64).reshape(-1, d)
        q_out = np.zeros((B, P, hq, d), np.float32)
        for b in range(B):
            sl = min(max(int(seq_len[b]), 0), maxp * PAGE)
            n = P if n_new is None else min(max(int(n_new[b]), 0), P)
            rows = heads[b, :n].copy()
            for j in range(n):
                p = min(sl + j, len(cos) - 1)
                rows[j, :hq + hkv] = rotate(rows[j, :hq + hkv], cos[p].astype(np.float64), sin[p].astype(np.float64),
                                            interleaved)
            q_out[b, :n] = rows[:, :hq].astype(np.float32)
            j = 0
            while j < n:
                t = sl + j
                take = min(PAGE - t % PAGE, n - j)
                page = table[b, t // PAGE] if t // PAGE < maxp else -1
                if 0 <= page < len(self.k):
                    for g in range(hkv):
                        self.append_block(self.k[page, g], self.ks, page, g, t % PAGE, rows[j:j + take, hq + g])
                        self.append_block(self.v[page, g].T, self.vs, page, g, t % PAGE, rows[j:j + take, hq + hkv + g])
                j += take
        return q_out

    def rows(self, table_row, n):
        """(K, V) [n][hkv][d] float64 of a sequence's first n tokens."""
        pages = np.clip(table_row[:-(-n // PAGE)], 0, len(self.k) - 1)
        k = self.k[pages].astype(np.float64) * self.ks[pages].astype(np.float64)[..., None, None]
        v = self.v[pages].astype(np.float64) * self.vs[pages].astype(np.float64)[..., None, None]
        k = k.transpose(0, 2, 1, 3).reshape(-1, self.hkv, self.d)[:n]
        return k, v.transpose(0, 3, 1, 2).reshape(-1, self.hkv, self.d)[:n]


def attend(cache, q, table, seq_len, max_len, n_new=None, prefill=True, scale=None, softcap=0.0, window=0, slopes=None):
    """q [B][P][hq][d]; returns (out, bound): float64 results (zeros in padding rows and
    for empty sequences) and how far binary32 results may be from them, element by element.

    The bound: an error e of the scores changes weights by the factor exp(+-e), so the
    result by at most 2 e max|v|.  e: q to half a step of max|q| / 4161536 in every
    product; eight binary32 roundings of the score, four of its cap (whose tanh is within
    4 units) and of its distance term (log2 e, joins and the differences to the maximum
    among them).  Weights: 22 bits and exp2 to one unit, 4 units in all; sums of n terms
    of one sign, and of n / 32 + 64 partial products twice over, in binary32."""
    B, P, hq, d = q.shape
    G, eps = hq // cache.hkv, 2.0 ** -24
    scale = 1.0 / np.sqrt(d) if scale is None else scale
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(B):
        for j in range(P if n_new is None else min(max(int(n_new[b]), 0), P)):
            L = min(max(int(seq_len[b]), 0) + j + (1 if prefill else 0), max_len)
            lo = max(0, L - window) if window else 0
            if L == 0:
                continue
            k, v = (x[lo:] for x in cache.rows(table[b], L))
            back = (L - 1 - np.arange(lo, L)).astype(np.float64)
            for h in range(hq):
                kk, vv, qq = k[:, h // G], v[:, h // G], q[b, j, h].astype(np.float64)
                s = raw = kk @ qq * scale
                s = softcap * np.tanh(s / softcap) if softcap else s
                far = slopes[h].astype(np.float64) * back if slopes is not None else 0.0 * back
                s = s - far
                w = np.exp(s - s.max())
                w /= w.sum()
                out[b, j, h] = w @ vv
                e = np.abs(qq).max() / (127 * 65536) * abs(scale) * np.abs(kk).sum(1) + eps * (
                    8 * np.abs(raw) + (8 * softcap if softcap else 0.0) + 4 * np.abs(far) + 4 * np.abs(s - s.max()))
                # each weight's share of the error; far tokens with no weight have none
                mean = (w * e).sum()
                n = L - lo
                sums = eps * (8 + 2 * (n / 32 + 64))
                top = np.abs(vv).max(0)
                bound[b, j, h] = (w * e) @ np.abs(vv) + mean * top + sums * (w @ np.abs(vv) + top * 2.0 ** -8) + eps * top
    return out, bound
