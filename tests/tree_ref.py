"""Plain statements of the calls for drafted tokens, sampling and pages, on the host:
numpy in 64 bits, loops in the order that the definitions name."""
import numpy as np

PAGE = 16


def random_trees(rng, B, N, span=4):
    """parent [B][N]: node 0 hangs from the cached tokens, now and then another does."""
    parent = np.full((B, N), -1, np.int32)
    for b in range(B):
        for j in range(1, N):
            parent[b, j] = -1 if rng.random() < 0.05 else rng.integers(max(0, j - span), j)
    return parent


def ancestors(parent):
    """Truth [N][N]: node j sees node i; and the depths."""
    N = len(parent)
    sees, depth = np.zeros((N, N), bool), np.zeros(N, np.int32)
    for j in range(N):
        p = parent[j] if 0 <= parent[j] < j else -1
        if p >= 0:
            sees[j], depth[j] = sees[p], depth[p] + 1
        sees[j, j] = True
    return sees, depth


def words(sees):
    """Truth [..., N] as 64-bit words [..., ceil(N / 64)] (int64)."""
    N = sees.shape[-1]
    pad = np.zeros((*sees.shape[:-1], -(-N // 64) * 64), np.uint8)
    pad[..., :N] = sees
    return np.ascontiguousarray(np.packbits(pad, axis=-1, bitorder="little")).view("<i8")


def accept(tokens, parent, picked, n):
    path = []
    cur = 0 if n > 0 else -1
    last = None
    while cur >= 0:
        path.append(cur)
        last = picked[cur]
        cur = next((j for j in range(cur + 1, n) if parent[j] == cur and tokens[j] == last), -1)
    return path, last


def keep_rows(cache, table, start, keep):
    """cache [pages][hkv][16][d], changed in place."""
    src = [cache[table[(start + i) // PAGE], :, (start + i) % PAGE].copy() for i in keep]
    for i, row in enumerate(src):
        cache[table[(start + i) // PAGE], :, (start + i) % PAGE] = row


def choose(l, u, T=1.0, k=0, p=1.0, mp=0.0):
    """(token, probability) by the definition; l binary32."""
    l = np.asarray(l, np.float32)
    real = ~np.isnan(l) & (l > -np.inf)
    if not real.any():
        return 0, 0.0
    order = np.argsort(-np.where(real, l + 0.0, -np.inf).astype(np.float64), kind="stable")[:real.sum()]
    if not T > 0:
        return int(order[0]), 1.0
    top = float(l[order[0]])
    with np.errstate(invalid="ignore"):
        w = np.where(l[order] == np.float32(top), 1.0, np.exp((l[order].astype(np.float64) - top) / float(T)))
    n = len(order) if k <= 0 else min(k, len(order))
    if p < 1:
        c = np.cumsum(w[:n])
        n = max(1, int((c - w[:n] < float(p) * c[-1]).sum()))
    if mp > 0:
        n = int((w[:n] >= min(float(mp), 1.0)).sum())
    kept = np.sort(order[:n])
    wk = np.zeros(len(l))
    wk[order] = w
    c = np.cumsum(wk[kept])
    u = u if u > 0 else 0.0
    i = min(int((c <= min(u, 1.0) * c[-1]).sum()), int(np.flatnonzero(wk[kept] > 0)[-1]))
    return int(kept[i]), wk[kept[i]] / c[-1]


def fork(ref, table, lens, src, dst):
    S = len(table)
    lens0, table0 = lens.copy(), table.copy()
    for i, (s, d) in enumerate(zip(src, dst)):
        if not (0 <= s < S and 0 <= d < S) or d in src or d in dst[:i]:
            continue
        for page in table[d]:
            if 0 <= page < len(ref):
                ref[page] -= 1
        held = -(-min(max(lens0[s], 0), PAGE * table.shape[1]) // PAGE)
        row = np.where(np.arange(table.shape[1]) < held, table0[s], -1)
        row[(row < 0) | (row >= len(ref))] = -1
        for page in row[row >= 0]:
            ref[page] += 1
        table[d] = row
        lens[d] = min(max(lens0[s], 0), PAGE * table.shape[1])


def reserve(ref, table, lens, need):
    """Served one after the other; (copies, lacking)."""
    r, t, copies, asked = ref.copy(), table.copy(), [], 0
    free = [i for i in range(len(ref)) if ref[i] == 0]
    maxp = table.shape[1]
    for b in range(len(table)):
        n, sl = max(int(need[b]), 0), min(max(int(lens[b]), 0), PAGE * maxp)
        if not n:
            continue
        first, end = sl // PAGE, min(-(-(sl + n) // PAGE), maxp)
        for e in range(first, end):
            page = t[b, e]
            ok = 0 <= page < len(ref)
            if ok and not (e == first and sl % PAGE and r[page] > 1):
                continue
            asked += 1
            if asked > len(free):
                if ok:
                    r[page] -= 1
                continue
            new = free[asked - 1]
            if ok:
                r[page] -= 1
                copies.append((int(page), new))
            t[b, e], r[new] = new, 1
    if asked > len(free):
        return [], asked - len(free)
    ref[:], table[:] = r, t
    return copies, 0


def free(ref, table, keep):
    for b in range(len(table)):
        for e in range(min(-(-max(int(keep[b]), 0) // PAGE), table.shape[1]), table.shape[1]):
            if 0 <= table[b, e] < len(ref):
                ref[table[b, e]] -= 1
            table[b, e] = -1
