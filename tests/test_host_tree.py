"""The host side of drafts, sampling with per-row settings and a cache's pages without
a device: what the calls refuse, and the grids and workspaces of those they take (on the
recording stand-in for the HIP runtime, tests/hip_stub.cpp)."""
import ctypes as C
import json
import os
import re
import subprocess
import sys

import pytest

import logicaffeine_amd as lgx

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = r"""
import ctypes as C, json, sys
stub = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
stub.stub_log.restype = C.c_char_p
import logicaffeine_amd as lgx
L = lgx.lib()
kinds = {"kv": lgx.KvF16C, "rope": lgx.RopeC, "opts": lgx.AttnOptsC, "pool": lgx.PagePoolC, "plane": lgx.PagePlaneC}
for line in sys.stdin:
    name, args = json.loads(line)
    h = C.c_void_p()                       # a context of its own: each call's workspace shows
    lgx._check(L.lgx_ctx_create(0, b"stub", C.byref(h)))
    keep = [(kinds[a[0]] * (len(a) - 1))(*[kinds[a[0]](*s) for s in a[1:]]) if isinstance(a, list) else a for a in args]
    stub.stub_reset()
    st = getattr(L, name)(h, *keep)
    print(json.dumps([lgx.STATUS_NAMES.get(st, st), stub.stub_log().decode().splitlines()]), flush=True)
"""
P, Q = 1 << 41, 1 << 42
NULL, INVALID, UNSUPPORTED, OUT = "LGX_NULL_POINTER", "LGX_INVALID_ARGUMENT", "LGX_UNSUPPORTED", "LGX_OUT_OF_BOUNDS"


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("stub") / "hip_stub.so")
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    subprocess.run(["g++", "-O1", "-fPIC", "-shared", "-std=c++17", f"-I{rocm}/include", "-o", so,
                    os.path.join(ROOT, "tests", "hip_stub.cpp")], check=True)

    def run(calls):
        r = subprocess.run([sys.executable, "-c", CHILD, so], cwd=ROOT, text=True, capture_output=True, timeout=300,
                           input="".join(json.dumps(c) + "\n" for c in calls))
        assert r.returncode == 0, r.stderr[-4000:]
        out = []
        for line in r.stdout.splitlines():
            st, log = json.loads(line)
            words = [ln.split() for ln in log]
            out.append((st, [(w[0], *map(int, w[1:])) for w in words if w[0] != "malloc"],
                        sum(int(w[1]) for w in words if w[0] == "malloc")))
        assert len(out) == len(calls)
        return out

    return run


def shape(pages=100, hkv=2, d=64, k=P, v=P):
    return [k, v, pages, hkv, d]


def kv(**a):
    return ["kv", shape(**a)]


def attn(B=2, N=5, hq=14, maxp=10, top=155, cache=0, opts=None, q=P, out=Q, table=P, lens=P, n=None, depth=None, mask=None):
    return ["lgx_gqa_tree_attn", [q, kv() if cache == 0 else cache, table, lens, n, depth, mask, B, N, hq, maxp, top, opts, out,
                                  None]]


def append(B=2, N=5, hq=14, maxp=10, cache=0, rope=0, x=P, q=Q, lens=P, table=P):
    return ["lgx_rope_kv_append_rows", [x, None, ["rope", [P, P, 64, 0, 100]] if rope == 0 else rope, lens, None, None, table,
                                        kv() if cache == 0 else cache, q, B, N, hq, maxp, None]]


def plan(B=2, N=5, parent=P, depth=P, mask=P):
    return ["lgx_tree_plan", [parent, None, B, N, depth, mask, None]]


def accept(B=2, N=5, tokens=P, parent=P, picked=P, lens=P, path=P, count=P, nxt=P, new=P):
    return ["lgx_tree_accept", [tokens, parent, picked, None, lens, B, N, path, count, nxt, new, None]]


def keep(B=2, N=5, maxp=10, caches=0, layers=None, table=P, start=P, rows=P, n=P):
    caches = kv() if caches == 0 else caches
    return ["lgx_kv_keep", [caches, (len(caches) - 1 if caches else 1) if layers is None else layers, table, start, rows, n, B, N,
                            maxp, None]]


def sample(m=3, vocab=1000, ld=None, logits=P, T=None, k=None, p=None, mp=None, u=P, out=P, prob=None):
    return ["lgx_sample_filtered", [logits, vocab if ld is None else ld, m, vocab, T, k, p, mp, u, out, prob, None]]


POOL = ["pool", [P, 100]]


def fork(S=5, n=2, maxp=10, pool=POOL, table=P, lens=P, src=P, dst=P):
    return ["lgx_pages_fork", [pool, table, lens, src, dst, S, n, maxp, None]]


def reserve(B=5, maxp=10, pool=POOL, table=P, lens=P, need=P, copies=P, n=P, lacking=P):
    return ["lgx_pages_reserve", [pool, table, lens, need, B, maxp, copies, n, lacking, None]]


def copy(planes=0, n_planes=None, pages=100, copies=P, n=P, most=5):
    planes = ["plane", [P, 4096]] if planes == 0 else planes
    return ["lgx_pages_copy", [planes, (len(planes) - 1 if planes else 1) if n_planes is None else n_planes, pages, copies, n, most,
                               None]]


def free(B=5, maxp=10, pool=POOL, table=P, rows=P):
    return ["lgx_pages_free", [pool, table, rows, B, maxp, None]]


REFUSED = [
    *[(attn(**{a: None}), NULL) for a in ("q", "out", "table", "lens", "cache")],
    (attn(cache=kv(k=None)), NULL), (attn(cache=kv(v=None)), NULL), (attn(cache=kv(v=P + 8)), INVALID),
    (attn(cache=kv(d=96)), UNSUPPORTED), (attn(cache=kv(d=256)), UNSUPPORTED), (attn(cache=kv(pages=0)), INVALID),
    (attn(cache=kv(hkv=0)), INVALID), (attn(q=P + 4), INVALID), (attn(out=P + 8), INVALID), (attn(B=0), INVALID),
    (attn(N=0), INVALID), (attn(N=257, top=0, maxp=100), INVALID), (attn(hq=13), INVALID), (attn(hq=0), INVALID),
    (attn(hq=34), UNSUPPORTED), (attn(top=-1), OUT), (attn(top=156), OUT), (attn(maxp=0), INVALID),
    (attn(maxp=(1 << 26) + 1, top=1), INVALID), (attn(B=1 << 24), OUT), (attn(out=P), INVALID),
    (attn(out=P + 4 * 2 * 5 * 14 * 64 - 16), INVALID), (attn(out=Q, q=Q + 16), INVALID),
    *[(attn(opts=["opts", o]), INVALID) for o in ([0.0, -1.0, 0, None], [0.0, float("inf"), 0, None], [0.0, 1e-38, 0, None],
                                                  [float("nan"), 0.0, 0, None], [0.0, 0.0, -1, None])],
    *[(append(**{a: None}), NULL) for a in ("x", "q", "lens", "table", "cache", "rope")],
    (append(rope=["rope", [None, P, 64, 0, 100]]), NULL), (append(rope=["rope", [P, P, 66, 0, 100]]), INVALID),
    (append(rope=["rope", [P, P, 7, 0, 100]]), INVALID), (append(rope=["rope", [P, P, -2, 0, 100]]), INVALID),
    (append(rope=["rope", [P, P, 64, 2, 100]]), INVALID), (append(rope=["rope", [P, P, 64, 0, 0]]), INVALID),
    (append(B=0), INVALID), (append(N=0), INVALID), (append(hq=0), INVALID), (append(hq=15), INVALID),
    (append(cache=kv(d=32)), UNSUPPORTED), (append(cache=kv(k=P + 2)), INVALID), (append(B=1 << 20, N=1 << 12), OUT),
    (append(B=1 << 15, N=1 << 15), OUT), (append(q=P), INVALID), (append(q=P + 4 * 2 * 5 * 18 * 64 - 16), INVALID),
    *[(plan(**{a: None}), NULL) for a in ("parent", "depth", "mask")], (plan(B=0), INVALID), (plan(N=0), INVALID),
    (plan(N=257), INVALID), (plan(B=(1 << 23) + 1), OUT),
    *[(accept(**{a: None}), NULL) for a in ("tokens", "parent", "picked", "path", "count", "nxt", "lens")],
    (accept(N=257), INVALID), (accept(B=0), INVALID), (accept(B=(1 << 25) + 1), OUT),
    *[(keep(**{a: None}), NULL) for a in ("table", "start", "rows", "n", "caches")],
    (keep(layers=0), INVALID), (keep(B=0), INVALID), (keep(N=0), INVALID), (keep(maxp=0), INVALID),
    (keep(caches=["kv", shape(), shape(pages=99)]), INVALID), (keep(caches=["kv", shape(), shape(d=128)]), INVALID),
    (keep(caches=["kv", shape(), shape(v=None)]), NULL), (keep(caches=kv(hkv=4 * 65535 + 1)), OUT),
    *[(sample(**{a: None}), NULL) for a in ("logits", "u", "out")], (sample(m=0), INVALID), (sample(m=65536), INVALID),
    (sample(vocab=0), UNSUPPORTED), (sample(vocab=(1 << 19) + 1), UNSUPPORTED), (sample(ld=999), INVALID),
    (sample(ld=1 << 60), INVALID),
    *[(fork(**{a: None}), NULL) for a in ("pool", "table", "lens", "src", "dst")], (fork(pool=["pool", [None, 100]]), NULL),
    (fork(pool=["pool", [P, 0]]), INVALID), (fork(S=0), INVALID), (fork(n=0), INVALID), (fork(n=1025), INVALID),
    (fork(maxp=0), INVALID), (fork(maxp=1 << 24), INVALID),
    *[(reserve(**{a: None}), NULL) for a in ("pool", "table", "lens", "need", "copies", "n", "lacking")],
    (reserve(B=0), INVALID), (reserve(B=1025), INVALID), (reserve(maxp=0), INVALID), (reserve(B=32, maxp=1 << 26), OUT),
    (reserve(B=1024, maxp=(1 << 21)), OUT),
    *[(copy(**{a: None}), NULL) for a in ("planes", "copies", "n")], (copy(planes=["plane", [P, 64], [None, 64]]), NULL),
    (copy(planes=["plane", [P, 0]]), INVALID), (copy(planes=["plane", [P, 1 << 62]]), INVALID), (copy(n_planes=0), INVALID),
    (copy(pages=0), INVALID), (copy(most=0), INVALID),
    *[(free(**{a: None}), NULL) for a in ("pool", "table", "rows")], (free(B=0), INVALID), (free(maxp=1 << 24), INVALID),
]


def test_refusals_launch_nothing(host):
    for (call, want), (st, launches, alloc) in zip(REFUSED, host([c for c, _ in REFUSED])):
        assert (st, launches, alloc) == (want, [], 0), call


@pytest.mark.parametrize("B,N,hq,hkv,d,top,opts", [
    (1, 1, 14, 2, 64, 0, None), (1, 6, 14, 2, 64, 200, None), (1, 64, 28, 4, 128, 8000, None), (32, 16, 28, 4, 128, 4096, None),
    (9, 201, 12, 2, 128, 1500, [0.0, 25.0, 0, None]), (64, 1, 28, 4, 128, 4096, [0.0, 0.0, 100, None]),
    (300, 2, 8, 8, 64, 2000, None), (1, 256, 16, 1, 64, 1 << 24, None), (2, 3, 2, 2, 128, 1 << 29, None),
    (255, 1, 1, 1, 64, 5000, [-1.0, 0.0, 0, None]), (1, 1, 4, 4, 64, 50000, [0.0, 0.0, 0, P]), (4000, 17, 16, 1, 128, 100, None)])
def test_attention_covers_every_column(host, B, N, hq, hkv, d, top, opts):
    """A workgroup for every 64 columns of every KV head at least, and where tiles are
    split among more, room for every workgroup's partial results."""
    (st, launches, alloc), = host([attn(B, N, hq, -(-(top + N) // 16), top, kv(pages=1000, hkv=hkv, d=d),
                                        ["opts", opts] if opts else None)])
    assert st == "LGX_OK"
    name, gx, gy, gz, block = launches[0]
    assert (name, gy, gz, block) == (f"lgx_k_tree_attn{'x' if opts else ''}_d{d}", 1, 1, 256) and gx % 8 == 0
    blocks = B * -(-N * (hq // hkv) // 64) * hkv
    if len(launches) == 1:
        assert blocks <= gx < blocks + 8 and alloc == 0
    else:
        assert gx >= blocks and B <= 256
        per = 1024 // d if "joinr" in launches[1][0] else 1
        assert launches[1][0] in (f"lgx_k_tree_join_d{d}", f"lgx_k_tree_joinr_d{d}") and len(launches) == 2
        assert launches[1][1] * per >= B * N * hq > (launches[1][1] - 1) * per
        assert alloc >= (gx - 7) // hkv * hkv * 64 * (d + 2) * 4 + blocks // hkv * 8


def test_short_calls_are_one_launch(host):
    for st, launches, alloc in host([attn(1, 6, 14, 20, 200), attn(64, 1, 14, 20, 250), append(), plan(), accept(new=None, lens=None),
                                     keep(), fork(), free(), copy()]):
        assert (st, len(launches), alloc) == ("LGX_OK", 1, 0)


@pytest.mark.parametrize("B,N,hq,hkv,d", [(1, 1, 14, 2, 64), (3, 7, 28, 4, 128), (64, 33, 28, 4, 128), (1, 100000, 1, 1, 64)])
def test_append_covers_every_head(host, B, N, hq, hkv, d):
    (st, launches, _), (st0, l0, _) = host([append(B, N, hq, cache=kv(hkv=hkv, d=d)),
                                            append(B, N, hq, cache=kv(hkv=hkv, d=d), rope=["rope", [None, None, 0, 0, 1]])])
    heads, per = B * N * (hq + 2 * hkv), 2048 // d
    assert st == st0 == "LGX_OK" and launches == l0 == [(f"lgx_k_append_rows_d{d}", -(-heads // per), 1, 1, 256)]


@pytest.mark.parametrize("layers,parts", [(1, [1]), (28, [28]), (64, [64]), (65, [64, 1]), (200, [64, 64, 64, 8])])
def test_keep_and_copy_go_over_every_layer(host, layers, parts):
    (st, launches, _), (st2, copies, _) = host([keep(B=3, caches=["kv", *[shape(hkv=9)] * layers]),
                                                copy(["plane", *[[P, 96]] * (2 * layers)], most=7)])
    assert st == st2 == "LGX_OK"
    assert launches == [("lgx_k_kv_keep_d64", 3, 2 * n, 3, 256) for n in parts]
    assert copies == [("lgx_k_pages_copy", 7, 2 * n, 1, 256) for n in parts]


@pytest.mark.parametrize("m,vocab,p,mp", [(1, 1, None, None), (1, 151936, P, None), (512, 152064, P, P), (3, 4097, None, P), (3, 4096, P, P),
                                          (65535, 64, P, None), (65535, 1 << 19, None, None), (7, 1 << 19, P, P)])
def test_sampling_workspace(host, m, vocab, p, mp):
    """Slices' sums and maxima, chunks' maxima, the list of wide rows and the bins of
    as many as 64 MiB hold, one at least."""
    (st, launches, alloc), = host([sample(m, vocab, p=p, mp=mp, ld=vocab + 3)])
    assert st == "LGX_OK"
    ns = -(-vocab // 4096)
    names = ["lgx_k_filter_scan", "lgx_k_filter_pick"] + ["lgx_k_filter_wide"] * bool((p or mp) and vocab > 4096)
    assert [x[0] for x in launches] == names and launches[0][1:3] == (ns, m) and launches[1][1] == m
    slot = ns * 256 * 8
    slots = min(m, max((64 << 20) // slot, 1)) if (p or mp) and vocab > 4096 else 0
    assert alloc >= m * ns * (8 + 4 + 64 * 4) + m * (8 + 4 + 4) + 4 + slots * (slot + 4)


def test_reserve_lists_no_more_pages_than_there_are(host):
    for pages, B, maxp in ((100, 5, 10), (1, 1024, 10), (10**6, 3, 7), (2**31 - 1, 1, 1 << 26)):
        (st, launches, alloc), = host([reserve(B, maxp, ["pool", [P, pages]])])
        assert st == "LGX_OK" and launches == [("lgx_k_pages_reserve", 1, 1, 1, 1024)]
        assert alloc >= 4 * min(pages, B * (maxp + 1))


def test_structs_match_the_header():
    """The ctypes mirrors have the header's fields in its order."""
    src = open(os.path.join(ROOT, "include", "lgx.h")).read()
    for name, mirror in (("lgx_kv_f16", lgx.KvF16C), ("lgx_page_pool", lgx.PagePoolC), ("lgx_page_plane", lgx.PagePlaneC)):
        body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct %s \{(.*?)\}" % name, src, re.S).group(1), flags=re.S)
        fields = [f for decl in body.split(";") for f in re.findall(r"(\w+)\s*(?:,|$)", decl.strip())]
        assert fields == [f for f, _ in mirror._fields_], name
