"""The host side of the 8-bit KV cache without a device: rotary tables, what the calls
refuse, and the grids and workspaces of those they take (on the recording stand-in for
the HIP runtime, tests/hip_stub.cpp)."""
import ctypes as C
import json
import os
import subprocess
import sys

import numpy as np
import pytest

import logicaffeine_amd as lgx

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = r"""
import ctypes as C, json, sys
stub = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
stub.stub_log.restype = C.c_char_p
import logicaffeine_amd as lgx
L = lgx.lib()
for line in sys.stdin:
    name, args = json.loads(line)
    h = C.c_void_p()                       # a context of its own: each call's workspace shows
    lgx._check(L.lgx_ctx_create(0, b"stub", C.byref(h)))
    kinds = {"kv": lgx.KvI8C, "rope": lgx.RopeC, "opts": lgx.AttnOptsC}
    keep = [kinds[a[0]](*a[1]) if isinstance(a, list) else a for a in args]
    stub.stub_reset()
    st = getattr(L, name)(h, *[C.byref(a) if isinstance(a, C.Structure) else a for a in keep])
    print(json.dumps([lgx.STATUS_NAMES.get(st, st), stub.stub_log().decode().splitlines()]), flush=True)
"""
P = 1 << 41


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


def kv(pages=100, hkv=2, d=64, k=P, v=P, ks=P, vs=P):
    return ["kv", [k, v, ks, vs, pages, hkv, d]]


def decode(B=2, hq=14, maxp=10, top=160, cache=None, opts=None, q=P, out=P, table=P, lens=P):
    return ["lgx_gqa_decode_attn_i8", [q, cache or kv(), table, lens, B, hq, maxp, top, opts, out, None]]


def prefill(B=2, rows=5, hq=14, maxp=10, top=160, cache=None, opts=None, new=None, q=P, out=P):
    return ["lgx_gqa_prefill_attn_i8", [q, cache or kv(), P, P, new, B, rows, hq, maxp, top, opts, out, None]]


def append(B=2, rows=5, hq=14, maxp=10, cache=None, rope=None, x=P, q=P, lens=P):
    return ["lgx_rope_kv_append_i8", [x, None, rope or ["rope", [P, P, 64, 0, 100]], lens, None, P, cache or kv(), q, B, rows,
                                      hq, maxp, None]]


def read(B=2, n=5, maxp=10, cache=None, out=P):
    return ["lgx_kv_read_i8", [cache or kv(), P, P, B, n, maxp, out, P, None]]


REFUSED = [
    (decode(q=None), "LGX_NULL_POINTER"), (decode(out=None), "LGX_NULL_POINTER"), (decode(table=None), "LGX_NULL_POINTER"),
    (decode(lens=None), "LGX_NULL_POINTER"), (decode(cache=kv(k=None)), "LGX_NULL_POINTER"),
    (decode(cache=kv(vs=None)), "LGX_NULL_POINTER"), (decode(cache=kv(d=96)), "LGX_UNSUPPORTED"),
    (decode(cache=kv(d=256)), "LGX_UNSUPPORTED"), (decode(cache=kv(pages=0)), "LGX_INVALID_ARGUMENT"),
    (decode(cache=kv(k=P + 8)), "LGX_INVALID_ARGUMENT"), (decode(q=P + 4), "LGX_INVALID_ARGUMENT"),
    (decode(out=P + 8), "LGX_INVALID_ARGUMENT"), (decode(B=0), "LGX_INVALID_ARGUMENT"), (decode(hq=13), "LGX_INVALID_ARGUMENT"),
    (decode(hq=34), "LGX_UNSUPPORTED"), (decode(top=0), "LGX_OUT_OF_BOUNDS"), (decode(top=161), "LGX_OUT_OF_BOUNDS"),
    (decode(maxp=1 << 27, top=1), "LGX_INVALID_ARGUMENT"), (decode(maxp=0), "LGX_INVALID_ARGUMENT"),
    (decode(opts=["opts", [0.0, -1.0, 0, None]]), "LGX_INVALID_ARGUMENT"),
    (decode(opts=["opts", [0.0, float("inf"), 0, None]]), "LGX_INVALID_ARGUMENT"),
    (decode(opts=["opts", [0.0, 1e-38, 0, None]]), "LGX_INVALID_ARGUMENT"),
    (decode(opts=["opts", [float("nan"), 0.0, 0, None]]), "LGX_INVALID_ARGUMENT"),
    (decode(opts=["opts", [0.0, 0.0, -1, None]]), "LGX_INVALID_ARGUMENT"),
    (prefill(rows=0), "LGX_INVALID_ARGUMENT"), (prefill(B=1 << 16, rows=1 << 15), "LGX_OUT_OF_BOUNDS"),
    (append(B=-1), "LGX_INVALID_ARGUMENT"), (append(rows=0), "LGX_INVALID_ARGUMENT"), (append(hq=0), "LGX_INVALID_ARGUMENT"),
    (append(x=None), "LGX_NULL_POINTER"), (append(lens=None), "LGX_NULL_POINTER"), (append(q=P + 4), "LGX_INVALID_ARGUMENT"),
    (append(rope=["rope", [None, P, 64, 0, 100]]), "LGX_NULL_POINTER"),
    (append(rope=["rope", [P, P, 66, 0, 100]]), "LGX_INVALID_ARGUMENT"),
    (append(rope=["rope", [P, P, 7, 0, 100]]), "LGX_INVALID_ARGUMENT"),
    (append(rope=["rope", [P, P, -2, 0, 100]]), "LGX_INVALID_ARGUMENT"),
    (append(rope=["rope", [P, P, 64, 2, 100]]), "LGX_INVALID_ARGUMENT"),
    (append(rope=["rope", [P, P, 64, 0, 0]]), "LGX_INVALID_ARGUMENT"),
    (append(B=1 << 20, rows=1 << 20), "LGX_OUT_OF_BOUNDS"), (append(hq=1 << 17), "LGX_OUT_OF_BOUNDS"),
    (read(n=0), "LGX_INVALID_ARGUMENT"), (read(out=None), "LGX_NULL_POINTER"), (read(out=P + 4), "LGX_INVALID_ARGUMENT"),
    (read(B=1 << 20, n=1 << 20), "LGX_OUT_OF_BOUNDS"), (read(cache=kv(hkv=70000)), "LGX_OUT_OF_BOUNDS"),
]


def test_refusals_launch_nothing(host):
    for (call, want), (st, launches, alloc) in zip(REFUSED, host([c for c, _ in REFUSED])):
        assert (st, launches, alloc) == (want, [], 0), call


def test_no_rotation_needs_no_tables(host):
    (st, launches, _), = host([append(rope=["rope", [None, None, 0, 0, 1]])])
    assert st == "LGX_OK" and len(launches) == 1


@pytest.mark.parametrize("B,rows,hq,hkv,d,top,cols", [
    (64, 1, 28, 4, 128, 4096, 16), (1, 9, 28, 4, 128, 1000, 16), (8, 16, 28, 4, 128, 2000, 16), (8, 64, 28, 4, 128, 2000, 32),
    (16, 64, 12, 2, 128, 700, 16), (16, 64, 28, 4, 128, 500, 32), (4, 256, 14, 2, 64, 1000, 16), (8, 512, 14, 2, 64, 2000, 32),
    (8, 512, 28, 4, 128, 4000, 128), (8, 1024, 28, 4, 128, 1100, 128), (16, 1024, 14, 2, 64, 2000, 128), (1, 1, 16, 1, 64, 10**6, 16)])
def test_columns_per_workgroup(host, B, rows, hq, hkv, d, top, cols):
    """The sizes measured on both sides of each rule."""
    cache = kv(pages=1000, hkv=hkv, d=d)
    call = prefill(B, rows, hq, -(-top // 16), top, cache) if rows > 1 else decode(B, hq, -(-top // 16), top, cache)
    (st, launches, _), = host([call])
    assert st == "LGX_OK" and launches[0][0] == f"lgx_k_attn8_d{d}_c{cols}"


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 18, 33, 2047])
def test_append_and_read_cover_every_page_that_rows_can_touch(host, rows):
    """From any slot of a page: ceil((15 + rows) / 16) pages at most."""
    most = max(-(-(s + rows) // 16) for s in range(16))
    for st, launches, _ in host([append(B=3, rows=rows), read(B=3, n=rows)]):
        name, gx, gy, gz, block = launches[0]
        assert st == "LGX_OK" and len(launches) == 1 and gx == 3 * most and gz == 1
        # 14 query heads by fours, then 2 K and 2 V heads; a wave for each of the 18
        # where a sequence has one row
        assert gy == (2 if "read" in name else 5 if rows == 1 else 8)


@pytest.mark.parametrize("B,hq,hkv,d,top,rows,window", [
    (1, 14, 2, 64, 17, 1, 0), (1, 28, 4, 128, 8191, 1, 0), (64, 28, 4, 128, 4096, 1, 0), (16, 12, 2, 128, 32768, 1, 0),
    (1, 8, 8, 64, 1 << 20, 1, 0), (4096, 8, 8, 64, 129 * 256, 1, 0), (1, 16, 1, 128, 1 << 24, 1, 0),
    (1, 28, 4, 128, 8000, 5, 0), (8, 28, 4, 128, 4000, 512, 0), (2, 14, 2, 64, 30000, 3, 700), (1, 14, 2, 64, 30000, 1, 1),
    (1, 28, 4, 128, 100000, 2047, 100), (1, 1, 1, 64, 64, 2047, 0), (300, 8, 8, 64, 2000, 100, 0)])
def test_attention_reaches_every_tile_of_every_column(host, B, hq, hkv, d, top, rows, window):
    """A workgroup for every block of columns of every KV head at least, and where
    their tiles are split among more, room for every workgroup's partial results."""
    opts = ["opts", [0.0, 0.0, window, None]] if window else None
    cache = kv(pages=1000, hkv=hkv, d=d)
    call = prefill(B, rows, hq, -(-top // 16), top, cache, opts) if rows > 1 else decode(B, hq, -(-top // 16), top, cache, opts)
    (st, launches, alloc), = host([call])
    assert st == "LGX_OK"
    name, gx, gy, gz, block = launches[0]
    assert name.startswith("lgx_k_attn8x_d" if window else "lgx_k_attn8_d") and gy == gz == 1
    cols = int(name.split("_c")[1])
    units = B * -(-rows * (hq // hkv) // cols)
    if len(launches) == 1:
        assert gx == units * hkv and alloc == 0
    else:
        assert gx % hkv == 0 and gx >= units * hkv and units <= 256
        assert launches[1][0] in (f"lgx_k_attn8_join_d{d}", f"lgx_k_attn8_joinw_d{d}")
        per = 4 if "joinw" in launches[1][0] else 1
        assert launches[1][1] * per >= B * rows * hq > (launches[1][1] - 1) * per
        assert alloc >= gx * cols * (d + 2) * 4 + units * 8


def angles(max_pos, rot, theta):
    return np.arange(max_pos)[:, None] * theta ** (-2.0 * np.arange(rot // 2) / rot)


def tables(max_pos, rot, theta, scaling=None):
    c, s = (np.full((max_pos, rot // 2), 9, np.float32) for _ in range(2))
    sc = lgx.RopeScalingC(*scaling) if scaling else None
    st = lgx.lib().lgx_rope_tables(max_pos, rot, theta, C.byref(sc) if sc else None, c.ctypes.data, s.ctypes.data)
    return lgx.STATUS_NAMES[st], c, s


@pytest.mark.parametrize("max_pos,rot,theta", [(1, 2, 1e4), (50, 64, 1e6), (70000, 10, 1e4)])
def test_rope_tables(max_pos, rot, theta):
    """Plain and scaled angles in 64 bits, within half a unit of binary32."""
    ang = angles(max_pos, rot, theta)
    w = ang[1] if max_pos > 1 else np.zeros(rot // 2)
    half = 2.0 ** -24 + 1e-10                        # the angles of 70000 positions lose 1e-11
    turns = 4096 * theta ** (-2.0 * np.arange(rot // 2) / rot) / (2 * np.pi)
    keep = np.clip((turns - 1) / 31, 0, 1)
    for scaling, want, amp in ((None, ang, 1), ((0, 0, 0.0, 0.0, 0.0), ang, 1), ((1, 0, 4.0, 0.0, 0.0), ang / 4, 1),
                               ((2, 0, 4.0, 0.0, 0.0), angles(max_pos, rot, theta * 4.0 ** (rot / (rot - 2)) if rot > 2 else theta), 1),
                               ((3, 4096, 8.0, 1.0, 32.0), ang * keep + ang / 8 * (1 - keep), 0.1 * np.log(8) + 1)):
        st, c, s = tables(max_pos, rot, theta, scaling)
        assert st == "LGX_OK"
        assert np.abs(c - amp * np.cos(want)).max() <= amp * half and np.abs(s - amp * np.sin(want)).max() <= amp * half
    if rot > 2:                                      # by base: the slowest pair 4 times slower, the fastest as it was
        _, c, _ = tables(max_pos, rot, theta, (2, 0, 4.0, 0.0, 0.0))
        assert np.allclose(c[:, 0], np.cos(np.arange(max_pos)), atol=2e-7)
        assert np.allclose(c[:, -1], np.cos(np.arange(max_pos) * w[-1] / 4), atol=2e-7)


@pytest.mark.parametrize("args", [(0, 4, 1e4), (4, 3, 1e4), (4, 0, 1e4), (4, 4, 0.0), (4, 4, float("inf")),
                                  (4, 4, 1e4, (4, 0, 1.0, 0.0, 0.0)), (4, 4, 1e4, (-1, 0, 1.0, 0.0, 0.0)),
                                  (4, 4, 1e4, (1, 0, 0.5, 0.0, 0.0)), (4, 4, 1e4, (2, 0, float("nan"), 0.0, 0.0)),
                                  (4, 4, 1e4, (3, 0, 2.0, 1.0, 32.0)), (4, 4, 1e4, (3, 10, 2.0, 32.0, 32.0))])
def test_rope_tables_refusals(args):
    st, c, s = tables(*args)
    assert st == "LGX_INVALID_ARGUMENT" and (c == 9).all() and (s == 9).all()


def test_structs_match_the_header():
    """The ctypes mirrors have the header's fields in its order."""
    import re

    src = open(os.path.join(ROOT, "include", "lgx.h")).read()
    for name, mirror in (("lgx_kv_i8", lgx.KvI8C), ("lgx_rope", lgx.RopeC), ("lgx_rope_scaling", lgx.RopeScalingC),
                         ("lgx_attn_opts", lgx.AttnOptsC)):
        body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct %s \{(.*?)\}" % name, src, re.S).group(1), flags=re.S)
        fields = [f for decl in body.split(";") for f in re.findall(r"(\w+)\s*(?:,|$)", decl.strip())]
        assert fields == [f for f, _ in mirror._fields_], name
