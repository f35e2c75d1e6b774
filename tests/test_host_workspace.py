"""The context's workspace over its lifetime, on a stand-in for the HIP runtime (no
device): memory that a recorded graph may hold is not freed when the workspace grows."""
import json
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# the recording stand-in with a log of frees, and with stream 2 under capture
STUB = r"""
#define hipFree stub_free_unlogged
#include "hip_stub.cpp"
#undef hipFree
extern "C" hipError_t hipFree(void* p) {
    g_log += "free " + std::to_string((size_t)p) + "\n";
    return hipSuccess;
}
extern "C" hipError_t hipStreamIsCapturing(hipStream_t s, hipStreamCaptureStatus* st) {
    *st = s == (hipStream_t)2 ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
    return hipSuccess;
}
"""

CHILD = r"""
import ctypes as C, json, sys
stub = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
stub.stub_log.restype = C.c_char_p
import logicaffeine_amd as lgx
L, P = lgx.lib(), 1 << 41
h = C.c_void_p()
lgx._check(L.lgx_ctx_create(0, b"stub", C.byref(h)))
for hq, top, stream in json.loads(sys.argv[2]):
    stub.stub_reset()
    kv = lgx.KvI8C(P, P, P, P, 100, hq, 128)
    if stream >= 0:
        lgx._check(L.lgx_gqa_decode_attn_i8(h, P, C.byref(kv), P, P, 2, hq, top // 16, top, None, P, stream or None))
    else:
        lgx._check(L.lgx_gqa_decode_attn(h, P, P, P, P, P, 2, hq, hq, 128, top // 16, 100, top, P, -stream))
    print(json.dumps([w.split() for w in stub.stub_log().decode().splitlines()]))
stub.stub_reset()
L.lgx_ctx_destroy(h)
print(json.dumps([w.split() for w in stub.stub_log().decode().splitlines()]))
"""


@pytest.fixture(scope="module")
def run(tmp_path_factory):
    at = tmp_path_factory.mktemp("stub")
    src, so = str(at / "stub.cpp"), str(at / "stub.so")
    with open(src, "w") as f:
        f.write(STUB)
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    subprocess.run(["g++", "-O1", "-fPIC", "-shared", "-std=c++17", f"-I{rocm}/include", f"-I{ROOT}/tests", "-o", so, src], check=True)

    def go(calls):
        r = subprocess.run([sys.executable, "-c", CHILD, so, json.dumps(calls)], cwd=ROOT, text=True, capture_output=True, timeout=300)
        assert r.returncode == 0, r.stderr[-4000:]
        return [json.loads(ln) for ln in r.stdout.splitlines()]

    return go


def only(log, what):
    return [int(w[1]) for w in log if w[0] == what]


# heads, tokens, stream (2: under capture; negative: the binary16 cache's attention)
SMALL, BIG, HUGE = (8, 4096), (8, 1 << 15), (8, 1 << 18)


def test_a_workspace_that_no_graph_holds_is_freed_when_it_grows(run):
    a, b, end = run([(*HUGE, -1), (16, 1 << 18, -1)])
    assert len(only(a, "malloc")) == 1 and only(a, "free") == []
    assert len(only(b, "malloc")) == 1 and len(only(b, "free")) == 1
    assert len(only(end, "free")) == 1


@pytest.mark.parametrize("first,stream", [((16, 1 << 14), -2), ((1, 1 << 20), 2)])
def test_a_workspace_that_a_graph_holds_stays(run, first, stream):
    """A step recorded once it has run, then a larger call on the same context, recorded
    or not: the replays still write into the first workspace, until the context ends."""
    eager = 1 if stream == 2 else -1
    logs = run([(*first, eager), (*first, stream), (*HUGE, -1), (16, 1 << 18, -1), (16, 1 << 19, -1)])
    assert len(only(logs[0], "malloc")) == 1 and only(logs[1], "malloc") == []
    grown = [len(only(x, "malloc")) for x in logs[2:5]]
    assert grown == [1, 1, 1]
    # the recorded one is kept; those after it were never recorded, and go
    assert [len(only(x, "free")) for x in logs[2:5]] == [0, 1, 1]
    assert len(only(logs[5], "free")) == 2


def test_memory_that_grows_under_capture_stays_too(run):
    logs = run([(*HUGE, -2), (16, 1 << 18, -2), (16, 1 << 19, -1)])
    assert [only(x, "free") for x in logs[:3]] == [[], [], []] and len(only(logs[3], "free")) == 3
