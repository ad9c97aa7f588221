"""How linear attention cuts chains of tokens into segments; host arithmetic, no GPU."""
import ctypes
import os
import subprocess
import tempfile

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ALL = 2**63 - 1


@pytest.fixture(scope="module")
def plan():
    out = os.path.join(tempfile.mkdtemp(), "plan.so")
    subprocess.check_call(["/usr/bin/g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-I", os.path.join(ROOT, "rwkv-rs-stable_b200", "csrc"),
                           os.path.join(ROOT, "tests", "cpp", "linear_attention_plan.cpp"), "-o", out])
    lib = ctypes.CDLL(out)
    lib.linear_attention_cut.argtypes = [ctypes.c_int64] * 5 + [ctypes.POINTER(ctypes.c_int64)]
    for f in (lib.linear_attention_segments_in, lib.linear_attention_state_bytes):
        f.argtypes, f.restype = [ctypes.c_int64] * 3, ctypes.c_int64
    return lib


def _cut(plan, *args):
    out = (ctypes.c_int64 * 2)()
    plan.linear_attention_cut(*args, out)
    return tuple(out)


def test_segments_cover_the_chunks_and_fit_the_places(plan):
    for chains in (0, 1, 2, 5, 12, 74, 148, 149, 4096):
        for chunks in (0, 1, 2, 3, 4, 5, 9, 16, 63, 256, 10**6):
            for places, launches in ((148, 4), (888, 1), (2368, 1), (1, 4), (0, 1)):
                for most in (0, 1, 2, 7, ALL):
                    segments, each = _cut(plan, chains, chunks, places, launches, most)
                    assert segments >= 1
                    if segments == 1:
                        assert each == chunks
                        continue
                    assert segments * chains <= places and segments <= most
                    assert (segments - 1) * each < chunks <= segments * each      # every segment has chunks
                    assert chunks > 2 * each + launches                           # and is worth its second walk


def test_a_workspace_of_what_was_asked_for_holds_the_cut(plan):
    for chains, chunks in ((1, 300), (12, 256), (24, 63), (32, 12)):
        segments, each = _cut(plan, chains, chunks, 148, 4, ALL)
        nbytes = plan.linear_attention_state_bytes(chains, segments, 64)
        assert _cut(plan, chains, chunks, 148, 4, plan.linear_attention_segments_in(nbytes, chains, 64)) == (segments, each)
        assert nbytes == (0 if segments == 1 else chains * segments * 64 * 64 * 4)
    assert plan.linear_attention_segments_in(10**9, 0, 64) == 0
