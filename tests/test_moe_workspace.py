"""Workspaces of the expert FFN over chunks of tokens, followed on the host (host_runtime.cpp in place of the GPU).

A long list of tokens runs as chunks through one workspace, and its last chunk is shorter. A shared expert in Q4_K /
Q6_K can need more memory for fewer rows (its products then split K, with a plane of partial sums each), so the
workspace has to cover both lengths.
"""
import ctypes
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
LIB = os.path.join(os.path.dirname(HERE), "inference_amd", "_lib", "libqmm.so")
F32, Q4K, Q6K, MXFP4 = 0, 12, 14, 39


@pytest.fixture(scope="module")
def runtime(tmp_path_factory):
    so = tmp_path_factory.mktemp("host") / "host_runtime.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    os.path.join(HERE, "host_runtime.cpp"), "-o", str(so)], check=True)
    return str(so)


class Host:
    """The library over the stand-in, in a process of its own."""

    def __init__(self, so):
        self.rt = ctypes.CDLL(so, mode=ctypes.RTLD_GLOBAL)
        self.L = ctypes.CDLL(LIB)
        for f in ("qmm_moe_ffn_scored_workspace_size", "qmm_moe_ffn_ex_workspace_size", "qmm_moe_ffn_workspace_size",
                  "qmm_ffn_workspace_size"):
            getattr(self.L, f).restype = ctypes.c_size_t
        self.L.qmm_last_error.restype = ctypes.c_char_p

    def weight(self, dtype, n, k):
        h = ctypes.c_void_p()
        rc = self.L.qmm_qtensor_quantize(dtype, ctypes.c_int64(n), ctypes.c_int64(k), ctypes.c_void_p(1 << 40), None,
                                         ctypes.byref(h))
        assert rc == 0, self.L.qmm_last_error()
        return h

    def call(self, t, e, k, h, x, shared, score, ws_bytes):
        """(status, names of the launches) of qmm_moe_ffn_scored, or without a score of qmm_moe_ffn_ex."""
        p, i64, f = ctypes.c_void_p(1 << 41), ctypes.c_int64, ctypes.c_float
        ws = ctypes.c_void_p(1 << 42)
        self.rt.host_clear()
        if score:
            rc = self.L.qmm_moe_ffn_scored(p, F32, i64(t), i64(h), p, e, k, 1, None, 1, 1, 1, 1, f(1), *x, *shared, None,
                                           p, F32, i64(h), ws, ctypes.c_size_t(ws_bytes), None)
        else:
            rc = self.L.qmm_moe_ffn_ex(p, i64(t), i64(h), p, e, k, 1, f(1), *x, *shared, None, p, i64(h), ws,
                                       ctypes.c_size_t(ws_bytes), None)
        self.rt.host_launch.restype = ctypes.c_char_p
        return rc, [self.rt.host_launch(i).decode() for i in range(self.rt.host_launches())]


def check_mxfp4(so):
    host = Host(so)
    L, none = host.L, (None,) * 3
    for topk, hidden, ffn, chunk, rest in ((8, 4096, 1024, 4096, 1536), (8, 7168, 1024, 4096, 1408), (2, 512, 256, 16384, 9)):
        e = 16
        x = [host.weight(MXFP4, *s) for s in ((e * 64, hidden), (e * 64, hidden), (e * hidden, 64))]
        shared = [host.weight(*s) for s in ((Q4K, ffn, hidden), (Q4K, ffn, hidden), (Q6K, hidden, ffn))]
        whole, last = (L.qmm_ffn_workspace_size(*shared, ctypes.c_int64(t), 0) for t in (chunk, rest))
        for t in (rest, chunk, chunk + rest, 3 * chunk + rest):
            args = (x[0], x[2], ctypes.c_int64(t), e, topk)
            routed = L.qmm_moe_ffn_scored_workspace_size(*args, *none)
            total = L.qmm_moe_ffn_scored_workspace_size(*args, *shared)
            assert total == L.qmm_moe_ffn_ex_workspace_size(*args, *shared)
            need = last if t == rest else whole if t == chunk else max(whole, last)
            # the shared expert's rows, then its own workspace
            assert total >= routed + 4 * min(t, chunk) * hidden + need, (topk, hidden, t, total, routed, whole, last)
            for score in (False, True):
                rc, names = host.call(t, e, topk, hidden, x, shared, score, total)
                assert rc == 0, (t, L.qmm_last_error())
                assert names.count("qmm_mx_combine") == -(-t // chunk)
                assert host.call(t, e, topk, hidden, x, shared, score, total - 1) == (1, [])
    assert last < whole  # (and a case in which the full chunk is the larger one)


def check_other_types(so):
    host = Host(so)
    L = host.L
    e = 8
    for topk, hidden, ffn, chunk, rest, more in ((1, 512, 8192, 4096, 3584, True), (8, 2048, 8192, 1024, 896, True),
                                                 (4, 1024, 8192, 2048, 1792, True), (2, 2048, 1024, 4096, 976, False)):
        x = [host.weight(*s) for s in ((Q4K, e * 256, hidden), (Q4K, e * 256, hidden), (Q6K, e * hidden, 256))]
        shared = [host.weight(*s) for s in ((Q4K, ffn, hidden), (Q4K, ffn, hidden), (Q6K, hidden, ffn))]
        whole, last = (L.qmm_moe_ffn_ex_workspace_size(x[0], x[2], ctypes.c_int64(t), e, topk, *shared) for t in (chunk, rest))
        assert (last > whole) == more
        for t in (chunk, chunk + rest, 2 * chunk + rest):
            args = (x[0], x[2], ctypes.c_int64(t), e, topk)
            for score, size in ((True, L.qmm_moe_ffn_scored_workspace_size), (False, L.qmm_moe_ffn_ex_workspace_size)):
                total = size(*args, *shared)
                rc, names = host.call(t, e, topk, hidden, x, shared, score, total)
                assert rc == 0, (topk, t, score, L.qmm_last_error())
                assert names.count("qmm_moe_combine") == -(-t // chunk)
                assert host.call(t, e, topk, hidden, x, shared, score, total - 1) == (1, [])
        # without a shared expert a whole chunk's workspace covers every shorter one
        total = L.qmm_moe_ffn_workspace_size(*args)
        assert total == L.qmm_moe_ffn_workspace_size(x[0], x[2], ctypes.c_int64(chunk), e, topk)
        for score in (False, True):
            total = (L.qmm_moe_ffn_scored_workspace_size if score else L.qmm_moe_ffn_ex_workspace_size)(*args, *(None,) * 3)
            assert host.call(t, e, topk, hidden, x, (None,) * 3, score, total)[0] == 0
            assert host.call(t, e, topk, hidden, x, (None,) * 3, score, total - 1) == (1, [])


def run(check, so):
    """A check of this file in a process of its own: the stand-in must not meet a GPU's runtime."""
    code = f"import sys; sys.path.insert(0, {HERE!r}); import test_moe_workspace as t; t.{check}({so!r})"
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]


def test_mxfp4_experts_with_a_shared_expert_of_another_type(runtime):
    run("check_mxfp4", runtime)


def test_other_experts_with_a_shared_expert(runtime):
    run("check_other_types", runtime)
