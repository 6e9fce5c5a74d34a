"""Refusals, workspaces and launches of the paged cache's and the beam search's entry points, followed on the host
(host_runtime.cpp in place of the GPU), and drafted trees as masks."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
LIB = os.path.join(os.path.dirname(HERE), "inference_amd", "_lib", "libqmm.so")
F32, F16, BF16 = 0, 1, 30


class Cache(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "v", "table", "lens", "refs")] + [("pages", ctypes.c_int64)] + \
        [(n, ctypes.c_int) for n in ("dtype", "layers", "kv_heads", "page_size", "head_dim", "slots", "max_pages")]


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
        self.rt.host_launch.restype = ctypes.c_char_p
        self.L.qmm_last_error.restype = ctypes.c_char_p
        for f in ("qmm_kv_attention_workspace_size", "qmm_kv_fork_workspace_size", "qmm_kv_compact_workspace_size",
                  "qmm_beam_select_workspace_size"):
            getattr(self.L, f).restype = ctypes.c_size_t

    def cache(self, **kw):
        base = dict(k=1 << 40, v=1 << 41, table=1 << 42, lens=1 << 43, refs=1 << 44, pages=100, dtype=BF16, layers=2,
                    kv_heads=4, page_size=16, head_dim=128, slots=3, max_pages=20)
        return Cache(**{**base, **kw})

    def done(self, rc):
        names = [self.rt.host_launch(i).decode() for i in range(self.rt.host_launches())]
        self.rt.host_clear()
        return rc, names

    def append(self, c, **kw):
        a = dict(layer=0, q=1 << 45, k=1 << 46, v=1 << 47, x=F32, rows=5, ldq=2048, ldk=512, ldv=512, starts=1 << 48,
                 depths=None, cos=1 << 50, sin=1 << 51, positions=64, out=1 << 52, ldo=2048, heads=16)
        a.update(kw)
        i64, p = ctypes.c_int64, ctypes.c_void_p
        return self.done(self.L.qmm_kv_append(
            ctypes.byref(c) if c else None, a["layer"], p(a["q"]), p(a["k"]), p(a["v"]), a["x"], i64(a["rows"]),
            i64(a["ldq"]), i64(a["ldk"]), i64(a["ldv"]), p(a["starts"]), p(a["depths"]), p(a["cos"]), p(a["sin"]),
            i64(a["positions"]), p(a["out"]), i64(a["ldo"]), a["heads"], None))

    def attention(self, c, **kw):
        a = dict(layer=0, q=1 << 45, x=F32, rows=5, ldq=2048, starts=1 << 48, masks=None, ldm=0, max_rows=5, max_len=300,
                 heads=16, scale=0.1, out=1 << 52, ldo=2048, ws=1 << 53, ws_bytes=1 << 30)
        a.update(kw)
        i64, p = ctypes.c_int64, ctypes.c_void_p
        return self.done(self.L.qmm_kv_attention(
            ctypes.byref(c) if c else None, a["layer"], p(a["q"]), a["x"], i64(a["rows"]), i64(a["ldq"]), p(a["starts"]),
            p(a["masks"]), i64(a["ldm"]), a["max_rows"], i64(a["max_len"]), a["heads"], ctypes.c_float(a["scale"]),
            p(a["out"]), i64(a["ldo"]), p(a["ws"]), ctypes.c_size_t(a["ws_bytes"]), None))

    def size(self, c, rows=5, max_rows=5, max_len=300, heads=16):
        return self.L.qmm_kv_attention_workspace_size(ctypes.byref(c), ctypes.c_int64(rows), max_rows,
                                                      ctypes.c_int64(max_len), heads)

    def fork(self, c, **kw):
        a = dict(parents=1 << 45, keep=None, reserve=1, table=c.table, lens=c.lens, refs=c.refs, short=1 << 46, ws=1 << 47,
                 ws_bytes=1 << 34)
        a.update(kw)
        p = ctypes.c_void_p
        return self.done(self.L.qmm_kv_fork(ctypes.byref(c), p(a["parents"]), p(a["keep"]), a["reserve"], p(a["table"]),
                                            p(a["lens"]), p(a["refs"]), p(a["short"]), p(a["ws"]),
                                            ctypes.c_size_t(a["ws_bytes"]), None))

    def accept(self, c, path=1 << 45, ld=4, counts=1 << 46, lens=1 << 47):
        p = ctypes.c_void_p
        return self.done(self.L.qmm_kv_accept(ctypes.byref(c), p(path), ctypes.c_int64(ld), p(counts), p(lens), None))

    def compact(self, c, table=1 << 45, refs=1 << 46, used=1 << 47, ws=1 << 48, ws_bytes=1 << 34):
        p = ctypes.c_void_p
        return self.done(self.L.qmm_kv_compact(ctypes.byref(c), p(table), p(refs), p(used), p(ws),
                                               ctypes.c_size_t(ws_bytes), None))

    def beam(self, **kw):
        a = dict(logits=1 << 45, x=F32, ld=1000, batch=2, beams=4, vocab=1000, scores=1 << 46, finished=None, eos=-1, count=8,
                 tokens=1 << 47, parents=1 << 48, out=1 << 49, done=None, ws=1 << 50, ws_bytes=1 << 34)
        a.update(kw)
        i64, p = ctypes.c_int64, ctypes.c_void_p
        return self.done(self.L.qmm_beam_select(
            p(a["logits"]), a["x"], i64(a["ld"]), i64(a["batch"]), a["beams"], i64(a["vocab"]), p(a["scores"]),
            p(a["finished"]), a["eos"], a["count"], p(a["tokens"]), p(a["parents"]), p(a["out"]), p(a["done"]), p(a["ws"]),
            ctypes.c_size_t(a["ws_bytes"]), None))

    def reorder(self, src=1 << 45, src_rows=10, ld_src=64, dst=1 << 46, ld_dst=64, nbytes=64, index=1 << 47, rows=5):
        i64, p = ctypes.c_int64, ctypes.c_void_p
        return self.done(self.L.qmm_reorder_rows(p(src), i64(src_rows), i64(ld_src), p(dst), i64(ld_dst), i64(nbytes),
                                                 p(index), i64(rows), None))


def refused(*results):
    for rc, names in results:
        assert rc == 1 and names == [], (rc, names)


def check_cache(so):
    h = Host(so)
    for bad in (dict(dtype=2), dict(head_dim=96), dict(head_dim=0), dict(page_size=8), dict(page_size=24),
                dict(page_size=2048), dict(layers=0), dict(layers=1025), dict(kv_heads=0), dict(kv_heads=257), dict(pages=0),
                dict(pages=(1 << 24) + 1), dict(slots=0), dict(slots=4097), dict(max_pages=0), dict(max_pages=1 << 21),
                dict(max_pages=1 << 20, page_size=512), dict(slots=1024, max_pages=1 << 19), dict(k=None), dict(v=None),
                dict(table=None), dict(lens=None), dict(refs=None), dict(k=8), dict(v=(1 << 41) + 4)):
        c = h.cache(**bad)
        refused(h.append(c), h.attention(c), h.fork(c), h.accept(c), h.compact(c))
        assert h.L.qmm_last_error()
    refused(h.append(None), h.attention(None))


def check_append(so):
    h = Host(so)
    c = h.cache()
    assert h.append(c) == (0, ["qmm_kv_append_rows"])
    assert h.append(c, q=None, out=None, cos=None, sin=None) == (0, ["qmm_kv_append_rows"])
    assert h.append(c, rows=0) == (0, []) and h.append(c, rows=0, q=None, k=None, v=None, starts=None) == (0, [])
    assert h.append(c, out=1 << 45)[0] == 0
    # q, k and v of one wide row, the result in q's place or behind them all
    whole = dict(k=(1 << 45) + 8192, v=(1 << 45) + 10240, ldq=5120, ldk=5120, ldv=5120, ldo=5120)
    assert h.append(c, out=1 << 45, **whole)[0] == 0 and h.append(c, out=(1 << 45) + 12288, **whole)[0] == 0
    refused(h.append(c, out=(1 << 45) + 8188, **whole), h.append(c, out=(1 << 45) + 12284, **whole),
            h.append(c, out=(1 << 45) + 12292, **whole))
    refused(*(h.append(c, **b) for b in (
        dict(layer=-1), dict(layer=2), dict(k=None), dict(v=None), dict(starts=None), dict(cos=None), dict(sin=None),
        dict(out=None), dict(x=8), dict(heads=0), dict(heads=8193), dict(positions=0), dict(ldq=2047), dict(ldk=511),
        dict(ldv=1), dict(ldo=100), dict(out=(1 << 45) + 16), dict(out=1 << 45, ldo=4096), dict(out=1 << 46), dict(out=(1 << 47) + 512), dict(rows=-1), dict(rows=(1 << 20) + 1), dict(rows=1 << 20, heads=2048, ldq=1 << 18, ldo=1 << 18))))


def check_attention(so):
    h = Host(so)
    c = h.cache()
    # a tile of 16 columns, of 32, groups of four; the names say the parts of q and of the weights
    assert h.attention(c, max_rows=1, rows=3)[1] == ["qmm_kv_attn_bf16_d128_n16_q3_p3", "qmm_kv_attn_join"]
    assert h.attention(c, max_rows=8, rows=9, x=BF16)[1] == ["qmm_kv_attn_bf16_d128_n32_q1_p2", "qmm_kv_attn_join"]
    assert h.attention(c, max_rows=9, rows=9, x=F16)[1][0] == "qmm_kv_attn_bf16_d128_wide_q2_p2"
    assert h.attention(h.cache(dtype=F16), x=BF16, max_rows=1)[1][0] == "qmm_kv_attn_f16_d128_n16_q1_p2"
    assert h.attention(h.cache(dtype=F32, head_dim=256), ldq=4096, ldo=4096)[1][0] == "qmm_kv_attn_f32_d256_n32_q1_p1"
    assert h.attention(c, max_len=100, max_rows=1)[1] == ["qmm_kv_attn_bf16_d128_n16_q3_p3"]  # one chunk: nothing to join
    assert h.attention(c, max_len=100, max_rows=1, ws=None, ws_bytes=0)[0] == 0
    assert h.attention(c, rows=0) == (0, [])
    refused(*(h.attention(c, **b) for b in (
        dict(layer=2), dict(q=None), dict(starts=None), dict(out=None), dict(x=14), dict(heads=15), dict(heads=0),
        dict(heads=4 * 33, ldq=1 << 20, ldo=1 << 20), dict(max_rows=0), dict(max_len=0), dict(ldq=2047), dict(ldo=2047),
        dict(rows=-1), dict(rows=(1 << 20) + 1), dict(masks=1 << 49, ldm=0), dict(masks=1 << 49, ldm=1, max_rows=65),
        dict(ws=None), dict(ws_bytes=h.size(c) - 1), dict(ws=(1 << 53) + 8), dict(scale=float("nan")),
        dict(scale=float("-inf")), dict(out=(1 << 45) + 4), dict(out=1 << 45, ldo=4096))))
    assert h.attention(c, out=1 << 45)[0] == 0 and h.attention(c, rows=1, out=1 << 45, ldo=1 << 30)[0] == 0
    assert h.attention(c, rows=0, q=None, starts=None, out=None) == (0, [])
    assert h.attention(c, masks=1 << 49, ldm=2, max_rows=65)[0] == 0
    assert h.attention(c, ws_bytes=h.size(c))[0] == 0
    assert h.size(h.cache(head_dim=100)) == 0 and h.size(c, heads=3) == 0 and h.size(c, max_rows=0) == 0
    # too many workgroups for a launch
    refused(h.attention(h.cache(slots=4096, kv_heads=256, max_pages=16), heads=256, rows=1 << 20, max_rows=1 << 20, ldq=1 << 15,
                        ldo=1 << 15, ws_bytes=1 << 60))
    # every plan covers the sequence, in chunks of whole key tiles
    for slots in (1, 7, 64):
        for rows in (1, 4, 30, 300):
            for n in (1, 127, 129, 5000, 1 << 17):
                c = h.cache(slots=slots, max_pages=1 << 14)
                size = h.size(c, rows=rows, max_rows=rows, max_len=n)
                rc, names = h.attention(c, rows=rows, max_rows=rows, max_len=n, ws=1 << 53 if size else None, ws_bytes=size)
                assert rc == 0 and (size > 0) == (names[-1] == "qmm_kv_attn_join")
                assert size % (16 * rows * (128 * 4 + 8)) == 0 or size % 256 == 0


def check_pages(so):
    h = Host(so)
    c = h.cache()
    assert h.fork(c) == (0, ["qmm_kv_fork_small", "qmm_kv_copy_pages"])
    assert h.fork(c, reserve=0) == (0, ["qmm_kv_fork_small"])
    assert h.fork(h.cache(pages=5000))[1] == ["qmm_kv_fork_begin", "qmm_kv_fork_count", "qmm_kv_fork_plan", "qmm_kv_fork_commit"]
    need = h.L.qmm_kv_fork_workspace_size(ctypes.byref(c))
    assert h.fork(c, ws_bytes=need)[0] == 0
    refused(*(h.fork(c, **b) for b in (
        dict(parents=None), dict(reserve=-1), dict(reserve=321), dict(table=None), dict(lens=None), dict(refs=None),
        dict(short=None), dict(ws=None), dict(ws_bytes=need - 1), dict(ws=(1 << 47) + 4))))
    assert h.accept(c) == (0, ["qmm_kv_accept_rows"])
    assert h.accept(c, lens=c.lens) == (0, ["qmm_kv_accept_rows", "qmm_kv_accept_lens"])
    assert h.accept(c, path=None) == (0, ["qmm_kv_accept_lens"])
    assert h.accept(c, lens=1 << 46) == (0, ["qmm_kv_accept_rows", "qmm_kv_accept_lens"])
    refused(h.accept(c, lens=c.lens + 4), h.accept(c, lens=(1 << 46) + 8), h.accept(c, lens=(1 << 45) + 44))
    refused(h.accept(c, counts=None), h.accept(c, lens=None), h.accept(c, ld=0), h.accept(c, ld=(1 << 20) + 1))
    need = h.L.qmm_kv_compact_workspace_size(ctypes.byref(c))
    assert h.compact(c, ws_bytes=need) == (0, ["qmm_kv_compact_plan", "qmm_kv_compact_commit"])
    refused(h.compact(c, table=None), h.compact(c, refs=None), h.compact(c, used=None), h.compact(c, ws=None),
            h.compact(c, ws_bytes=need - 1), h.compact(c, ws=(1 << 48) + 2))


def check_beam(so):
    h = Host(so)
    assert h.beam() == (0, ["qmm_beam_slices_f32", "qmm_beam_merge"])
    assert h.beam(x=BF16, finished=1 << 51, eos=0, done=1 << 52)[1][0] == "qmm_beam_slices_bf16"
    i64 = ctypes.c_int64
    need = h.L.qmm_beam_select_workspace_size(i64(2), 4, i64(1000), 8)
    assert need and h.beam(ws_bytes=need)[0] == 0
    refused(*(h.beam(**b) for b in (
        dict(logits=None), dict(scores=None), dict(tokens=None), dict(parents=None), dict(out=None), dict(x=3), dict(ld=999),
        dict(batch=0), dict(beams=0), dict(beams=65), dict(vocab=0), dict(vocab=(1 << 20) + 1, ld=1 << 21), dict(count=0),
        dict(count=129), dict(batch=20000), dict(eos=-2), dict(eos=1000), dict(finished=1 << 51), dict(ws=None),
        dict(ws_bytes=need - 1), dict(ws=(1 << 50) + 8))))
    assert h.beam(batch=1, beams=1, ld=0)[0] == 0  # one row has no stride
    assert h.L.qmm_beam_select_workspace_size(i64(1), 65, i64(10), 1) == 0
    assert h.reorder() == (0, ["qmm_beam_reorder"])
    assert h.reorder(rows=0) == (0, []) and h.reorder(src_rows=0) == (0, []) and h.reorder(nbytes=0) == (0, [])
    refused(h.reorder(src=None), h.reorder(dst=None), h.reorder(index=None), h.reorder(rows=-1), h.reorder(src_rows=-1),
            h.reorder(nbytes=-1), h.reorder(ld_src=63), h.reorder(ld_dst=63), h.reorder(rows=(1 << 20) + 1),
            h.reorder(src_rows=1 << 30, ld_src=1 << 40), h.reorder(dst=(1 << 45) + 639), h.reorder(src=(1 << 46) + 100, dst=1 << 46))
    assert h.reorder(dst=(1 << 45) + 640)[0] == 0


@pytest.mark.parametrize("check", ["check_cache", "check_append", "check_attention", "check_pages", "check_beam"])
def test_host(runtime, check):
    code = f"import sys; sys.path.insert(0, {HERE!r}); import test_kv_host as t; t.{check}({runtime!r}); print('fine')"
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip().endswith("fine"), r.stdout + r.stderr


def test_struct_is_the_headers():
    """The Python mirror of qmm_kv_cache has the header's fields in its order."""
    import re
    from inference_amd import paged
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(os.path.dirname(HERE), "include", "qmm.h")).read(), flags=re.S)
    body = re.search(r"typedef struct qmm_kv_cache \{(.*?)\} qmm_kv_cache;", text, flags=re.S).group(1)
    names = [n.strip(" *") for line in body.split(";") if line.strip()
             for n in re.sub(r"^\s*(void|int32_t|int64_t|int)\b", "", line).split(",")]
    assert names == [f[0] for f in paged._Cache._fields_] == [f[0] for f in Cache._fields_]


def test_tree_masks():
    from inference_amd import QmmError
    from inference_amd.paged import tree_masks
    masks, depths = tree_masks([[-1, 0, 0, 1, -1], [], [-1]])
    assert masks.tolist() == [[1], [3], [5], [11], [16], [1]] and depths.tolist() == [0, 1, 1, 2, 0, 0]
    chain, deep = tree_masks([[j - 1 for j in range(130)]])
    assert chain.shape == (130, 3) and deep.tolist() == list(range(130))
    for j in range(130):
        bits = sum((int(w) & (1 << 64) - 1) << 64 * i for i, w in enumerate(chain[j].tolist()))
        assert bits == (1 << j + 1) - 1
    assert tree_masks([[-1]], words=3)[0].shape == (1, 3)
    assert tree_masks([])[0].shape == (0, 1)
    for bad in ([[0]], [[-1, 1]], [[-2]]):
        with pytest.raises(QmmError):
            tree_masks(bad)
    with pytest.raises(QmmError):
        tree_masks([[-1] * 65], words=1)


def test_cpu_tensors_are_refused():
    from inference_amd import PagedKVCache, QmmError, beam_select, reorder_rows
    z = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(QmmError):
        PagedKVCache(torch.zeros(1, 4, 1, 16, 64), torch.zeros(1, 4, 1, 16, 64), torch.zeros(2, 3, dtype=torch.int32), z, z)
    with pytest.raises(QmmError):
        beam_select(torch.zeros(2, 10), torch.zeros(2), 2, 2)
    with pytest.raises(QmmError):
        reorder_rows(torch.zeros(2, 10), z)


def check_masks(so):
    h = Host(so)
    c = h.cache()
    for most in (2 ** 31 - 1, 2 ** 31 - 63, 2 ** 31 - 64):
        refused(h.attention(c, masks=1 << 49, ldm=1, max_rows=most), h.attention(c, masks=1 << 49, ldm=1 << 20, max_rows=most))
    assert h.attention(c, masks=1 << 49, ldm=1 << 20, max_rows=1 << 26)[0] == 0 and h.attention(c, max_rows=2 ** 31 - 1)[0] == 0


def check_fork_lists(so):
    h = Host(so)
    c = h.cache(slots=4, max_pages=8, pages=16)
    need = h.L.qmm_kv_fork_workspace_size(ctypes.byref(c))
    other = dict(table=1 << 50, lens=1 << 51, refs=1 << 52, ws_bytes=need)
    assert h.fork(c)[0] == 0 and h.fork(c, **other)[0] == 0
    # each new list may be the cache's own, and they may differ in that; parents and keep are read first
    for own in ("table", "lens", "refs"):
        assert h.fork(c, **{**other, own: getattr(c, own)})[0] == 0
    assert h.fork(c, parents=c.lens, keep=c.lens)[0] == 0 and h.fork(c, keep=1 << 51, **other)[0] == 0
    # lists end to end
    assert h.fork(c, table=c.table + 128, lens=c.lens + 16, refs=c.refs - 64)[0] == 0
    for out, size in (("table", 128), ("lens", 16), ("refs", 64), ("short", 4)):
        for name in ("table", "lens", "refs"):
            if name != out:
                refused(h.fork(c, **{out: getattr(c, name)}))
            refused(h.fork(c, **{out: getattr(c, name) + 4}))
            if size > 4:
                refused(h.fork(c, **{out: getattr(c, name) - 4}))
        for b, at in (("table", 1 << 50), ("lens", 1 << 51), ("refs", 1 << 52), ("short", 1 << 46), ("ws", 1 << 47)):
            if b != out:
                refused(h.fork(c, **{**other, "ws_bytes": need, out: at}))
        refused(h.fork(c, **{**other, out: (1 << 47) + need - 4}))
    for at in (c.table, c.lens, c.refs, 1 << 45, 1 << 49):
        refused(h.fork(c, keep=1 << 49, ws=at), h.fork(c, keep=1 << 49, ws=at - 16 * (need // 16) + 16, ws_bytes=need))


def check_compact_lists(so):
    h = Host(so)
    c = h.cache(slots=4, max_pages=8, pages=16)
    need = h.L.qmm_kv_compact_workspace_size(ctypes.byref(c))
    assert h.compact(c)[0] == 0 and h.compact(c, table=c.table)[0] == 0 and h.compact(c, refs=c.refs)[0] == 0
    assert h.compact(c, table=c.table, refs=c.refs, used=c.refs + 64, ws=(1 << 48), ws_bytes=need)[0] == 0
    for out, size in (("table", 128), ("refs", 64), ("used", 4)):
        for name in ("table", "lens", "refs"):
            if name != out:
                refused(h.compact(c, **{out: getattr(c, name)}))
            refused(h.compact(c, **{out: getattr(c, name) + 4}))
            if size > 4:
                refused(h.compact(c, **{out: getattr(c, name) - 4}))
        for b, at in (("table", 1 << 45), ("refs", 1 << 46), ("used", 1 << 47), ("ws", 1 << 48)):
            if b != out:
                refused(h.compact(c, ws_bytes=need, **{out: at}))
        refused(h.compact(c, ws_bytes=need, **{out: (1 << 48) + need - 4}))
    for at in (c.table, c.lens, c.refs):
        refused(h.compact(c, ws=at))


def check_accept_lists(so):
    h = Host(so)
    c = h.cache(slots=4, max_pages=8, pages=16)
    for path in (1 << 45, None):
        assert h.accept(c, path=path, lens=c.table + 128)[0] == 0 and h.accept(c, path=path, lens=c.refs - 16)[0] == 0
        refused(h.accept(c, path=path, lens=c.table), h.accept(c, path=path, lens=c.table + 124),
                h.accept(c, path=path, lens=c.refs + 60), h.accept(c, path=path, lens=c.refs - 4))


def check_beam_outputs(so):
    h = Host(so)
    base = dict(finished=1 << 51, eos=0, done=1 << 52)
    assert h.beam(**base)[0] == 0
    # in place where a search has as many continuations as beams
    assert h.beam(count=4, **{**base, "out": 1 << 46, "done": 1 << 51})[0] == 0
    refused(h.beam(**{**base, "out": 1 << 46}), h.beam(**{**base, "done": 1 << 51}))
    need = h.L.qmm_beam_select_workspace_size(ctypes.c_int64(2), 4, ctypes.c_int64(1000), 4)
    size = 2 * 4 * 4
    logits = (1 << 45, 4 * 8 * 1000)
    for out in ("tokens", "parents", "out", "done"):
        for name, at, n in (("logits", *logits), ("scores", 1 << 46, size), ("finished", 1 << 51, size), ("tokens", 1 << 47, size),
                            ("parents", 1 << 48, size), ("out", 1 << 49, size), ("done", 1 << 52, size), ("ws", 1 << 50, need)):
            if name == out:
                continue
            for to in (at - size + 4, at + 4, at + n - 4) + (() if (out, name) in (("out", "scores"), ("done", "finished")) else (at,)):
                refused(h.beam(count=4, **{**base, out: to}))
            assert h.beam(count=4, ws_bytes=need, **{**base, out: at + n})[0] == 0 and h.beam(count=4, **{**base, out: at - size})[0] == 0
    for at in (1 << 45, 1 << 46, 1 << 51, (1 << 45) + 31984):
        refused(h.beam(count=4, **{**base, "ws": at}))
    assert h.beam(count=4, **{**base, "ws": (1 << 45) + 32000})[0] == 0


@pytest.mark.parametrize("check", ["check_masks", "check_fork_lists", "check_compact_lists", "check_accept_lists", "check_beam_outputs"])
def test_host_refusals(runtime, check):
    test_host(runtime, check)
