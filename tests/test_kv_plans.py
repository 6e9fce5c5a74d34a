"""How an attention over a cache in pages is planned (host_runtime.cpp in place of the GPU): the kernel's form by rows and
heads, chunks that cover a sequence, records that fit the workspace; and that the GPU tests of a form do plan as it."""
import ctypes
import subprocess
import sys

import pytest

from test_kv_host import BF16, F16, F32, HERE, Host, runtime  # noqa: F401


class Attention(ctypes.Structure):  # the kernels' argument
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "v", "table", "lens", "refs")] + \
        [(n, ctypes.c_int) for n in ("pages", "dtype", "layers", "kv_heads", "page_log", "head_dim", "slots", "max_pages")] + \
        [("starts", ctypes.c_void_p), ("rows", ctypes.c_int), ("max_rows", ctypes.c_int)] + \
        [(n, ctypes.c_void_p) for n in ("q", "masks", "out", "part", "state")] + \
        [(n, ctypes.c_int64) for n in ("ldq", "ldm", "ldo")] + \
        [(n, ctypes.c_int) for n in ("layer", "x_type", "heads", "wide", "out_wide", "splits", "chunk", "tiles",
                                     "group_rows", "join_lanes")] + [("scale", ctypes.c_float)]


def plan(h, c, rows, max_rows, max_len, heads, **kw):
    """(names, the argument, workspace bytes) of a call."""
    size = h.size(c, rows=rows, max_rows=max_rows, max_len=max_len, heads=heads)
    h.rt.host_argument.restype = ctypes.c_void_p
    h.rt.host_keep(ctypes.c_size_t(ctypes.sizeof(Attention)))
    done, seen = h.done, []

    def keep(rc):
        names = [h.rt.host_launch(i).decode() for i in range(h.rt.host_launches())]
        seen.extend(Attention.from_buffer_copy(ctypes.string_at(h.rt.host_argument(i), ctypes.sizeof(Attention)))
                    for i in range(len(names)))
        return done(rc)
    h.done = keep
    ld = heads * c.head_dim
    rc, names = h.attention(c, rows=rows, max_rows=max_rows, max_len=max_len, heads=heads, ldq=ld, ldo=ld,
                            ws=1 << 53 if size else None, ws_bytes=size, **kw)
    h.done = done
    h.rt.host_keep(ctypes.c_size_t(0))
    assert rc == 0 and all(bytes(a) == bytes(seen[0]) for a in seen)
    return names, seen[0], size


def form(rows, group):
    """rows of a sequence at most, heads over a kv head: the kernel's form, and rows of a workgroup."""
    if rows * group <= 16:
        return "n16", 16 // group
    return ("n32", 32 // group) if rows <= 32 // group else ("wide", 4 * (32 // group))


def check_plans(so):
    h = Host(so)
    types = {F32: "f32", F16: "f16", BF16: "bf16"}
    for dtype, dim in ((F32, 64), (F32, 128), (F32, 256), (BF16, 128), (F16, 256)):
        for slots, kv, group in ((1, 4, 4), (7, 1, 1), (64, 2, 12), (900, 3, 32), (5, 8, 5)):
            for rows in (1, 2, 3, 4, 6, 8, 16, 17, 32, 33, 300):
                for most in (1, 127, 128, 129, 5000, 1 << 17, 1 << 30):
                    c = h.cache(slots=slots, kv_heads=kv, dtype=dtype, head_dim=dim, max_pages=1 << 13)
                    names, a, size = plan(h, c, rows + 5, rows, most, kv * group)
                    kind, per = form(rows, group)
                    assert names[0].startswith(f"qmm_kv_attn_{types[dtype]}_d{dim}_{kind}_q"), names
                    assert a.group_rows == per and a.tiles == -(-rows // per) and (a.tiles == 1 or kind == "wide")
                    assert a.splits >= 1 and a.chunk % 128 == 0 and a.splits * a.chunk >= min(most, (1 << 13) * 16)
                    assert names[1:] == (["qmm_kv_attn_join"] if a.splits > 1 else [])
                    # the records of every row, head and chunk: head_dim floats, and two more behind them all
                    records = (rows + 5) * kv * group * a.splits if a.splits > 1 else 0
                    assert (size == 0) == (records == 0)
                    if records:
                        assert a.part == 1 << 53 and a.state >= a.part + records * dim * 4
                        assert a.state + records * 8 <= (1 << 53) + size
                    assert a.rows == rows + 5 and a.max_rows == rows and a.heads == kv * group
                    assert 1 <= a.join_lanes <= 1024 // dim


def check_forms(so):
    """The calls of test_gpu_kv_forms.py: each form is what its name says, on one chunk and on several."""
    import test_gpu_kv_forms as g
    h = Host(so)
    types = {"f32": F32, "f16": F16, "bf16": BF16}
    seen = set()
    for cache, x in g.PAIRS:
        for dim in g.DIMS:
            for kind, heads, kv, r in g.FORMS:
                for lens in (g.SHORT, g.LONG):
                    rows = g.rows_of(r)
                    pages = max(-(-(a + b) // 16) for a, b in zip(lens, rows))
                    c = h.cache(dtype=types[cache], head_dim=dim, kv_heads=kv, slots=len(lens), max_pages=pages)
                    names, a, _ = plan(h, c, sum(rows), r, pages * 16, heads, x=types[x])
                    assert f"_d{dim}_{kind}_" in names[0] and (a.splits > 1) == (lens is g.LONG or r == 150), (names, a.splits)
                    seen.add(names[0])
    # every kernel of the attention
    assert len(seen) == 3 * 3 * (1 + 2 + 3) == len(g.DIMS) * 3 * 6


@pytest.mark.parametrize("check", ["check_plans", "check_forms"])
def test_plans(runtime, check):  # noqa: F811
    code = f"import sys; sys.path.insert(0, {HERE!r}); import test_kv_plans as t; t.{check}({runtime!r}); print('fine')"
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip().endswith("fine"), r.stdout + r.stderr
