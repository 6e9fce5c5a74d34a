"""Attention over a cache in pages against 64 bits: types, head layouts, pages that end inside a tile, lengths from
nothing on, drafted trees, and infinities and NaN wherever a row does not look.

Tolerance of an output (in units of the sum of weight * |v|, the largest it can be): a score is off by its products'
roundings, dim of them in chains of dim / 4 at most, each 2^-24 of sum |q k|, and by 2^-22 of its own size in the
exponent; a weight is off twice by that (itself and the sum's), by 2^-22 of the exponential and, where the output has
16 bits, 2^-15 of its two parts; the running sums add a rounding for each of 64 steps and of n / 128 tiles. The result
is then rounded to its type: eps / 2 of it."""
import numpy as np
import pytest
import torch

from inference_amd import PagedKVCache, QmmError
from inference_amd.paged import tree_masks
from oracle import paged

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def step(seed, lens, rows, heads, kv, dim, page, x, cache, layers=1, layer=0, spare=3, bad=True, max_pages=None):
    """A cache whose pages lie anywhere, the positions lens[s] + rows[s] of every slot in it, everything else
    infinite or NaN; and q."""
    g = torch.Generator().manual_seed(seed)
    total = [a + b for a, b in zip(lens, rows)]
    need = [-(-t // page) for t in total]
    pages = sum(need) + spare
    wide = max_pages or max(max(need), 1)
    ids = torch.randperm(pages, generator=g).tolist()
    junk = torch.tensor([np.nan, np.inf, -np.inf, 1.0])
    pools = []
    for _ in range(2):
        p = junk[torch.randint(0, 4, (layers, pages, kv, page, dim), generator=g)] if bad else \
            torch.zeros(layers, pages, kv, page, dim)
        pools.append(p.to(T[cache]))
    table = torch.full((len(lens), wide), -1, dtype=torch.int32)
    for s, t in enumerate(total):
        for j in range(need[s]):
            p = ids.pop()
            table[s, j] = p
            n = min(page, t - j * page)
            for pool in pools:
                pool[layer, p, :, :n] = torch.randn((kv, n, dim), generator=g).to(T[cache])
    starts = torch.tensor(np.cumsum([0] + rows), dtype=torch.int32)
    q = torch.randn((sum(rows), heads, dim), generator=g).to(T[x])
    c = PagedKVCache(pools[0].to(DEV), pools[1].to(DEV), table.to(DEV), torch.tensor(lens, dtype=torch.int32).to(DEV),
                     torch.zeros(pages, dtype=torch.int32, device=DEV))
    return c, q, starts, pools, table


def check(got, q, pools, table, lens, starts, masks, scale, layer=0, max_rows=None):
    kp, vp = (p[layer].float().numpy() for p in pools)
    m = None if masks is None else masks.numpy().astype(np.int64).view(np.uint64)
    with np.errstate(invalid="ignore"):
        want, mag, dot, top = paged.attention(q.float().numpy(), kp, vp, table.numpy(), lens, starts.numpy(), m, scale,
                                              max_rows)
    n, dim = max(lens) + q.shape[0], q.shape[2]
    e = torch.finfo(got.dtype).eps / 2
    score = dot * (dim / 4 + 4) * 2.0 ** -24 + top * 2.0 ** -22
    tol = mag * (2 * score + 2.0 ** -22 + (2.0 ** -15 if got.dtype != torch.float32 else 0)
                 + (64 + n / 128) * 2.0 ** -24) + np.abs(want) * e + 2.0 ** -24 * (got.dtype == torch.float16)
    got = got.float().cpu().numpy().astype(np.float64)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    off = np.abs(got - want) - tol
    assert np.nanmax(off, initial=-1) <= 0, (np.nanmax(np.abs(got - want) / np.maximum(tol, 1e-300)))


LAYOUTS = [(8, 2, 64), (6, 2, 64), (4, 4, 128), (32, 8, 128), (8, 1, 128), (5, 1, 128), (16, 2, 256), (32, 1, 64)]


@pytest.mark.parametrize("cache,x", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32"),
                                     ("f32", "bf16"), ("bf16", "f16"), ("f16", "bf16")])
@pytest.mark.parametrize("heads,kv,dim", LAYOUTS)
def test_tokens_and_runs(cache, x, heads, kv, dim):
    lens, rows = [0, 1, 31, 32, 77, 300, 5], [1, 1, 2, 9, 1, 3, 0]
    for page in (16, 64):
        c, q, starts, pools, table = step(heads + dim + page, lens, rows, heads, kv, dim, page, x, cache)
        got = c.attention(0, q.to(DEV), starts.to(DEV))
        check(got, q, pools, table, lens, starts, None, dim ** -0.5)


@pytest.mark.parametrize("cache,x", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("page", [16, 32, 128])
def test_trees(cache, x, page):
    rng = np.random.default_rng(page)
    lens, rows = [0, 45, 130, 513, 64, 3], [5, 26, 64, 17, 1, 33]
    parents = [[int(rng.integers(-1, j)) if j else -1 for j in range(n)] for n in rows]
    masks, _ = tree_masks(parents)
    for heads, kv, dim in ((8, 2, 128), (4, 4, 64), (6, 1, 256)):
        c, q, starts, pools, table = step(page + dim, lens, rows, heads, kv, dim, page, x, cache)
        got = c.attention(0, q.to(DEV), starts.to(DEV), masks=masks.to(DEV), max_rows=64, max_len=600)
        check(got, q, pools, table, lens, starts, masks, dim ** -0.5)


def test_wide_trees_and_free_masks():
    """More than 64 nodes; masks that see nothing, later rows, or rows past the sequence's."""
    rng = np.random.default_rng(3)
    lens, rows = [40, 0, 7], [150, 70, 2]
    masks = torch.from_numpy(rng.integers(-2 ** 63, 2 ** 63, (sum(rows), 3)))
    masks[::7] = 0
    masks[150:170] = 0  # (of the sequence without a text: rows that see nothing)
    for cache, x in (("f32", "f32"), ("bf16", "bf16")):
        c, q, starts, pools, table = step(9, lens, rows, 8, 2, 128, 16, x, cache)
        got = c.attention(0, q.to(DEV), starts.to(DEV), masks=masks.to(DEV))
        assert not got[150:170].any()
        check(got, q, pools, table, lens, starts, masks, 128 ** -0.5)


@pytest.mark.parametrize("cache", ["f32", "bf16", "f16"])
def test_nothing_unseen_reaches_a_row(cache):
    """Nodes of a tree that a row does not see hold infinities and NaN, in keys and in values."""
    lens, rows = [50, 0], [20, 9]
    for value in (np.nan, np.inf, -np.inf):
        for part in (0, 1):
            c, q, starts, pools, table = step(4, lens, rows, 8, 2, 128, 16, "f32" if cache == "f32" else cache, cache)
            bad = {(0, 3), (0, 11), (1, 4)}
            for s, i in bad:
                t = lens[s] + i
                pools[part][0, table[s, t // 16], :, t % 16] = value
            c = PagedKVCache(pools[0].to(DEV), pools[1].to(DEV), c.table, c.lens, c.refs)
            masks = torch.zeros((29, 1), dtype=torch.int64)
            for s in range(2):
                for j in range(rows[s]):
                    for i in range(j + 1):
                        if (s, i) not in bad and (i + j) % 3 != 1:
                            masks[int(starts[s]) + j, 0] |= 1 << i
            got = c.attention(0, q.to(DEV), starts.to(DEV), masks=masks.to(DEV))
            assert torch.isfinite(got).all()
            check(got, q, pools, table, lens, starts, masks, 128 ** -0.5)
            # causal: row j sees all up to itself, so rows before the bad one stay as they are
            got = c.attention(0, q.to(DEV), starts.to(DEV))
            assert torch.isfinite(got[:3]).all() and torch.isfinite(got[20:24]).all()


@pytest.mark.parametrize("cache", ["f32", "bf16"])
def test_infinite_values_that_a_row_sees(cache):
    """An infinity in a value that rows see is theirs, and only theirs."""
    lens, rows = [20], [6]
    c, q, starts, pools, table = step(5, lens, rows, 4, 1, 64, 16, "f32", cache)
    t = lens[0] + 2
    pools[1][0, table[0, t // 16], :, t % 16, 5] = float("inf")
    c = PagedKVCache(pools[0].to(DEV), pools[1].to(DEV), c.table, c.lens, c.refs)
    got = c.attention(0, q.to(DEV), starts.to(DEV))
    assert torch.isfinite(got[:2]).all() and torch.isinf(got[2:, :, 5]).all()
    assert torch.isfinite(got[2:, :, :5]).all() and torch.isfinite(got[2:, :, 6:]).all()


def test_long_sequences_and_large_scores():
    """Splits over workgroups; scores far above what an exponential holds."""
    for cache, x, heads, kv, dim, page, lens, rows, amp in (
            ("f32", "f32", 8, 2, 128, 16, [5000, 1], [1, 1], 1.0),
            ("bf16", "f32", 8, 2, 128, 64, [4099, 2000, 0], [3, 40, 1], 1.0),
            ("f16", "f16", 4, 1, 64, 32, [6001], [2], 30.0),
            ("f32", "f32", 4, 1, 256, 32, [1500], [9], 100.0)):
        c, q, starts, pools, table = step(len(lens) + dim, lens, rows, heads, kv, dim, page, x, cache)
        q = (q.float() * amp).to(T[x])
        for max_len in (None, max(lens) + 50, 100):
            got = c.attention(0, q.to(DEV), starts.to(DEV), max_len=max_len, max_rows=max(rows))
            check(got, q, pools, table, lens, starts, None, dim ** -0.5)


def test_strides_layers_and_padding():
    """Rows inside wider ones, another layer than the first, rows behind the last sequence left as they were, rows
    past max_rows left out, q in two dimensions."""
    lens, rows = [30, 12], [3, 5]
    c, q, starts, pools, table = step(6, lens, rows, 4, 2, 64, 16, "bf16", "bf16", layers=3, layer=2)
    wide = torch.full((12, 4 * 64 + 24), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:8, 8:8 + 256] = q.to(DEV).view(8, 256)
    out = torch.full((12, 300), 7.0, dtype=torch.bfloat16, device=DEV)
    c.attention(2, wide[:, 8:264], starts.to(DEV), out=out[:, 3:259])
    check(out[:8, 3:259].unflatten(1, (4, 64)), q, pools, table, lens, starts, None, 0.125, layer=2)
    assert (out[8:] == 7).all() and (out[:, :3] == 7).all() and (out[:, 259:] == 7).all()
    out = torch.full((8, 4, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    c.attention(2, q.to(DEV), starts.to(DEV), max_rows=3, out=out)
    check(out[:6], q[:6], pools, table, lens, torch.tensor([0, 3, 6]), None, 0.125, layer=2)
    assert (out[6:] == 7).all()
    got = c.attention(2, q.to(DEV), starts.to(DEV), scale=0.4)
    check(got, q, pools, table, lens, starts, None, 0.4, layer=2)


def test_missing_pages_and_odd_lists():
    """A position whose page is missing is NaN for the rows that see it, and reads nothing; lists outside their range
    leave rows out."""
    lens, rows = [40, 40], [1, 1]
    c, q, starts, pools, table = step(7, lens, rows, 4, 1, 128, 16, "f32", "f32")
    for entry in (-1, c.pages, 2 ** 31 - 1, -2 ** 31):
        t = table.clone()
        t[1, 1] = entry
        cc = PagedKVCache(c.k, c.v, t.to(DEV), c.lens, c.refs)
        got = cc.attention(0, q.to(DEV), starts.to(DEV))
        assert torch.isnan(got[1]).all() and torch.isfinite(got[0]).all()
    # a length past the slot's pages: cut to them (the row has no position of its own then)
    cc = PagedKVCache(c.k, c.v, c.table, torch.tensor([2 ** 31 - 1, -5], dtype=torch.int32, device=DEV), c.refs)
    out = cc.attention(0, q.to(DEV), starts.to(DEV))
    assert torch.isfinite(out[1]).all()
    for odd in ([-1, 1, 2], [5, 6, 7], [0, 2 ** 31 - 1, 2 ** 31 - 1], [2, 1, 0], [0, 0, 0]):
        out = torch.full_like(q, 7.0).to(DEV)
        c.attention(0, q.to(DEV), torch.tensor(odd, dtype=torch.int32, device=DEV), out=out)
        torch.cuda.synchronize()
    assert (out == 7).all()


def test_past_32_bit_offsets():
    """A pool of more than 2^32 bytes and 2^31 values: pages at its end."""
    pages, page, kv, dim = 4 * 8300, 64, 8, 128
    k = torch.zeros((1, pages, kv, page, dim), dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    assert k.numel() > 2 ** 31
    lens = [100]
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32)
    g = torch.Generator().manual_seed(1)
    small = [torch.zeros((1, 4, kv, page, dim), dtype=torch.bfloat16) for _ in range(2)]
    for pool, s in ((k, small[0]), (v, small[1])):
        for i, p in enumerate(table[0].tolist()):
            s[0, i] = torch.randn((kv, page, dim), generator=g).bfloat16()
            pool[0, p] = s[0, i].to(DEV)
    c = PagedKVCache(k, v, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV),
                     torch.zeros(pages, dtype=torch.int32, device=DEV))
    q = torch.randn((2, 16, dim), generator=g).bfloat16()
    starts = torch.tensor([0, 2], dtype=torch.int32)
    got = c.attention(0, q.to(DEV), starts.to(DEV))
    check(got, q, small, torch.tensor([[0, 1, 2]]), lens, starts, None, dim ** -0.5)


def test_streams_captures_and_repeats():
    """Two calls at once on streams of their own; a captured call replayed with other lists; the same bits each time."""
    lens, rows = [900, 77], [2, 30]
    c, q, starts, pools, table = step(8, lens, rows, 8, 2, 128, 32, "f32", "bf16")
    q, starts = q.to(DEV), starts.to(DEV)
    want = c.attention(0, q, starts, max_rows=32, max_len=950)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(c.attention(0, q, starts, max_rows=32, max_len=950))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.attention(0, q, starts, max_rows=32, max_len=950)
    for n in (900, 33, 0, 900):
        c.lens[0] = n
        out.fill_(3.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, c.attention(0, q, starts, max_rows=32, max_len=950))
    assert torch.equal(out, want)


def test_no_rows_and_rows_in_place():
    """A step without a row; results written over q; and over what overlaps it otherwise: refused."""
    lens, rows = [70, 3, 400], [1, 26, 9]
    for cache, x, n in (("f32", "f32", 26), ("bf16", "bf16", 26), ("f16", "f32", 1)):
        c, q, starts, pools, table = step(10, lens, [min(r, n) for r in rows], 8, 2, 128, 16, x, cache)
        want = c.attention(0, q.to(DEV), starts.to(DEV))
        here = q.to(DEV)
        assert c.attention(0, here, starts.to(DEV), out=here) is here and torch.equal(here, want)
        none = torch.empty((0, 8, 128), dtype=T[x], device=DEV)
        assert c.attention(0, none, torch.zeros(4, dtype=torch.int32, device=DEV)).shape == none.shape
        kv = torch.empty((0, 2, 128), dtype=T[x], device=DEV)
        assert c.append(0, kv, kv, torch.zeros(4, dtype=torch.int32, device=DEV), q=none).shape == none.shape
    total = q.shape[0]
    both = torch.zeros((total, 2, 8, 128), device=DEV)  # (rows between each other)
    both[:, 0] = q.to(DEV)
    c.attention(0, both[:, 0], starts.to(DEV), out=both[:, 1])
    assert torch.equal(both[:, 1], want)
    flat = torch.zeros((total + 1) * 1024, device=DEV)
    a, b = flat[:total * 1024].view(total, 8, 128), flat[128:128 + total * 1024].view(total, 8, 128)
    with pytest.raises(QmmError):
        c.attention(0, a, starts.to(DEV), out=b)
    with pytest.raises(QmmError):
        c.append(0, a[:, :2], a[:, 2:4], starts.to(DEV), q=a[:, 4:], out=a[:, 3:7])
    for bad in (dict(scale=float("nan")), dict(scale=float("inf")), dict(max_rows=0), dict(max_len=0)):
        with pytest.raises(QmmError):
            c.attention(0, q.to(DEV), starts.to(DEV), **bad)
    for layer in (-1, 1, 2 ** 32):
        with pytest.raises(QmmError):
            c.attention(layer, q.to(DEV), starts.to(DEV))
    with pytest.raises(AttributeError):
        c.table = c.table.clone()


@pytest.mark.parametrize("cache,x", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32")])
def test_scales(cache, x):
    """Scales below 0 and 0 itself (equal weights), in each form."""
    for rows in ([1, 1], [4, 2], [33, 1]):
        for scale in (-0.1, 0.0, 1e-30, -3.0):
            c, q, starts, pools, table = step(11, [50, 7], rows, 8, 2, 64, 16, x, cache)
            check(c.attention(0, q.to(DEV), starts.to(DEV), scale=scale), q, pools, table, [50, 7], starts, None, scale)


@pytest.mark.parametrize("cache", ["f16", "bf16"])
@pytest.mark.parametrize("part", [0, 1])
def test_values_below_the_normal_range(cache, part):
    """Keys (against a q as much larger), or values, that are denormal numbers of the cache's type."""
    low = 2.0 ** (-18 if cache == "f16" else -127)
    for rows in ([1, 1], [4, 2], [33, 1]):
        c, q, starts, pools, table = step(12, [50, 300], rows, 8, 2, 128, 16, "f32", cache, bad=False)
        pools[part] = (pools[part].double() * low).to(T[cache])
        (c.v if part else c.k).copy_(pools[part].to(DEV))
        if part == 0:
            q = q * (1 / low if cache == "f16" else 2.0 ** 122)
        check(c.attention(0, q.to(DEV), starts.to(DEV)), q, pools, table, [50, 300], starts, None, 128 ** -0.5)


@pytest.mark.parametrize("cache,x", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16")])
def test_wide_groups_of_heads(cache, x):
    """32 heads over one, 12 over one and 3 over one, a run of many rows; odd strides and boundaries; one chunk and many."""
    for heads, kv, dim in ((32, 1, 64), (12, 1, 128), (3, 1, 256)):
        for lens, rows, max_len in (([20, 0], [37, 9], 60), ([700, 0], [37, 9], None)):
            c, q, starts, pools, table = step(13 + heads, lens, rows, heads, kv, dim, 16, x, cache, max_pages=100)
            n = heads * dim
            wide = torch.full((48, n + 7), float("nan"), dtype=T[x], device=DEV)
            wide[:46, 3:3 + n] = q.to(DEV).view(46, n)
            out = torch.full((48, n + 5), 7.0, dtype=T[x], device=DEV)
            c.attention(0, wide[:, 3:3 + n], starts.to(DEV), max_len=max_len, out=out[:, 1:1 + n])
            check(out[:46, 1:1 + n].unflatten(1, (heads, dim)), q, pools, table, lens, starts, None, dim ** -0.5)
            assert (out[46:] == 7).all() and (out[:, 0] == 7).all() and (out[:, 1 + n:] == 7).all()


def test_two_graphs():
    """Two captured calls of different sizes, replayed in turn with eager ones between: each keeps its workspace."""
    lens, rows = [3000, 800], [1, 40]
    c, q, starts, pools, table = step(14, lens, rows, 8, 2, 128, 32, "bf16", "bf16")
    q, starts = q.to(DEV), starts.to(DEV)
    calls = [dict(max_rows=40, max_len=3000), dict(max_rows=41, max_len=100)]
    want = [c.attention(0, q, starts, **k) for k in calls]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for k in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c.attention(0, q, starts, **k))
        graphs.append(g)
    for i in (0, 1, 1, 0, 1, 0):
        outs[i].fill_(5.0)
        graphs[i].replay()
        assert torch.equal(c.attention(0, q, starts, **calls[1 - i]), want[1 - i])
        torch.cuda.synchronize()
        assert torch.equal(outs[i], want[i])


def test_masks_narrower_than_the_step():
    """A bound past the masks' bits is refused; without one, the rows past the bits of a sequence are zeros in a new
    result and stay in a given one."""
    lens, rows = [20, 6], [70, 3]
    c, q, starts, pools, table = step(15, lens, rows, 4, 2, 64, 16, "f32", "f32")
    masks = torch.from_numpy(np.random.default_rng(15).integers(-2 ** 63, 2 ** 63, (73, 1)))
    args = q.to(DEV), starts.to(DEV), masks.to(DEV)
    for most in (65, 70, 73, 1000):
        with pytest.raises(QmmError):
            c.attention(0, *args, max_rows=most)
    with pytest.raises(QmmError):
        c.attention(0, *args[:2], masks=args[2][:, :0])
    dirty = torch.full_like(args[0], 7.0)  # (what a new result's memory held)
    del dirty
    got = c.attention(0, *args)
    out = torch.full_like(args[0], 7.0)
    c.attention(0, *args, out=out)
    assert not got[64:70].any() and (out[64:70] == 7).all()
    keep = [r for r in range(73) if not 64 <= r < 70]
    assert torch.equal(got[keep], out[keep])
    want = out.clone()
    want[64:70] = float("nan")
    check(want, q, pools, table, lens, starts, masks, 0.125, max_rows=64)
    assert torch.equal(c.attention(0, *args, max_rows=64, out=out)[keep], got[keep])


def test_one_head_of_any_stride():
    """A dimension of one head has no stride: rows, results and what is appended with such views."""
    lens, rows = [40, 3], [2, 5]
    c, q, starts, pools, table = step(16, lens, rows, 1, 1, 64, 16, "f32", "f32")
    flat = torch.full((7, 200), 7.0, device=DEV)
    view = flat[:, None, 8:72]
    assert view.stride(1) != 64
    view.copy_(q.to(DEV))
    out = torch.full((7, 200), 9.0, device=DEV)
    got = c.attention(0, view, starts.to(DEV), out=out[:, None, 4:68])
    check(got, q, pools, table, lens, starts, None, 0.125)
    assert (out[:, :4] == 9).all() and (out[:, 68:] == 9).all()
    k, v = (torch.randn((7, 90), device=DEV)[:, None, 1:65] for _ in range(2))
    turned = torch.full((7, 200), 9.0, device=DEV)
    c.append(0, k, v, starts.to(DEV), q=view, out=turned[:, None, 100:164])
    assert torch.equal(turned[:, None, 100:164], view)
    for s in range(2):
        for j in range(rows[s]):
            t = lens[s] + j
            assert torch.equal(c.v[0, int(table[s, t // 16]), 0, t % 16], v[int(starts[s]) + j, 0])
