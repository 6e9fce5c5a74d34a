"""The attention over a cache in pages in each of its three forms (one tile of 16 columns, one of 32, groups of four:
test_kv_plans.py follows that these calls plan so), for every type, head size and kind of mask, on one chunk of positions
and on several; runs of a prompt's length; many sequences. Tolerances are test_gpu_kv_attention.py's."""
import numpy as np
import pytest
import torch

from inference_amd import PagedKVCache
from inference_amd.paged import tree_masks
from test_gpu_kv_attention import check, step

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DIMS = (64, 128, 256)
PAIRS = [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f16"), ("bf16", "f32"), ("f16", "f16"),
         ("f16", "bf16"), ("f16", "f32")]
# form, heads, kv heads, rows of a sequence at most
FORMS = [("n16", 8, 2, 1), ("n16", 5, 1, 3), ("n16", 3, 3, 16), ("n32", 8, 2, 5), ("n32", 5, 1, 6), ("n32", 32, 1, 1),
         ("n32", 2, 2, 31), ("wide", 8, 2, 9), ("wide", 12, 1, 3), ("wide", 2, 2, 150)]
SHORT, LONG = [0, 45, 70, 33], [3, 701, 0, 260]


def rows_of(r):
    return [r, max(r // 2, 1), r, max(r - 1, 1)]


def trees(rows, seed):
    rng = np.random.default_rng(seed)
    return tree_masks([[int(rng.integers(max(-1, j - 9), j)) if j else -1 for j in range(n)] for n in rows])[0]


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("cache,x", PAIRS)
def test_forms(cache, x, dim):
    for at, (form, heads, kv, r) in enumerate(FORMS):
        rows = rows_of(r)
        if r == 150 and (cache, x) not in (("f32", "f32"), ("bf16", "f32")):
            continue
        for lens in (SHORT, LONG):
            c, q, starts, pools, table = step(at + dim, lens, rows, heads, kv, dim, 16, x, cache)
            masks = trees(rows, at)
            for m in (None, masks):
                got = c.attention(0, q.to(DEV), starts.to(DEV), masks=None if m is None else m.to(DEV), max_rows=r)
                check(got, q, pools, table, lens, starts, m, dim ** -0.5)


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("cache,x", PAIRS)
def test_nothing_unseen_reaches_a_row_in_any_form(cache, x, dim):
    """Infinities and NaN in keys and in values of rows that a mask, or the order of a run, hides; and rows that see
    nothing at all."""
    for at, (form, heads, kv, r) in enumerate([("n16", 8, 2, 4), ("n32", 8, 2, 7), ("wide", 8, 2, 20)]):
        rows, g = rows_of(r), torch.Generator().manual_seed(at)
        for lens in ([0, 45, 0, 3], [3, 701, 0, 260]):
            bad = [0, r - 1, 1, 2]  # the hidden row of each step
            for part, value in ((0, float("nan")), (1, float("inf"))):
                c, q, starts, pools, table = step(at + dim + part, lens, rows, heads, kv, dim, 16, x, cache)
                masks = torch.randint(0, 2 ** 31, (sum(rows), 1), generator=g)
                for s, i in enumerate(bad):
                    t = lens[s] + i
                    if i < rows[s]:
                        pools[part][0, table[s, t // 16], :, t % 16] = value
                    masks[int(starts[s]):int(starts[s + 1])] &= ~(1 << i)
                masks[int(starts[2])] = 0  # (of the sequence without a text)
                c = PagedKVCache(pools[0].to(DEV), pools[1].to(DEV), c.table, c.lens, c.refs)
                got = c.attention(0, q.to(DEV), starts.to(DEV), masks=masks.to(DEV), max_rows=r)
                assert torch.isfinite(got).all() and not got[int(starts[2])].any()
                check(got, q, pools, table, lens, starts, masks, dim ** -0.5)
                # a run: the rows before the bad one
                got = c.attention(0, q.to(DEV), starts.to(DEV), max_rows=r)
                for s, i in enumerate(bad):
                    first = int(starts[s])
                    assert torch.isfinite(got[first:first + min(i, rows[s])]).all()


def exact(q, k, v, base, scale):
    """A run's result in 64 bits, with the three sums that a tolerance needs (test_gpu_kv_attention.py): q [rows, heads,
    dim], k and v [kv heads, positions, dim]."""
    rows, heads, dim = q.shape
    g = heads // k.shape[0]
    n = k.shape[1]
    seen = torch.arange(n, device=DEV) <= base + torch.arange(rows, device=DEV)[:, None]
    out, mag, dot, top = (torch.empty((rows, heads, d), dtype=torch.float64, device=DEV) for d in (dim, dim, 1, 1))
    for h in range(heads):
        x, kk, vv = q[:, h].double(), k[h // g].double(), v[h // g].double()
        sc = (x @ kk.t().contiguous() * scale).masked_fill(~seen, -float("inf"))
        w = torch.softmax(sc, -1)
        out[:, h], mag[:, h] = w @ vv, w @ vv.abs()
        dot[:, h, 0] = (x.abs() @ kk.abs().t().contiguous()).masked_fill(~seen, 0.0).amax(-1) * abs(scale)
        top[:, h, 0] = sc.masked_fill(~seen, 0.0).abs().amax(-1)
    return out, mag, dot, top


@pytest.mark.parametrize("cache,x,dim,heads,kv", [("f32", "f32", 128, 8, 2), ("bf16", "bf16", 128, 8, 2),
                                                  ("f16", "f16", 128, 8, 2), ("bf16", "f32", 128, 4, 4),
                                                  ("f32", "f32", 64, 6, 2), ("bf16", "bf16", 64, 8, 1),
                                                  ("f32", "f32", 256, 4, 2), ("bf16", "f32", 256, 4, 1)])
def test_runs_of_a_prompts_length(cache, x, dim, heads, kv):
    """Prompts of 1000 rows and more, into an empty slot and behind a text, beside a token of another sequence."""
    for lens, rows in (([0, 300, 40], [1500, 1, 0]), ([517, 0], [1111, 64])):
        g = torch.Generator(device=DEV).manual_seed(dim + rows[0])
        total = [a + b for a, b in zip(lens, rows)]
        c = PagedKVCache.empty(1, sum(-(-t // 64) for t in total) + 1, kv, 64, dim, len(lens), 40, T[cache], DEV)
        first = 0
        for s, t in enumerate(total):
            need = -(-t // 64)
            c.table[s, :need] = first + torch.randperm(need, device=DEV, generator=g).int()
            first += need
        c.k.normal_(generator=g), c.v.normal_(generator=g)
        c.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        starts = torch.tensor(np.cumsum([0] + rows), dtype=torch.int32, device=DEV)
        q = torch.randn((sum(rows), heads, dim), device=DEV, generator=g).to(T[x])
        got = c.attention(0, q, starts, max_rows=max(rows), max_len=max(total))
        for s, (a, b) in enumerate(zip(lens, rows)):
            ids = c.table[s, :-(-(a + b) // 64)].long()
            k, v = (p[0, ids].transpose(0, 1).reshape(kv, -1, dim)[:, :a + b] for p in (c.k, c.v))
            at = int(starts[s])
            if b == 0:
                continue
            want, mag, dot, top = exact(q[at:at + b], k, v, a, dim ** -0.5)
            e = torch.finfo(T[x]).eps / 2
            score = dot * (dim / 4 + 4) * 2.0 ** -24 + top * 2.0 ** -22
            tol = mag * (2 * score + 2.0 ** -22 + (2.0 ** -15 if x != "f32" else 0) + (64 + (a + b) / 128) * 2.0 ** -24) + \
                want.abs() * e + 2.0 ** -24 * (x == "f16")
            assert bool(((got[at:at + b].double() - want).abs() <= tol).all())


@pytest.mark.parametrize("cache,x", [("f32", "f32"), ("bf16", "bf16")])
def test_many_sequences(cache, x):
    """More sequences than a workgroup has threads: rows and results, and what is appended."""
    n = 700
    rng = np.random.default_rng(5)
    lens, rows = rng.integers(0, 40, n).tolist(), rng.integers(0, 3, n).tolist()
    rows[0] = rows[255] = rows[256] = rows[600] = rows[699] = 2
    lens[3], lens[600] = 3300, 3500
    c, q, starts, pools, table = step(17, lens, rows, 4, 1, 64, 16, x, cache, max_pages=400)
    for max_len in (48, None):  # (whole, and the two long ones in two chunks)
        got = c.attention(0, q.to(DEV), starts.to(DEV), max_rows=2, max_len=max_len)
        check(got, q, pools, table, lens, starts, None, 0.125)
    g = torch.Generator().manual_seed(6)
    k, v = (torch.randn((sum(rows), 1, 64), generator=g).to(T[x]) for _ in range(2))
    out = c.append(0, k.to(DEV), v.to(DEV), starts.to(DEV), q=q.to(DEV))
    assert torch.equal(out, q.to(DEV))
    for s in range(n):
        for j in range(rows[s]):
            t = lens[s] + j
            for pool, new in zip(pools, (k, v)):
                pool[0, table[s, t // 16], :, t % 16] = new[int(starts[s]) + j].to(T[cache])
    # (as bits: what is not written holds NaN)
    bits = torch.int32 if cache == "f32" else torch.int16
    assert torch.equal(c.k.view(bits).cpu(), pools[0].view(bits)) and torch.equal(c.v.view(bits).cpu(), pools[1].view(bits))


def test_row_lists_out_of_range():
    """Of row lists outside their range, which rows are written and what they hold; on one chunk and on several."""
    for lens, wide in (([40, 33], 3), ([900, 1200], 80)):
        rows = [1, 1]
        # (a list that gives a slot both rows has its second position on a page of zeros)
        c, q, starts, pools, table = step(18, lens, rows, 4, 1, 128, 16, "f32", "f32", bad=False, max_pages=wide)
        for odd, written in (([-1, 1, 2], [1]), ([5, 6, 7], []), ([0, 2 ** 31 - 1, 2 ** 31 - 1], [0, 1]), ([2, 1, 0], []),
                             ([0, 0, 0], []), ([0, 1, 1], [0]), ([-2 ** 31, 0, 2], [0, 1]), ([0, 0, 2 ** 31 - 1], [0, 1])):
            out = torch.full_like(q, 7.0).to(DEV)
            odd = torch.tensor(odd, dtype=torch.int32)
            c.attention(0, q.to(DEV), odd.to(DEV), out=out)
            left = [r for r in range(2) if r not in written]
            assert (out[left] == 7).all() and not (out[written] == 7).any()
            out[left] = float("nan")
            check(out, q, pools, table, lens, odd, None, 128 ** -0.5)
