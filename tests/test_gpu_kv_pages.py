"""Appends, forks, accepted paths and packing of a cache in pages, against plain loops: lists have to be equal, and
pages are moved bit for bit. A rotated value is two products and a sum in f32 (2 roundings of the larger product, one
of the sum: 2^-23 of the products' sizes), then a rounding to its type."""
import numpy as np
import pytest
import torch

from inference_amd import PagedKVCache, QmmError
from oracle import paged

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def cache_of(seed, lens, page, pages, wide, layers=1, kv=2, dim=64, dtype="f32", share=()):
    """A cache with sequences of those lengths on pages anywhere, random contents; share: (slot, other, pages) rows
    that begin with another slot's pages."""
    g = torch.Generator().manual_seed(seed)
    ids = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(lens), wide), -1, dtype=torch.int32)
    for s, n in enumerate(lens):
        for j in range(-(-n // page)):
            table[s, j] = ids.pop()
    for s, o, n in share:
        for j in range(n):
            ids.append(int(table[s, j]))
            table[s, j] = table[o, j]
    refs = torch.zeros(pages, dtype=torch.int32)
    for p in table.flatten().tolist():
        if p >= 0:
            refs[p] += 1
    k, v = (torch.randn((layers, pages, kv, page, dim), generator=g).to(T[dtype]) for _ in range(2))
    return PagedKVCache(k.to(DEV), v.to(DEV), table.to(DEV), torch.tensor(lens, dtype=torch.int32).to(DEV), refs.to(DEV))


def host(c):
    return c.table.cpu().numpy(), c.lens.cpu().numpy(), c.refs.cpu().numpy()


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------

def rotation(positions, dim):
    f = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(0, dim, 2) / dim)
    f = np.concatenate([f, f], 1)
    return np.cos(f).astype(np.float32), np.sin(f).astype(np.float32)


@pytest.mark.parametrize("x", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,heads,kv", [(64, 6, 2), (128, 8, 8), (256, 3, 1)])
def test_append(x, dtype, dim, heads, kv):
    lens, rows = [0, 17, 40, 3, 31], [1, 20, 0, 7, 1]
    total = [a + b for a, b in zip(lens, rows)]
    g = torch.Generator().manual_seed(dim)
    c = cache_of(dim, total, 16, 20, 4, layers=2, kv=kv, dim=dim, dtype=dtype)
    c.lens.copy_(ints(lens))
    starts = np.cumsum([0] + rows)
    n = sum(rows) + 3  # (three rows behind the last sequence)
    q, k, v = (torch.randn((n, h, dim), generator=g).to(T[x]) for h in (heads, kv, kv))
    depths = torch.randint(0, 5, (n,), generator=g).int()
    cos, sin = rotation(64, dim)
    before = c.k.clone(), c.v.clone()
    for d in (None, depths):
        c.k.copy_(before[0]), c.v.copy_(before[1])
        out = torch.full_like(q, 9.0).to(DEV)
        got = c.append(1, k.to(DEV), v.to(DEV), ints(starts.tolist()), q=q.to(DEV), cos=torch.from_numpy(cos).to(DEV),
                       sin=torch.from_numpy(sin).to(DEV), depths=None if d is None else d.to(DEV), out=out)
        assert got is out and (out[-3:] == 9).all()
        wk, wv = before[0].clone(), before[1].clone()
        table = c.table.cpu().numpy()
        e = torch.finfo(T[x]).eps / 2
        for s in range(len(lens)):
            for j in range(rows[s]):
                r = int(starts[s]) + j
                p = lens[s] + (j if d is None else int(d[r]))
                want = paged.turn(q[r].double().numpy(), cos[p].astype(np.float64), sin[p].astype(np.float64))
                size = np.abs(q[r].double().numpy()) * np.abs(cos[p]) + \
                    np.abs(np.roll(q[r].double().numpy(), dim // 2, -1)) * np.abs(sin[p])
                assert (np.abs(out[r].double().cpu().numpy() - want) <= 2.0 ** -23 * size + e * np.abs(want) + 2.0 ** -25).all()
                t = lens[s] + j
                page, row = int(table[s, t // 16]), t % 16
                want = paged.turn(k[r].double().numpy(), cos[p].astype(np.float64), sin[p].astype(np.float64))
                size = np.abs(k[r].double().numpy()) * np.abs(cos[p]) + \
                    np.abs(np.roll(k[r].double().numpy(), dim // 2, -1)) * np.abs(sin[p])
                have = c.k[1, page, :, row].double().cpu().numpy()
                ec = torch.finfo(T[dtype]).eps / 2
                assert (np.abs(have - want) <= 2.0 ** -23 * size + ec * np.abs(want) + 2.0 ** -25).all()
                wk[1, page, :, row] = c.k[1, page, :, row]
                wv[1, page, :, row] = v[r].float().to(T[dtype]).to(DEV)
        # (nothing else has changed, and values are rounded once)
        assert torch.equal(c.k, wk) and torch.equal(c.v, wv)
        assert torch.equal(c.lens, ints(lens))


def test_append_equals_the_contiguous_form():
    """f32 rows rotate to the same bits as qmm_rope_kv_append_n's."""
    from inference_amd import qmm
    L = qmm.lib()
    heads, kv, dim, n, seq = 8, 2, 128, 5, 32
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn((n, h, dim), generator=g).to(DEV) for h in (heads, kv, kv))
    cos, sin = (torch.from_numpy(t).to(DEV) for t in rotation(seq, dim))
    c = cache_of(3, [16], 16, 4, 1, kv=kv, dim=dim)
    c.lens.fill_(7)
    out = c.append(0, k, v, ints([0, n]), q=q, cos=cos, sin=sin)
    kc, vc = torch.zeros((kv, seq, dim), device=DEV), torch.zeros((kv, seq, dim), device=DEV)
    qq, kk = q.clone(), k.clone()
    qmm._check(L.qmm_rope_kv_append_n(qq.data_ptr(), kk.data_ptr(), v.data_ptr(), heads * dim, kv * dim, kv * dim,
                                      cos.data_ptr(), sin.data_ptr(), 7, n, kc.data_ptr(), vc.data_ptr(), heads, kv,
                                      dim, seq, qmm._stream(DEV)))
    p = int(c.table[0, 0])
    assert torch.equal(out, qq) and torch.equal(c.k[0, p, :, 7:12], kc[:, 7:12]) and torch.equal(c.v[0, p, :, 7:12], vc[:, 7:12])


def test_append_leaves_out_what_has_no_place():
    """Rows past the slot's pages or on a missing one, positions past the tables, odd strides and boundaries, q alone
    rotated in place, no rotation."""
    g = torch.Generator().manual_seed(4)
    c = cache_of(5, [32, 32], 16, 8, 2, kv=1, dim=64)
    c.lens.copy_(ints([30, 10]))
    c.table[1, 0] = 77
    wide = torch.randn((7, 3 * 64 + 5), generator=g).to(DEV)
    q, k, v = wide[:, 1:65], wide[:, 66:130], wide[:, 131:195]
    before = c.k.clone(), c.v.clone()
    assert c.append(0, k, v, ints([0, 4, 7])) is None
    wk, wv = before
    p = int(c.table[0, 1])
    wk[0, p, 0, 14:16], wv[0, p, 0, 14:16] = k[:2], v[:2]
    assert torch.equal(c.k, wk) and torch.equal(c.v, wv)
    # slot 1's entry names no page: nothing written; its rows' q still turn, those past the tables do not
    cos, sin = (torch.from_numpy(t).to(DEV) for t in rotation(32, 64))
    buf = torch.full((7, 64 + 3), 5.0, device=DEV)
    buf[:, 2:66] = q
    c.append(0, k, v, ints([0, 4, 7]), q=buf[:, 2:66], cos=cos, sin=sin, out=buf[:, 2:66])
    assert torch.equal(buf[2:4, 2:66], q[2:4])  # positions 32, 33
    want = paged.turn(q.double().cpu().numpy()[4:], cos[10:13].double().cpu().numpy(), sin[10:13].double().cpu().numpy())
    np.testing.assert_allclose(buf[4:, 2:66].cpu().numpy(), want, rtol=0, atol=2.0 ** -20)
    assert (buf[:, :2] == 5).all() and (buf[:, 66:] == 5).all()
    assert torch.equal(c.v, wv)
    # a depth far outside: nothing is read there
    c.append(0, k, v, ints([0, 4, 7]), q=buf[:, 2:66], cos=cos, sin=sin, depths=ints([2 ** 31 - 1, -2 ** 31] * 3 + [-11]),
             out=buf[:, 2:66])
    torch.cuda.synchronize()


# ---------------------------------------------------------------------------
# fork
# ---------------------------------------------------------------------------

def check_fork(c, parents, keep=None, reserve=0, out=False):
    t, l, r = host(c)
    pools = [c.k.cpu(), c.v.cpu()]
    wt, wl, wr, missing, copies = paged.fork(t, l, r, c.page_size, parents, keep, reserve)
    for src, dst, rows in copies:
        for p in pools:
            p[:, dst, :, :rows] = p[:, src, :, :rows]
    new = tuple(torch.full_like(x, 55) for x in (c.table, c.lens, c.refs)) if out else None
    short = c.fork(ints(parents), keep=None if keep is None else ints(keep), reserve=reserve, out=new)
    gt, gl, gr = [x.cpu().numpy() for x in (new or (c.table, c.lens, c.refs))]
    assert int(short) == missing
    np.testing.assert_array_equal(gt, wt)
    np.testing.assert_array_equal(gl, wl)
    np.testing.assert_array_equal(gr, wr)
    assert torch.equal(c.k.cpu(), pools[0]) and torch.equal(c.v.cpu(), pools[1])
    if out:
        np.testing.assert_array_equal(c.table.cpu().numpy(), t)
    return missing


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("out", [False, True])
def test_fork(dtype, page, out):
    for seed, (lens, parents, keep, reserve) in enumerate((
            ([100, 33, 16, 0], [0, 1, 2, 3], None, 0),
            ([100, 33, 16, 0], [0, 1, 2, 3], None, 1),
            ([100, 33, 16, 0], [0, 0, 0, 0], None, 1),
            ([100, 33, 16, 7], [3, 2, 1, 0], None, 20),
            ([100, 33, 16, 7], [1, 1, -1, 1], None, 5),
            ([100, 33, 128, 7], [2, 2, 0, 0], [-1, 50, 17, 0], 3),
            ([100, 33, 128, 7], [2, 2, 2, 2], [40, 40, 90, 128], 200),
            ([5], [0], [3], 0), ([5], [7], None, 4), ([0], [0], None, 1), ([64], [-1], None, 0))):
        c = cache_of(seed, lens, page, 80, 24, layers=2, dtype=dtype)
        assert check_fork(c, parents, keep, reserve, out) == 0


def test_fork_again_and_again():
    """Random forks of a few beams, one after the other, with rows accepted between: lists and pages all along."""
    rng = np.random.default_rng(6)
    c = cache_of(9, [40, 0, 3, 90, 17, 64], 16, 90, 12, layers=1)
    for step in range(25):
        keep = [int(rng.integers(-1, 120)) for _ in range(6)] if step % 3 == 0 else None
        reserve = int(rng.integers(0, 30))
        check_fork(c, [int(rng.integers(-1, 6)) for _ in range(6)], keep, reserve)
        # every page is counted once for each entry that names it
        t, l, r = host(c)
        want = np.zeros(90, int)
        np.add.at(want, t[t >= 0], 1)
        np.testing.assert_array_equal(r, want)
        n = ints([int(min(reserve, x)) for x in rng.integers(0, 12, 6)])
        alive = torch.from_numpy((t[:, 0] >= 0)).to(DEV)
        c.accept(None, torch.where(alive, n, torch.zeros_like(n)))


def test_fork_pinned_pages_and_readers():
    """A page that somebody else counts, or that another slot reads further on, is copied by all who write it."""
    c = cache_of(1, [40, 90], 16, 30, 8, share=((0, 1, 2),))
    assert check_fork(c, [0, 1], [20, -1], 1) == 0  # slot 0 writes into a page that slot 1 has whole
    c = cache_of(2, [20, 0], 16, 30, 8)
    c.refs[c.table[0, 1].long()] += 1
    assert check_fork(c, [0, 0], None, 1) == 0


def test_fork_without_room():
    """Too few pages, in the pool or in a slot's row: nothing changes, and the number says how many."""
    for out in (False, True):
        c = cache_of(3, [40, 20], 16, 6, 8)
        assert check_fork(c, [0, 0], None, 64, out) > 0
        c = cache_of(3, [40, 20], 16, 20, 4)
        assert check_fork(c, [0, 1], None, 40, out) == 1
    c = cache_of(3, [40, 20], 16, 20, 4)
    assert check_fork(c, [0, 1], None, 30) == 1  # 70 positions: five pages of four
    c = cache_of(3, [40, 20], 16, 5, 4)
    assert check_fork(c, [0, 1], None, 0) == 0
    assert check_fork(c, [1, 1], None, 1) == 0


def test_fork_of_many():
    """More slots than threads of a workgroup, rows of many pages, a large pool."""
    rng = np.random.default_rng(7)
    lens = [int(x) for x in rng.integers(0, 60, 1500)]
    c = cache_of(4, lens, 16, 9000, 8, kv=1)
    assert check_fork(c, [int(x) for x in rng.integers(-1, 1500, 1500)], None, 5) == 0
    lens = [16 * 300 - 5, 100]
    c = cache_of(5, lens, 16, 5000, 700, kv=1)
    assert check_fork(c, [0, 0], [-1, 3001], 3000) == 0


def test_fork_odd_lists():
    """Entries, lengths and parents outside their range are read as none, cut, and none."""
    c = cache_of(6, [40, 20, 33], 16, 12, 4)
    c.table[0, 1] = 99
    c.table[1, 3] = -7
    c.lens[2] = 1000
    check_fork(c, [0, 9, 2], None, 0)
    c = cache_of(6, [40, 20, 33], 16, 12, 4)
    c.lens[1] = -4
    check_fork(c, [1, -2 ** 31, 2 ** 31 - 1], None, 3)


def test_fork_captured():
    """A captured fork, replayed: each replay goes on from the lists as they are."""
    c = cache_of(8, [37, 5, 60, 0], 16, 40, 8, layers=2)
    other = cache_of(8, [37, 5, 60, 0], 16, 40, 8, layers=2)
    parents = ints([2, 0, 0, 1])
    short = torch.empty(1, dtype=torch.int32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.fork(parents, reserve=1, shortage=short)
    for new in ([2, 0, 0, 1], [3, 3, 1, 2], [0, 0, 0, 0], [-1, 1, 1, 2]):
        parents.copy_(ints(new))
        graph.replay()
        torch.cuda.synchronize()
        other.fork(ints(new), reserve=1)
        for a, b in ((c.table, other.table), (c.lens, other.lens), (c.refs, other.refs), (c.k, other.k), (c.v, other.v)):
            assert torch.equal(a, b)
        assert int(short) == 0


# ---------------------------------------------------------------------------
# accept
# ---------------------------------------------------------------------------

def check_accept(c, path, counts, out=False):
    t, l, _ = host(c)
    pools = [c.k.cpu(), c.v.cpu()]
    want = paged.accept([p.view(torch.int16 if p.element_size() == 2 else torch.int32).numpy() for p in pools], t, l,
                        None if path is None else np.array(path), counts)
    new = torch.full_like(c.lens, 55) if out else None
    got = c.accept(None if path is None else ints(path), ints(counts), out=new)
    np.testing.assert_array_equal(got.cpu().numpy(), want)
    if out:
        np.testing.assert_array_equal(c.lens.cpu().numpy(), l)
    assert torch.equal(c.k.cpu(), pools[0]) and torch.equal(c.v.cpu(), pools[1])


@pytest.mark.parametrize("dtype,dim", [("f32", 256), ("bf16", 128), ("f16", 64), ("f32", 64)])
@pytest.mark.parametrize("out", [False, True])
def test_accept(dtype, dim, out):
    lens, room = [0, 30, 16, 60], 40
    path = [[0, 1, 2, 3, 4], [2, 5, 9, 30, 39], [1, 2, 3, 4, 5], [7, 8, 20, 21, 22]]
    for counts in ([5, 5, 5, 5], [0, 1, 2, 3], [99, 4, -3, 5]):
        c = cache_of(dim, [n + room for n in lens], 16, 40, 8, layers=3, dim=dim, dtype=dtype)
        c.lens.copy_(ints(lens))
        check_accept(c, path, counts, out)
    c = cache_of(dim, [n + room for n in lens], 16, 40, 8, layers=1, dim=dim, dtype=dtype)
    c.lens.copy_(ints(lens))
    check_accept(c, None, [3, 0, 40, 1], out)


def test_accept_long_paths():
    """Paths over several pages, longer than a workgroup's threads have columns."""
    rng = np.random.default_rng(1)
    c = cache_of(1, [700, 600], 16, 100, 60, layers=2)
    c.lens.copy_(ints([100, 3]))
    path = [sorted(rng.choice(600, 300, replace=False).tolist()) for _ in range(2)]
    check_accept(c, path, [300, 251])


def test_accept_into_the_counts():
    """The new lengths over the counts; over part of them or of a path: refused."""
    c = cache_of(3, [60] * 4, 16, 40, 4)
    c.lens.copy_(ints([10, 20, 5, 3]))
    path, both = ints([[1, 3, 9, 11]] * 4), ints([2, 4, 0, 3, 0])
    counts = both[:4]
    c.accept(path, counts, out=counts)
    assert both.tolist() == [12, 24, 5, 6, 0] and c.lens.tolist() == [10, 20, 5, 3]
    for bad in (both[1:], path.view(-1)[:4], path.view(-1)[12:]):
        with pytest.raises(QmmError):
            c.accept(path, counts, out=bad)


def test_accept_paths_that_end_early():
    """Entries that do not rise, lie below 0, or outside the slot's pages end a path."""
    path = [[3, 3, 4, 5], [5, 2, 8, 9], [-1, 0, 1, 2], [0, 9, 90, 91], [2, 4, 2 ** 31 - 1, 5], [1, 40, 41, 42]]
    c = cache_of(2, [60] * 6, 16, 40, 4)
    c.lens.copy_(ints([10, 20, 5, 3, 4, 15]))
    c.table[5, 3] = -1
    check_accept(c, path, [4] * 6)
    c = cache_of(2, [60] * 6, 16, 40, 4)
    c.lens.copy_(ints([10, 63, 64, 2 ** 31 - 1, -9, 15]))
    c.table[0, 1] = 4000
    check_accept(c, None, [4, 4, 4, 2 ** 31 - 1, 2 ** 31 - 1, 100])


# ---------------------------------------------------------------------------
# compact
# ---------------------------------------------------------------------------

def check_compact(c, out=False):
    t, _, r = host(c)
    pools = [c.k.cpu(), c.v.cpu()]
    wt, wr, used, moves = paged.compact(t, r)
    for a, b in moves:
        for p in pools:
            p[:, b] = p[:, a]
    new = (torch.full_like(c.table, 55), torch.full_like(c.refs, 55)) if out else None
    got = c.compact(out=new)
    gt, gr = [x.cpu().numpy() for x in (new or (c.table, c.refs))]
    assert int(got) == used
    np.testing.assert_array_equal(gt, wt)
    np.testing.assert_array_equal(gr, wr)
    assert torch.equal(c.k.cpu(), pools[0]) and torch.equal(c.v.cpu(), pools[1])


@pytest.mark.parametrize("out", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_compact(out, dtype):
    for seed, (lens, pages) in enumerate((([100, 0, 33], 40), ([0], 1), ([5], 1), ([0, 0], 70), ([200, 300, 10], 33),
                                          ([500] * 20, 1500), ([16] * 1024, 2049), ([160], 4000))):
        c = cache_of(seed, lens, 16, pages, 40, layers=2, kv=1, dtype=dtype)
        check_compact(c, out)
    c = cache_of(3, [90, 90, 20], 16, 50, 8, share=((0, 1, 4),))
    c.refs[int(torch.nonzero(c.refs == 0)[-1])] = 1  # (a page that only its owner knows)
    c.table[2, 7] = 4444
    check_compact(c, out)
    check_compact(c, out)
