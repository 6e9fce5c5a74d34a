"""The paged cache's operators and the beam selection at the ends of their documented ranges."""
import numpy as np
import pytest
import torch

from inference_amd import PagedKVCache, beam_select
from oracle import paged

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.empty_cache()


def test_a_sequence_of_the_most_positions():
    """2^28 positions on pages of 1024: the last row, which sees four keys far apart above all others."""
    page, pages, dim = 1024, 1 << 18, 64
    n = page * pages
    k = torch.empty((1, pages, 1, page, dim), dtype=torch.bfloat16, device=DEV).normal_()
    v = torch.empty_like(k).normal_()
    table = (torch.arange(pages, device=DEV).flip(0) ^ 5).int().view(1, pages)
    c = PagedKVCache(k, v, table, ints([n - 1]), torch.ones(pages, dtype=torch.int32, device=DEV))
    g = torch.Generator(device=DEV).manual_seed(2)
    q = torch.randn((1, 2, dim), device=DEV, generator=g).bfloat16()
    new = torch.randn((1, 1, dim), device=DEV, generator=g).bfloat16()
    c.append(0, q[:, :1], new, ints([0, 1]))
    at = [0, 1 << 27, n - 1030, n - 1]  # (the last is the appended row)
    where = [(int(table[0, t // page]), t % page) for t in at]
    for p, r in where[:3]:
        k[0, p, 0, r] = q[0, 0]
    q = (q.float() * torch.tensor([6.0, 0.0], device=DEV)[:, None]).bfloat16()
    got = c.attention(0, q, ints([0, 1])).double()[0]
    # the first head: scores of 6 |q|^2 / 8 against a standard deviation of 6 |q| / 8; 2^28 others at six of those hold
    # e^(19.4 + 18 |q|^2 / 64) against 4 e^(48 |q|^2 / 64)
    keys, values = (torch.stack([x[0, p, 0, r] for p, r in where]).double() for x in (k, v))
    size = float(q[0, 0].double().square().sum()) / 36
    rest = np.exp(np.log(2.0 ** 28) + 18 * size / 64 - 48 * size / 64) / 4
    assert rest < 1e-2  # (the tolerance counts it)
    w = torch.softmax(keys @ q[0, 0].double() * dim ** -0.5, 0)
    assert float((got[0] - w @ values).abs().max()) <= 2 * rest * 6 + 2.0 ** -7
    # the second head's weights are equal: the mean of the values, of 2^28 within 6 / 2^14 of 0
    assert float(got[1].abs().max()) <= 6 * 2.0 ** -14 + 2.0 ** -12
    # a path over the end of the slot, and one up to it
    c.lens.fill_(n - 4)
    assert c.accept(ints([[1, 3, 4]]), ints([3]), out=ints([0])).tolist() == [n - 2]
    assert c.accept(None, ints([9]), out=ints([0])).tolist() == [n]


def test_tables_of_the_most_entries():
    """256 slots of 2^20 pages, 2^20 pages in the pool: a fork whose lists are long, a packing, and the rows behind."""
    slots, wide, pages, page = 256, 1 << 20, 1 << 20, 16
    c = PagedKVCache.empty(1, pages, 1, page, 64, slots, wide, torch.bfloat16, DEV)
    g = torch.Generator(device=DEV).manual_seed(3)
    ids = torch.randperm(pages, device=DEV, generator=g).int()
    long = 900000
    c.table[7, :long] = ids[:long]
    c.table[255, :3] = ids[long:long + 3]
    c.refs[ids[:long + 3].long()] = 1
    c.lens[7], c.lens[255] = long * page - 5, 40
    rows = {s: torch.randn((3, 64), device=DEV, generator=g).bfloat16() for s in (7, 255)}
    for s in rows:  # the last three positions of each
        for i in range(3):
            t = int(c.lens[s]) - 3 + i
            c.k[0, int(c.table[s, t // page]), 0, t % page] = rows[s][i]
    parents = torch.full((slots,), -1, dtype=torch.int32, device=DEV)
    parents[7], parents[100], parents[255], parents[0] = 7, 7, 255, 255
    keep = torch.full((slots,), -1, dtype=torch.int32, device=DEV)
    keep[100] = 33
    assert int(c.fork(parents, keep=keep, reserve=20)) == 0
    assert c.lens[[0, 7, 100, 255]].tolist() == [40, long * page - 5, 33, 40]
    want = torch.zeros(pages, dtype=torch.int64, device=DEV)
    named = c.table[c.table >= 0].long()
    want.scatter_add_(0, named, torch.ones_like(named))
    assert torch.equal(want, c.refs.long())
    free = torch.ones(pages, dtype=torch.bool, device=DEV)
    free[ids[:long + 3].long()] = False
    low = torch.nonzero(free).flatten()[:5].tolist()
    # slot 0 keeps its page, 7 reserves one (15 positions past 11), 100 copies and reserves one, 255 copies and reserves one
    assert int(c.table[0, 2]) == int(ids[long + 2]) and int(c.table[0, 3]) == low[0]
    for again in range(2):
        for s, r in ((0, rows[255]), (7, rows[7]), (255, rows[255])):
            for i in range(3):
                t = int(c.lens[s]) - 3 + i
                assert torch.equal(c.k[0, int(c.table[s, t // page]), 0, t % page], r[i])
        if again == 0:
            used = int(c.compact())
            assert used == int((want > 0).sum()) and int(c.refs[used:].sum()) == 0 and int(c.table.max()) == used - 1


@pytest.mark.parametrize("batch,beams,vocab,count", [(65535, 1, 3, 2), (1023, 64, 2, 128), (21845, 3, 5, 7),
                                                     (1, 64, 2 ** 20, 128)])
def test_beam_searches_of_the_largest_sizes(batch, beams, vocab, count):
    g = torch.Generator().manual_seed(beams)
    lg = (torch.randn((batch * beams, vocab), generator=g) * 2).bfloat16()
    sc = -torch.rand(batch * beams, generator=g) * 9
    got = [x.cpu().numpy() for x in beam_select(lg.to(DEV), sc.to(DEV), beams, count)]
    for part in ([0, batch // 2, batch - 1] if batch > 1 else [0]):
        rows = slice(part * beams, (part + 1) * beams)
        want = paged.beam(lg[rows].float().numpy(), sc[rows].numpy(), beams, count)
        np.testing.assert_array_equal(got[0][part], want[0][0])
        np.testing.assert_array_equal(got[1][part], np.where(want[1][0] < 0, -1, want[1][0] + part * beams))


def test_the_most_slots_heads_and_layers():
    """4096 slots; 256 kv heads; 1024 layers."""
    n = 4096
    c = PagedKVCache.empty(1, n, 1, 16, 64, n, 1, torch.float32, DEV)
    c.table.copy_(torch.randperm(n, device=DEV).int()[:, None])
    c.refs.fill_(1)
    kv = torch.randn((n, 1, 64), device=DEV)
    starts = torch.arange(n + 1, dtype=torch.int32, device=DEV)
    c.append(0, kv, kv, starts)
    assert torch.equal(c.attention(0, kv, starts, max_rows=1), kv)  # (one position: its own value)
    assert int(c.accept(None, torch.ones(n, dtype=torch.int32, device=DEV)).sum()) == n
    parents = torch.arange(n, device=DEV).flip(0).int()
    assert int(c.fork(parents)) == 0
    assert torch.equal(c.k[0, c.table[:, 0].long(), 0, 0], kv[:, 0].flip(0))
    c = PagedKVCache.empty(1, 4, 256, 16, 64, 2, 2, torch.float16, DEV)
    assert int(c.fork(ints([0, 1]), reserve=0)) == 0
    c.table.copy_(ints([[3, 1], [0, 2]]))
    kv, q = torch.randn((2, 256, 64), device=DEV).half(), torch.randn((2, 1024, 64), device=DEV).half()
    c.append(0, kv, kv, ints([0, 1, 2]))
    got = c.attention(0, q, ints([0, 1, 2]))
    assert torch.equal(got, kv[:, :, None].expand(2, 256, 4, 64).reshape(2, 1024, 64))
    c = PagedKVCache.empty(1024, 3, 1, 16, 64, 1, 3, torch.bfloat16, DEV)
    c.table.copy_(ints([[2, 0, 1]]))
    c.refs.fill_(1)
    c.lens.fill_(15)
    c.k.normal_(), c.v.normal_()
    k, v = c.k.clone(), c.v.clone()
    assert c.accept(ints([[2, 4]]), ints([2])).tolist() == [17]
    for was, now in ((k, c.k), (v, c.v)):
        was[:, 2, :, 15], was[:, 0, :, 0] = was[:, 0, :, 1].clone(), was[:, 0, :, 3].clone()
        assert torch.equal(was, now)
