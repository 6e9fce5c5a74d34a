"""A beam search's selection and the reordering of its rows. Tokens and parents have to be the definition's; a score
is off by the exponentials' 2^-30 and one rounding to f32."""
import numpy as np
import pytest
import torch

from inference_amd import beam_select, reorder_rows
from oracle import paged

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def check(lg, scores, beams, count, finished=None, eos=-1, dev_logits=None):
    f = None if finished is None else torch.tensor(finished, dtype=torch.int32, device=DEV)
    got = beam_select(lg.to(DEV) if dev_logits is None else dev_logits, scores.to(DEV), beams, count, finished=f, eos=eos)
    want = paged.beam(lg.float().numpy(), scores.numpy(), beams, count, finished, eos)
    tokens, parents, sc, done = (x.cpu().numpy() for x in got)
    np.testing.assert_array_equal(tokens, want[0])
    np.testing.assert_array_equal(parents, want[1])
    np.testing.assert_array_equal(done, want[3])
    fin = np.isfinite(want[2])
    np.testing.assert_array_equal(sc[~fin], want[2][~fin].astype(np.float32))
    assert (np.abs(sc[fin] - want[2][fin]) <= 2.0 ** -24 * np.abs(want[2][fin]) + 2.0 ** -29).all()
    return tokens


def inputs(seed, rows, vocab, x, std=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((rows, vocab), generator=g) * std).to(T[x]), -torch.rand(rows, generator=g) * 9 - 1


@pytest.mark.parametrize("x", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 3, 100, 4095, 4096, 4097, 32001, 128256])
def test_select(x, vocab):
    for batch, beams, count in ((1, 1, 1), (1, 4, 4), (3, 5, 10), (2, 16, 32)):
        lg, sc = inputs(vocab + beams, batch * beams, vocab, x)
        check(lg, sc, beams, count)


def test_many_beams_and_lists():
    for beams, count, vocab in ((64, 128, 5000), (64, 64, 100), (2, 128, 40), (1, 128, 20000), (33, 7, 9001)):
        lg, sc = inputs(beams, 2 * beams, vocab, "f32")
        check(lg, sc, beams, count)
    lg, sc = inputs(1, 3, 2 ** 20, "bf16")
    check(lg, sc, 3, 9)


def test_ties():
    """Equal logits: the lower token; equal beams: the lower beam; a whole row of one value; the best of a row next to
    each other in one thread's logits."""
    g = torch.Generator().manual_seed(1)
    lg = torch.randint(-3, 3, (6, 9000), generator=g).float()
    sc = torch.full((6,), -2.0)
    check(lg, sc, 3, 64)
    check(torch.zeros(4, 10000), torch.full((4,), -1.0), 4, 128)
    lg = torch.zeros(2, 9000)
    lg[:, 4000:4130] = 5.0 + torch.arange(130) / 1000
    check(lg, torch.tensor([-1.0, -1.0]), 2, 128)
    lg = torch.randn((1, 8192), generator=g).sort(descending=True).values
    check(lg, torch.zeros(1), 1, 128)
    check(-torch.zeros(2, 50), torch.zeros(2), 2, 60)  # -0 and 0 are one value
    lg = torch.zeros(1, 50)
    lg[0, ::2] = -0.0
    check(lg, torch.zeros(1), 1, 50)


def test_close_scores_of_different_beams():
    """Scores that f32 sums would tie or order the other way."""
    lg = torch.full((2, 3000), -60.0)
    lg[0, 7], lg[0, 8] = 5.0, 4.9999995
    lg[1, 2], lg[1, 3] = 5.0, 4.999999
    check(lg, torch.tensor([-16.0, -16.000001]), 2, 4)
    check(lg, torch.tensor([-16.000001, -16.0]), 2, 4)


def test_nothing_to_choose():
    """-inf, NaN and +inf logits, beams that have not begun, rows without a token: what is missing is -1."""
    inf, nan = float("inf"), float("nan")
    lg, sc = inputs(3, 6, 5000, "f32")
    lg[0, :] = -inf
    lg[1, 10:] = nan
    lg[2, 5] = inf
    lg[3, :4999] = -inf
    check(lg, sc, 6, 20)
    check(lg, sc, 2, 7)
    sc2 = torch.tensor([-1.0, -inf, nan, -inf, -2.0, -inf])
    check(lg, sc2, 3, 9)
    check(lg, torch.full((6,), -inf), 2, 5)
    assert (check(torch.full((4, 300), nan), torch.zeros(4), 2, 3) == -1).all()
    check(torch.full((2, 5), -inf).index_fill(1, torch.tensor([3]), 0.5), torch.zeros(2), 2, 6)


def test_finished_beams():
    """A finished beam goes on as its end, at its score; its logits (NaN here) are not looked at."""
    for x in ("f32", "bf16"):
        lg, sc = inputs(4, 8, 5000, x)
        lg[1] = float("nan")
        lg[6] = 1e30
        check(lg, sc, 4, 8, finished=[0, 1, 0, 0, 0, 0, 3, 0], eos=2)
        check(lg, sc, 4, 4, finished=[1] * 8, eos=4999)
        lg[:, 2] += 9
        tokens = check(lg, sc, 4, 8, eos=2)
        assert (tokens == 2).any()
    check(lg, torch.tensor([-1.0, float("-inf")] * 4), 2, 3, finished=[0, 1] * 4, eos=0)


def test_strides_and_boundaries():
    lg, sc = inputs(5, 6, 5001, "bf16")
    for off, pad in ((0, 3), (1, 0), (1, 4), (4, 4), (3, 7)):
        wide = torch.full((6, 5001 + off + pad), 1e4, dtype=torch.bfloat16, device=DEV)
        wide[:, off:off + 5001] = lg.to(DEV)
        check(lg, sc, 3, 6, dev_logits=wide[:, off:off + 5001])
    check(lg, sc, 3, 6, dev_logits=lg.to(DEV).t().contiguous().t())


def test_streams_and_captures():
    lg, sc = inputs(6, 8, 20000, "f32")
    lg, sc = lg.to(DEV), sc.to(DEV)
    want = beam_select(lg, sc, 4, 8)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(beam_select(lg, sc, 4, 8))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = beam_select(lg, sc, 4, 8)
        moved = reorder_rows(lg, out[1].view(-1))
    for step in range(4):
        lg.mul_(-1.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, beam_select(lg, sc, 4, 8)))
        assert torch.equal(moved, lg[out[1].view(-1).long()])


@pytest.mark.parametrize("shape", [(7, 5), (7, 4, 3), (9, 1024), (3, 1), (5, 70001), (4, 0), (6,)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.bfloat16, torch.uint8, torch.float64])
def test_reorder(shape, dtype):
    g = torch.Generator().manual_seed(1)
    src = torch.randint(0, 200, shape, generator=g).to(dtype).to(DEV)
    index = torch.tensor([2, 0, 0, -1, shape[0] - 1, shape[0], 2 ** 31 - 1, 1, -2 ** 31], dtype=torch.int32)
    out = torch.full((9, *shape[1:]), 77, dtype=dtype, device=DEV)
    want = out.clone()
    for i, p in enumerate(index.tolist()):
        if 0 <= p < shape[0]:
            want[i] = src[p]
    assert reorder_rows(src, index.to(DEV), out=out) is out
    assert torch.equal(out, want)
    good = index[:3].to(DEV)
    assert torch.equal(reorder_rows(src, good), src[good.long()])


def test_reorder_strides():
    base = torch.arange(8 * 40, dtype=torch.int16, device=DEV).view(8, 40)
    out = torch.zeros((4, 21), dtype=torch.int16, device=DEV)
    index = torch.tensor([3, 3, 7, 0], dtype=torch.int32, device=DEV)
    for off in (0, 1, 8):
        reorder_rows(base[:, off:off + 16], index, out=out[:, 2:18])
        assert torch.equal(out[:, 2:18], base[index.long(), off:off + 16]) and not out[:, :2].any() and not out[:, 18:].any()
    assert torch.equal(reorder_rows(base.t(), index), base.t()[index.long()])
    assert reorder_rows(base, index[:0]).shape == (0, 40)


def test_scores_below_the_range_of_f32():
    """Lowest values beside an infinite logit, or under a lowest score, have 64-bit scores below f32's: continuations all
    the same, in both ways that a search's lists are merged (the last size here has more entries than are ranked). Their
    f32 scores round to -inf."""
    low, inf = torch.finfo(torch.float32).min, float("inf")
    below = 0
    for beams, count, vocab in ((1, 2, 2), (1, 5, 5000), (2, 9, 5000), (3, 64, 70), (1, 128, 128256)):
        lg = torch.full((2 * beams, vocab), low)
        lg[0, vocab // 2] = inf
        lg[beams:, :2] = torch.tensor([1.0, 2.0])
        for score in (-1.0, low):
            sc = torch.full((2 * beams,), score)
            sc[0] = -2.0
            tokens, parents, out, _ = (x.cpu().numpy() for x in beam_select(lg.to(DEV), sc.to(DEV), beams, count))
            want = paged.beam(lg.numpy(), sc.numpy(), beams, count)
            np.testing.assert_array_equal(tokens, want[0])
            np.testing.assert_array_equal(parents, want[1])
            with np.errstate(over="ignore"):
                near = want[2].astype(np.float32)
            below += int((np.isneginf(near) & (tokens >= 0)).any())
            np.testing.assert_array_equal(np.isneginf(out), np.isneginf(near))
            fine = np.isfinite(near)
            assert (np.abs(out[fine] - want[2][fine]) <= 2.0 ** -24 * np.abs(want[2][fine]) + 2.0 ** -29).all()
    assert below >= 5


def test_certain_tokens():
    """A token of probability one leaves a score as it is, bit for bit: it ties with a beam that has ended."""
    for vocab in (1, 300, 9000):
        for value in (0.0, 5.5, -3.25, 1e30):
            lg = torch.full((4, vocab), -float("inf"))
            lg[:, vocab // 3] = value
            sc = torch.tensor([-1.0, -1.0, -0.3, 0.0])
            out = beam_select(lg.to(DEV), sc.to(DEV), 1, 1)[2]
            assert torch.equal(out.cpu().view(-1), sc)
            check(lg, sc, 2, 2, finished=[1, 0, 0, 0], eos=0)
            check(lg, sc, 2, 2, finished=[0, 1, 0, 0], eos=0)
            check(lg, torch.full((4,), -2.0), 4, 4, finished=[0, 1, 0, 1], eos=0)
            check(lg, torch.full((4,), 0.0), 4, 3, finished=[1, 0, 0, 1], eos=0)


def test_scores_of_minus_zero():
    """-0 and 0 are one score: the lower beam is first, whichever of them it has."""
    lg, _ = inputs(7, 8, 300, "f32")
    zero = torch.tensor([-0.0, 0.0, -0.0, 0.0])
    for sc in (zero, -zero):
        for count in (1, 2, 3, 4):
            check(lg[:4], sc, 4, count, finished=[1] * 4, eos=3)
            check(lg[:4], sc, 2, count, finished=[1] * 4, eos=0)
    single = torch.zeros(4, 1)  # (one token, of probability one: scores stay as they are)
    check(single, zero, 4, 2)
    check(single, zero, 4, 3, finished=[1, 0, 0, 1], eos=0)


def test_results_in_place():
    """The C entry point's scores and ends in place, where a search has as many continuations as beams; elsewhere: refused."""
    from inference_amd import qmm
    L = qmm.lib()
    for batch, beams, count in ((5, 4, 4), (1, 1, 1), (3, 64, 64), (2, 3, 4)):
        rows = batch * beams
        lg, sc = inputs(8 + beams, rows, 5000, "f32")
        end = torch.zeros(rows, dtype=torch.int32)
        end[::3] = 1
        lg, sc, end = lg.to(DEV), sc.to(DEV), end.to(DEV)
        want = beam_select(lg, sc, beams, count, finished=end, eos=7)
        size = L.qmm_beam_select_workspace_size(batch, beams, 5000, count)
        ws = torch.empty(size, dtype=torch.uint8, device=DEV)
        tokens, parents = torch.empty((2, batch, count), dtype=torch.int32, device=DEV)
        rc = L.qmm_beam_select(lg.data_ptr(), 0, 5000, batch, beams, 5000, sc.data_ptr(), end.data_ptr(), 7, count,
                               tokens.data_ptr(), parents.data_ptr(), sc.data_ptr(), end.data_ptr(), ws.data_ptr(), size,
                               qmm._stream(DEV))
        assert (rc == 0) == (count == beams)
        if rc == 0:
            for a, b in zip(want, (tokens, parents, sc, end)):
                assert torch.equal(a.view(-1), b.view(-1))
