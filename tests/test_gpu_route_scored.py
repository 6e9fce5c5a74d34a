"""Scored routing (softmax or sigmoid, bias, groups, scaled weights) against its rules in 64 bits (oracle/mx.py):
the same lists, weights to f32 rounding."""
import numpy as np
import pytest
import torch

from inference_amd import QmmError, moe_route
from oracle import mx

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def run(lg, k, bias=None, **kw):
    b = None if bias is None else torch.from_numpy(np.asarray(bias, np.float32)).to(DEV)
    got = [v.cpu().numpy() for v in moe_route(torch.from_numpy(lg).to(DEV), k, score=kw.pop("score", "softmax"), bias=b,
                                              renormalize=kw.pop("renormalize", True),
                                              routed_scaling_factor=kw.pop("scale", 1.0), **kw)]
    return got


def check(lg, k, bias=None, **kw):
    want = mx.lists(*mx.route(lg, k, bias=bias, **kw), lg.shape[1])
    got = run(lg, k, bias, **kw)
    for i in (0, 1, 2, 4):
        np.testing.assert_array_equal(got[i], want[i])
    # one rounding to f32 of a 64-bit value
    assert (np.abs(got[3] - want[3]) <= 2.0 ** -23 * np.abs(want[3]) + 1e-45).all()


CASES = [(1, 1, 1, 1, 1, 1), (1, 8, 2, 1, 1, 1), (5, 8, 8, 1, 1, 1), (16, 64, 6, 8, 3, 1), (17, 64, 6, 8, 3, 2),
         (33, 60, 4, 4, 2, 2), (64, 96, 8, 8, 4, 2), (65, 128, 1, 64, 1, 2), (100, 160, 8, 8, 5, 1), (257, 256, 8, 8, 4, 2),
         (12, 300, 10, 10, 4, 2), (9, 100, 4, 4, 2, 2), (16, 256, 8, 1, 1, 1), (8, 100, 4, 4, 2, 2),
         (4, 256, 8, 8, 4, 2), (1, 300, 10, 10, 4, 2), (70, 1024, 32, 64, 3, 2),
         (1000, 16, 4, 1, 1, 1), (3, 7, 3, 7, 3, 1)]


@pytest.mark.parametrize("t,n,k,groups,kept,top", CASES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("renorm", [False, True])
def test_lists(t, n, k, groups, kept, top, score, bias, renorm):
    rng = np.random.default_rng(t * n + k)
    lg = (rng.standard_normal((t, n)) * 2).astype(np.float32)
    b = (rng.standard_normal(n) * 0.2).astype(np.float32) if bias else None
    check(lg, k, b, score=score, groups=groups, topk_groups=kept, group_top=top, renormalize=renorm, scale=2.5)


@pytest.mark.parametrize("t", [2, 40])
@pytest.mark.parametrize("n", [8, 130, 256, 520])
def test_ties_go_to_the_lower_expert(t, n):
    rng = np.random.default_rng(n)
    lg = rng.integers(0, 2, (t, n)).astype(np.float32)
    lg[0] = 0
    for score in ("softmax", "sigmoid"):
        check(lg, 6, score=score)
        check(lg, 2, score=score, groups=2, topk_groups=1, group_top=2)


def test_close_scores_are_ordered_as_the_exact_ones():
    """Experts whose scores differ by less than an f32 step: the logits' order decides."""
    base = np.float32(12.0)
    lg = np.full((20, 64), base, np.float32)
    rng = np.random.default_rng(3)
    for row in lg:
        row[:] = base + np.float32(2.0 ** -20) * rng.permutation(64).astype(np.float32)
    check(lg, 6, score="sigmoid")
    check(lg, 6, score="softmax")


@pytest.mark.parametrize("t", [8, 24])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_infinities_and_nan(t, score):
    rng = np.random.default_rng(t)
    n, inf = 16, np.inf
    lg = rng.standard_normal((t, n)).astype(np.float32)
    lg[0] = -inf                       # nothing left: the lowest experts, weights 0
    lg[1, 3:] = -inf                   # fewer finite logits than experts asked for
    lg[2, 5] = inf
    lg[3, 5] = lg[3, 9] = inf
    lg[4, 2] = np.nan
    lg[5] = np.nan
    lg[6] = np.finfo(np.float32).min   # a mask of the type's lowest value everywhere
    lg[7, 1:] = np.finfo(np.float32).min
    for kw in ({}, dict(renormalize=False, scale=3.0), dict(groups=4, topk_groups=2, group_top=2)):
        check(lg, 4, score=score, **kw)
        assert np.isfinite(run(lg, 4, score=score, **kw)[3]).all()
    bias = rng.standard_normal(n).astype(np.float32) * 0.1
    bias[1], bias[2], bias[3], bias[7] = np.nan, -inf, inf, inf
    check(lg, 4, bias, score=score)
    check(lg, 6, bias, score=score, groups=4, topk_groups=2, group_top=2)


def test_many_tokens():
    rng = np.random.default_rng(9)
    for t, n, k in ((8192, 8, 2), (4096, 256, 8), (3000, 40, 5)):
        check((rng.standard_normal((t, n)) * 2).astype(np.float32), k, score="sigmoid")


def test_largest():
    """65536 tokens: the counts and places are a permutation, experts in order, tokens in order within them."""
    t, n, k = 65536, 64, 4
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    counts, offsets, ptok, pw, tp = moe_route(torch.randn(t, n, generator=g, device=DEV), k, score="softmax")
    assert int(offsets[-1]) == t * k and torch.equal(offsets[1:] - offsets[:-1], counts)
    assert torch.equal(torch.sort(tp.long()).values, torch.arange(t * k, device=DEV))
    owner = torch.arange(t, device=DEV).repeat_interleave(k)
    assert torch.equal(ptok[tp.long()].long(), owner)
    expert = torch.bucketize(torch.arange(t * k, device=DEV), offsets[1:].long(), right=True)
    inside = expert[1:] == expert[:-1]
    assert (ptok[1:][inside] > ptok[:-1][inside]).all()
    torch.testing.assert_close(torch.zeros(t, device=DEV).index_add_(0, ptok.long(), pw), torch.ones(t, device=DEV),
                               rtol=4 * 2.0 ** -23, atol=0)
    with pytest.raises(QmmError, match="routing limits"):
        moe_route(torch.zeros(65537, 8, device=DEV), 2, score="softmax")


def test_types_and_strides():
    rng = np.random.default_rng(5)
    lg = (rng.standard_normal((40, 32)) * 2).astype(np.float32)
    ref = run(lg, 4, score="sigmoid")
    d = torch.from_numpy(lg).to(DEV)
    wide = torch.zeros(40, 64, device=DEV)
    wide[:, 1::2] = d
    for src in (wide[:, 1::2], d.t().contiguous().t(), d.double()):
        for a, b in zip(moe_route(src, 4, score="sigmoid"), ref):
            np.testing.assert_array_equal(a.cpu().numpy(), b)
    h = d.bfloat16()
    want = mx.lists(*mx.route(h.float().cpu().numpy(), 4, score="sigmoid"), 32)
    np.testing.assert_array_equal(moe_route(h, 4, score="sigmoid")[2].cpu().numpy(), want[2])


def test_graph_replays():
    for t in (4, 100):
        xs = [torch.randn(t, 64, device=DEV) for _ in range(3)]
        kw = dict(score="sigmoid", groups=8, topk_groups=4, group_top=2, bias=torch.randn(64, device=DEV) * 0.1)
        want = [moe_route(x, 6, **kw) for x in xs]
        x = xs[0].clone()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = moe_route(x, 6, **kw)
        for i in (1, 2, 0):
            x.copy_(xs[i])
            g.replay()
            moe_route(xs[(i + 1) % 3], 6, **kw)
            torch.cuda.synchronize()
            for a, b in zip(out, want[i]):
                assert torch.equal(a, b)


@pytest.mark.parametrize("n", [16, 100, 256, 300])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("t", [1, 40])
def test_close_choices_of_either_sign(n, sign, t):
    """Choices that differ beyond their first 21 significant bits alone, above and below zero, some of them equal."""
    rng = np.random.default_rng(n)
    bias = np.float32(sign * 2) + np.float32(sign * 2.0 ** -22) * rng.integers(0, 8, n).astype(np.float32)
    lg = np.full((t, n), -60, np.float32)
    lg[:, rng.integers(0, n)] = -59.5
    check(lg, 6, bias, score="sigmoid")
    check(lg, 6, bias, score="sigmoid", groups=2, topk_groups=1, group_top=2)
