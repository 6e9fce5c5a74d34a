"""MXFP4 FFNs over inner widths of several chunks, closely enough to see a lost digit; products against rows that are
not rounded to digits.

The inner rows a = silu(g) * u of the reference are in 64 bits, the kernel's from sums in f32, off by d at most:
|silu'(g)| <= 1.1 times g's bound, |silu(g)| times u's, and 2^-20 of a for silu's own f32 steps. A value d from
another falls on the other side of a digit border with probability d / s at most, s the digits' step (2^-6 of the
block's scale at most), and then moves by s; where it does not fall apart it is the same. The weights of the down
product are independent of that and of mean zero, so the moves add up to a variance of sum(w^2 s d) over the outputs,
whatever their signs. The norm of the error over all outputs is held to twice the standard deviation, and the f32
additions of the down product on top. Losing the second digits moves every value, by up to 2^-2 of the block's scale."""
import ctypes

import numpy as np
import pytest
import torch

from inference_amd import GgmlDType, QMatMul, QTensor, moe_ffn, qmm
from oracle import mx

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
MX = GgmlDType.MXFP4


def randn(seed, *shape, std=1.0):
    return (np.random.default_rng(seed).standard_normal(shape) * std).astype(np.float32)


def weight(seed, n, k, std):
    return QTensor.from_ggml(mx.to_mxfp4(randn(seed, n, k, std=std)).reshape(-1), MX, (n, k), device=DEV)


def f64(a):
    return torch.from_numpy(np.asarray(a, np.float64)).to(DEV)


def ffn(x, g, u, d):
    """(output, variance bound, f32 sums' bound, the output with the second digits lost), f64."""
    xv = f64(mx.digit_values(x))

    def part(w):
        return xv @ w.t(), (w.shape[1] / 32 + 34) * 2.0 ** -23 * (xv.abs() @ w.abs().t())

    (a, da), (b, db) = part(g), part(u)
    silu = a / (1 + torch.exp(-a))
    h = silu * b
    off = 1.1 * da * (b.abs() + db) + silu.abs() * db + 2.0 ** -20 * h.abs()
    e, hi, _ = mx.digits(h.cpu().numpy())
    scale = np.exp2(e - 127.0)[..., None]
    step = f64(np.broadcast_to(scale * 2.0 ** -6, hi.shape).reshape(h.shape))
    one = f64((mx.E2M3[hi & 31] * np.where(hi & 32, -1, 1) * scale).reshape(h.shape))
    hv = f64(mx.digit_values(h.cpu().numpy()))
    f32 = (d.shape[1] / 32 + 34) * 2.0 ** -23 * (hv.abs() @ d.abs().t())
    return hv @ d.t(), (step * off) @ (d * d).t(), f32, one @ d.t()


def close(got, want, var, f32, one):
    tol = 2 * float(var.sum().sqrt()) + float(f32.norm()) + 2.0 ** -23 * float(want.norm())
    err = float((got - want).norm())
    assert err <= tol, (err / float(want.norm()), tol / float(want.norm()))
    assert 4 * tol <= float((one - want).norm())  # (the bound is close enough for what it is there to see)


@pytest.mark.parametrize("m,h,f", [(1, 1056, 4128), (2, 320, 8224), (7, 544, 2080), (40, 288, 2080), (200, 160, 4128),
                                   (300, 544, 1056)])
def test_ffn(m, h, f):
    wg, wu, wd = weight(1, f, h, h ** -0.5), weight(2, f, h, h ** -0.5), weight(3, h, f, f ** -0.5)
    x = randn(m, m, h)
    want = ffn(x, *(w.dequantize().double() for w in (wg, wu, wd)))
    L = qmm.lib()
    xd, y = torch.from_numpy(x).to(DEV), torch.empty(m, h, device=DEV)
    ws = torch.empty(L.qmm_ffn_workspace_size(wg.handle, wu.handle, wd.handle, m, 0), dtype=torch.uint8, device=DEV)
    qmm._check(L.qmm_ffn(wg.handle, wu.handle, wd.handle, xd.data_ptr(), m, h, None, 0.0, 0, y.data_ptr(), h,
                         ws.data_ptr(), ws.numel(), qmm._stream(DEV)))
    close(y.double(), *want)


@pytest.mark.parametrize("t,e,k,h,f", [(1, 8, 2, 1056, 4128), (2, 4, 2, 288, 2080), (1, 16, 6, 544, 1056), (3, 8, 2, 288, 2080),
                                       (24, 8, 3, 544, 1056), (120, 4, 2, 288, 2080), (500, 3, 2, 160, 1120)])
def test_experts(t, e, k, h, f):
    wg, wu, wd = weight(1, e * f, h, h ** -0.5), weight(2, e * f, h, h ** -0.5), weight(3, e * h, f, f ** -0.5)
    x, lg = randn(t, t, h), randn(4, t, e)
    experts, weights = mx.route(lg, k, score="sigmoid")
    vg, vu, vd = (w.dequantize().double() for w in (wg, wu, wd))
    want = [torch.zeros(t, h, device=DEV, dtype=torch.float64) for _ in range(4)]
    for i in range(e):
        rows = [r for r in range(t) if i in experts[r]]
        if rows:
            c = f64([weights[r][experts[r].index(i)] for r in rows])[:, None]
            parts = ffn(x[rows], vg[i * f:(i + 1) * f], vu[i * f:(i + 1) * f], vd[i * h:(i + 1) * h])
            for j, p in enumerate(parts):
                want[j][rows] += (c * c if j == 1 else c) * p
    # (the weighted sum: k + 16 more additions of f32 terms)
    want[2] = want[2] * (1 + (k + 16) / (f / 32 + 34))
    y = moe_ffn(torch.from_numpy(x).to(DEV), torch.from_numpy(lg).to(DEV), wg, wu, wd, k, score="sigmoid")
    close(y.double(), *want)


@pytest.mark.parametrize("m,n,k", [(1, 100, 4096), (2, 70, 1056), (5, 130, 4128), (40, 260, 2080), (333, 128, 1024)])
def test_products_of_unrounded_rows(m, n, k):
    """A value is off by 2^-9 of its block's largest at most: against the plain product of x, that much of the block's
    absolute weights, and the f32 additions."""
    w = weight(n, n, k, 0.02)
    x = randn(m, m, k)
    y = QMatMul(w).forward(torch.from_numpy(x).to(DEV)).double()
    xv, v = f64(x), w.dequantize().double()
    top = xv.abs().view(m, k // 32, 32).amax(-1)
    tol = 2.0 ** -9 * (top @ v.abs().view(n, k // 32, 32).sum(-1).t())
    tol = tol + (k / 32 + 34) * 2.0 ** -23 * (1 + 2.0 ** -8) * (xv.abs() @ v.abs().t()) + 2.0 ** -24 * (xv @ v.t()).abs()
    want = xv @ v.t()
    assert bool(((y - want).abs() <= tol).all())
    # a row loses what its digits lose of its norm (1.1e-3 for normal values); the norms over n products with independent
    # weights scatter by 1 / sqrt(2 n) of themselves each, 9% at n = 70
    rel = (f64(mx.digit_values(x)) - xv).norm(dim=1) / xv.norm(dim=1)
    assert bool(((y - want).norm(dim=1) <= 1.5 * rel * want.norm(dim=1)).all()) and float(rel.max()) < 2.0 ** -9
