"""MXFP4 weights and their products on the GPU against a 64-bit restatement (oracle/mx.py).

Quantizers and converters: the same bytes. Products: every term of a row's sum is exact in f32 (a 10-bit value
times a 2-bit one), so the error is that of the additions: with k columns two matrix instructions per 64 of
them add into a running f32 sum and at most 32 partial sums are joined, each addition off by at most one unit
in the last place of the terms' absolute sum S (an instruction may cut rather than round): (k / 32 + 34) 2^-23 S.
A 16-bit output adds half a step of the value, a bias half an f32 step of the sum.
"""
import ctypes

import numpy as np
import pytest
import torch

from inference_amd import (GgmlDType, MatmulStrategy, QLinear, QMatMul, QmmError, QTensor, QuantizedLinear, block_dots,
                           matmul_grouped, matmul_multi, matmul_q, moe_ffn, moe_route, qmm, quantize_rows)
from oracle import mx

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
MX = GgmlDType.MXFP4


def randn(seed, *shape, std=1.0):
    return (np.random.default_rng(seed).standard_normal(shape) * std).astype(np.float32)


def weight(seed, n, k):
    b = mx.to_mxfp4(randn(seed, n, k, std=0.02))
    return QTensor.from_ggml(b.reshape(-1), MX, (n, k), device=DEV), b


def check(y, want, mag, k, dtype=torch.float32, bias=0.0):
    y = y.detach().double().cpu().numpy()
    tol = (k / 32 + 34) * 2.0 ** -23 * mag + 2.0 ** -24 * np.abs(want + bias)
    if dtype != torch.float32:
        tol = tol * (1 + 2.0 ** -8) + torch.finfo(dtype).eps / 2 * np.abs(want + bias) + torch.finfo(dtype).tiny * 2.0 ** -10
    bad = np.abs(y - (want + bias)) > tol
    assert not bad.any(), (np.argwhere(bad)[:4].tolist(), np.abs(y - want - bias)[bad][:4], tol[bad][:4])


# -- weights ------------------------------------------------------------------

def odd_values(n, k, seed=0):
    """Normal values with blocks of zeros, of one value, of powers of two at rounding borders, subnormals, huge."""
    w = randn(seed, n, k)
    b = w.reshape(-1, 32)
    b[0] = 0
    if len(b) > 8:
        b[1] = 0
        b[1, 5] = -3e-42
        b[2] *= np.float32(2.0 ** 100)
        b[3] = np.float32(2.0 ** -126) * np.arange(32)
        b[4, :4] = [7.0, 1.75, 0.25, -0.25]
        b[5] = np.float32(3e38)
        b[6, 0] = -0.0
        b[7] = np.linspace(-8, 8, 32)
    return w


@pytest.mark.parametrize("n,k", [(1, 32), (3, 96), (32, 256), (33, 288), (64, 512), (100, 1056), (257, 4096)])
def test_quantize_bytes(n, k):
    w = odd_values(n, k)
    qt = QTensor.quantize(torch.from_numpy(w).to(DEV), MX)
    assert qt.shape == (n, k) and qt.storage_size_in_bytes() == n * k // 32 * 17
    np.testing.assert_array_equal(qt.to_ggml().reshape(n, -1, 17), mx.to_mxfp4(w))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float64])
def test_quantize_other_types(dtype):
    w = torch.from_numpy(randn(1, 48, 320)).to(DEV).to(dtype)
    for src in (w, w.t().contiguous().t(), torch.cat([w.flatten()[:1], w.flatten()])[1:].view(48, 320)):
        got = QTensor.quantize(src, MX).to_ggml().reshape(48, -1, 17)
        np.testing.assert_array_equal(got, mx.to_mxfp4(w.float().cpu().numpy()))


def test_not_a_number():
    w = randn(2, 4, 128)
    w[0, 3], w[1, 40], w[2, 127] = np.nan, np.inf, -np.inf
    qt = QTensor.quantize(torch.from_numpy(w).to(DEV), MX)
    b = qt.to_ggml().reshape(4, 4, 17)
    np.testing.assert_array_equal(b[..., 0] == 255, [[1, 0, 0, 0], [0, 1, 0, 0], [0, 0, 0, 1], [0, 0, 0, 0]])
    d = qt.dequantize().cpu().numpy().reshape(4, 4, 32)
    np.testing.assert_array_equal(np.isnan(d).all(-1), b[..., 0] == 255)
    # such a block makes its output column NaN, such an activation its row, and no other
    for m in (1, 40):
        x = randn(3, m, 128)
        x[m // 2, 64] = np.inf
        y = QMatMul(qt).forward(torch.from_numpy(x).to(DEV)).cpu().numpy()
        want = np.zeros((m, 4), bool)
        want[:, :3] = True
        want[m // 2] = True
        np.testing.assert_array_equal(np.isnan(y), want)


@pytest.mark.parametrize("n,k", [(1, 32), (31, 64), (40, 352), (130, 768)])
@pytest.mark.parametrize("on_gpu", [False, True])
def test_import_export_dequantize(n, k, on_gpu):
    rng = np.random.default_rng(n + k)
    b = rng.integers(0, 256, (n, k // 32, 17), dtype=np.uint8)
    b[..., 0] = rng.integers(90, 160, b.shape[:2])
    b[0, 0, 0] = 0
    b[-1, -1, 0] = 254 if n > 1 else 0
    src = torch.from_numpy(b).to(DEV) if on_gpu else b.reshape(-1)
    qt = QTensor.from_ggml(src, MX, (n, k), device=DEV)
    np.testing.assert_array_equal(qt.to_ggml().reshape(b.shape), b)
    want = mx.from_mxfp4(b)
    np.testing.assert_array_equal(qt.dequantize().double().cpu().numpy(), want.astype(np.float32).astype(np.float64))
    for dt in (torch.float16, torch.bfloat16):
        ref = torch.from_numpy(want).float().to(dt)  # one rounding: the values have two significant bits
        assert torch.equal(qt.dequantize(dt).cpu(), ref)


def test_gguf_tensor(tmp_path):
    import gguf_writer as W
    from inference_amd.gguf import Content, unpermute_rows
    b = mx.to_mxfp4(randn(5, 64, 96))
    img = W.build([("general.architecture", W.T_STRING, "llama")], [("w", (64, 96), 39, b.tobytes())])
    p = tmp_path / "w.gguf"
    p.write_bytes(img)
    for heads in (0, 4):
        qt = Content.read(p).tensor("w", DEV, unpermute_heads=heads)
        want = b[unpermute_rows(64, heads)] if heads else b
        assert qt.dtype() == MX
        np.testing.assert_array_equal(qt.to_ggml().reshape(b.shape), want)


# -- rows ------------------------------------------------------------------------

@pytest.mark.parametrize("m,k,pad", [(1, 32, 0), (3, 96, 1), (17, 1024, 4), (65, 352, 0)])
def test_quantize_rows_bytes(m, k, pad):
    x = odd_values(m, k, seed=m)
    buf = torch.zeros((m, k + pad), device=DEV)
    buf[:, :k] = torch.from_numpy(x)
    got = quantize_rows(GgmlDType.MXFP6X2, buf[:, :k]).cpu().numpy().reshape(m, -1, 49)
    np.testing.assert_array_equal(got, mx.to_mxfp6x2(x))


# -- products --------------------------------------------------------------------

SHAPES = [(1, 1, 32), (1, 1024, 4096), (1, 33, 288), (2, 64, 256), (3, 40, 96), (8, 100, 1056), (16, 257, 512),
          (31, 32, 768), (32, 96, 14336), (33, 64, 256), (47, 130, 992), (64, 65, 544), (100, 300, 640), (128, 128, 2048),
          (129, 513, 384), (200, 1000, 320), (333, 260, 1024), (513, 384, 256), (700, 96, 4096)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_forward(m, n, k):
    qt, b = weight(n, n, k)
    x = randn(m, m, k)
    want, mag = mx.product(x, b)
    y = QMatMul.from_qtensor(qt).forward(torch.from_numpy(x).to(DEV))
    assert y.dtype == torch.float32
    check(y, want, mag, k)


@pytest.mark.parametrize("m,n,k", [(1, 100, 288), (2, 32, 64), (5, 70, 512), (40, 131, 352), (130, 260, 1056), (300, 96, 288)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bias", [None, torch.float32, torch.bfloat16, torch.float64])
def test_linear_types(m, n, k, dtype, bias):
    qt, b = weight(n, n, k)
    x = torch.from_numpy(randn(m, m, k)).to(dtype)
    bv = None if bias is None else torch.from_numpy(randn(7, n)).to(bias)
    want, mag = mx.product(x.float().numpy(), b)
    y = QuantizedLinear(QMatMul(qt), None if bv is None else bv.to(DEV)).forward(x.to(DEV))
    assert y.dtype == dtype and y.shape == (m, n)
    check(y, want, mag, k, dtype, 0.0 if bv is None else bv.float().double().numpy())


@pytest.mark.parametrize("m", [1, 5, 40, 140])
def test_wide_ranges(m):
    """Rows and weights whose blocks lie many binades apart (outlier channels), and tiny values."""
    n, k = 70, 1024
    w = randn(11, n, k, std=0.02) * np.exp2(np.random.default_rng(1).integers(-12, 12, (n, k // 32, 1))).repeat(
        32, -1).reshape(n, k).astype(np.float32)
    x = randn(12, m, k)
    x[:, 64:70] *= 300
    x[:, 512:544] *= np.float32(2.0 ** -130)
    b = mx.to_mxfp4(w)
    want, mag = mx.product(x, b)
    check(QMatMul(QTensor.from_ggml(b.reshape(-1), MX, (n, k), device=DEV)).forward(torch.from_numpy(x).to(DEV)), want,
          mag, k)


def test_strides_and_shapes():
    qt, b = weight(3, 48, 160)
    for m in (1, 2, 6, 70):
        base = torch.from_numpy(randn(m, m, 200)).to(DEV)
        for x in (base[:, 3:163], base[:, :160], base.t().contiguous().t()[:, 8:168]):
            want, mag = mx.product(x.cpu().numpy(), b)
            check(QMatMul(qt).forward(x), want, mag, 160)
            check(QuantizedLinear(QMatMul(qt), None).forward(x.bfloat16()), *mx.product(x.bfloat16().float().cpu().numpy(), b),
                  160, torch.bfloat16)
    x = torch.from_numpy(randn(4, 2, 3, 160)).to(DEV)
    want, mag = mx.product(x.reshape(6, 160).cpu().numpy(), b)
    y = QMatMul(qt).forward(x)
    assert y.shape == (2, 3, 48)
    check(y.reshape(6, 48), want, mag, 160)
    one = torch.from_numpy(randn(5, 160)).to(DEV)
    assert QMatMul(qt).forward(one).shape == (48,)
    row = one.expand(5, 160)  # one row five times (stride 0)
    check(QMatMul(qt).forward(row.contiguous()), *mx.product(row.cpu().numpy(), b), 160)
    check(QuantizedLinear(QMatMul(qt), None).forward(row), *mx.product(row.cpu().numpy(), b), 160)
    for d in (torch.float32, torch.bfloat16):
        assert QuantizedLinear(QMatMul(qt), None).forward(torch.empty(0, 160, device=DEV, dtype=d)).shape == (0, 48)


@pytest.mark.parametrize("m", [1, 4, 50])
def test_output_rows_keep_their_padding(m):
    """An output with a row stride: nothing past a row's n columns is written."""
    n, k = 45, 96
    qt, b = weight(4, n, k)
    x = randn(m, m, k)
    want, mag = mx.product(x, b)
    L = qmm.lib()
    y = torch.full((m, n + 7), 5.0, device=DEV)
    xd = torch.from_numpy(x).to(DEV)
    ws = torch.empty(L.qmm_matmul_workspace_size(qt.handle, m), dtype=torch.uint8, device=DEV)
    qmm._check(L.qmm_matmul(qt.handle, xd.data_ptr(), m, k, y.data_ptr(), n + 7, ws.data_ptr(), ws.numel(), qmm._stream(DEV)))
    check(y[:, :n], want, mag, k)
    assert (y[:, n:] == 5).all()


@pytest.mark.parametrize("m", [1, 8, 9, 40, 150])
def test_prequantized_rows_and_several_weights(m):
    """matmul_q, qmm_matmul_multi, qmm_matmul_multi_q, qmm_matmul_noalloc: the bits of QMatMul::forward."""
    k = 352
    (q1, b1), (q2, _), (q3, _) = weight(1, 40, k), weight(2, 96, k), weight(3, 33, k)
    x = torch.from_numpy(randn(m, m, k)).to(DEV)
    ref = [QMatMul(q).forward(x) for q in (q1, q2, q3)]
    check(ref[0], *mx.product(x.cpu().numpy(), b1), k)
    xq = quantize_rows(GgmlDType.MXFP6X2, x)
    for q, r in zip((q1, q2, q3), ref):
        assert torch.equal(matmul_q(q, xq, m), r)
    for y, r in zip(matmul_multi([q1, q2, q3], x), ref):
        assert torch.equal(y, r)
    L = qmm.lib()
    ys = [torch.empty_like(r) for r in ref]
    hs = (ctypes.c_void_p * 3)(*[q.handle.value for q in (q1, q2, q3)])
    yp = (ctypes.c_void_p * 3)(*[y.data_ptr() for y in ys])
    ld = (ctypes.c_int64 * 3)(*[y.shape[1] for y in ys])
    ws = torch.empty(L.qmm_matmul_q_workspace_size(q1.handle, m), dtype=torch.uint8, device=DEV)
    qmm._check(L.qmm_matmul_multi_q(hs, 3, xq.data_ptr(), m, yp, ld, ws.data_ptr(), ws.numel(), qmm._stream(DEV)))
    for y, r in zip(ys, ref):
        assert torch.equal(y, r)
    y = torch.empty_like(ref[0])
    qmm._check(L.qmm_matmul_noalloc(q1.handle, x.data_ptr(), m, k, y.data_ptr(), 40, qmm._stream(DEV)))
    assert torch.equal(y, ref[0])
    # accumulating, from blocks
    y = torch.ones_like(ref[0])
    qmm._check(L.qmm_matmul_q_ex(q1.handle, xq.data_ptr(), m, y.data_ptr(), 40, 1, ws.data_ptr(), ws.numel(), qmm._stream(DEV)))
    assert torch.equal(y, ref[0] + 1)


@pytest.mark.parametrize("m", [1, 2, 3, 40, 130])
def test_norm_and_residual(m):
    """qmm_matmul_ex: RMSNorm as qmm_rms_norm makes it, then the product, added to the residual."""
    k, n = 288, 100
    qt, _ = weight(6, n, k)
    x, g = torch.from_numpy(randn(m, m, k)).to(DEV), torch.from_numpy(randn(8, k)).to(DEV)
    L = qmm.lib()
    xn = torch.empty_like(x)
    qmm._check(L.qmm_rms_norm(x.data_ptr(), m, k, k, g.data_ptr(), 1e-5, xn.data_ptr(), k, qmm._stream(DEV)))
    res = torch.from_numpy(randn(9, m, n)).to(DEV)
    y = res.clone()
    ws = torch.empty(L.qmm_matmul_ex_workspace_size(qt.handle, m, 1), dtype=torch.uint8, device=DEV)
    h, yp, ld = (ctypes.c_void_p * 1)(qt.handle.value), (ctypes.c_void_p * 1)(y.data_ptr()), (ctypes.c_int64 * 1)(n)
    qmm._check(L.qmm_matmul_ex(h, 1, x.data_ptr(), m, k, g.data_ptr(), 1e-5, 1, yp, ld, ws.data_ptr(), ws.numel(),
                               qmm._stream(DEV)))
    assert torch.equal(y, QMatMul(qt).forward(xn) + res)


@pytest.mark.parametrize("m", [1, 3, 33, 130])
@pytest.mark.parametrize("norm", [False, True])
def test_ffn(m, norm):
    """qmm_ffn with MXFP4 weights against its parts: the f32 gate and up, silu(g) * u, the down product."""
    h, f = 96, 416
    (wg, _), (wu, _), (wd, bd) = weight(1, f, h), weight(2, f, h), weight(3, h, f)
    x, g = torch.from_numpy(randn(m, m, h)).to(DEV), torch.from_numpy(randn(8, h)).to(DEV)
    L = qmm.lib()
    xn = x
    if norm:
        xn = torch.empty_like(x)
        qmm._check(L.qmm_rms_norm(x.data_ptr(), m, h, h, g.data_ptr(), 1e-5, xn.data_ptr(), h, qmm._stream(DEV)))
    a, u = QMatMul(wg).forward(xn), QMatMul(wu).forward(xn)
    act = torch.empty_like(a)
    qmm._check(L.qmm_silu_mul(a.data_ptr(), u.data_ptr(), act.data_ptr(), a.numel(), qmm._stream(DEV)))
    want, mag = mx.product(act.cpu().numpy(), bd)
    nws = L.qmm_ffn_workspace_size(wg.handle, wu.handle, wd.handle, m, int(norm))
    ws = torch.empty(nws, dtype=torch.uint8, device=DEV)
    y = x.clone()
    qmm._check(L.qmm_ffn(wg.handle, wu.handle, wd.handle, x.data_ptr(), m, h, g.data_ptr() if norm else None, 1e-5, 1,
                         y.data_ptr(), h, ws.data_ptr(), nws, qmm._stream(DEV)))
    # silu in other instructions moves a value by some 2^-22 of itself, and with it at most one unit (2^-9 of the
    # block's maximum) of a digit that lay on a border: allowed for in one term of a row in 32
    slack = 2.0 ** -22 * mag + 2.0 ** -9 * np.abs(act.cpu().double().numpy()).max(1)[:, None] * \
        np.abs(mx.from_mxfp4(bd)).max(1)[None] * (f / 32)
    got = (y - x).double().cpu().numpy()
    tol = (f / 32 + 34) * 2.0 ** -23 * mag + slack + 2.0 ** -23 * (np.abs(x.cpu().numpy()) + np.abs(want))
    assert (np.abs(got - want) <= tol).all()


def test_other_strategies_and_refusals():
    qt, b = weight(1, 64, 256)
    q8 = QTensor.quantize(torch.randn(64, 256, device=DEV), GgmlDType.Q8_0)
    x = torch.from_numpy(randn(2, 12, 256)).to(DEV)
    # the dense strategy and the f16 form read the dequantized weight
    dense = QLinear(qt, strategy=MatmulStrategy.DEQUANT_DENSE).forward(x)
    assert torch.equal(dense, torch.nn.functional.linear(x, qt.dequantize()))
    assert QMatMul(qt).forward_via_f16(x).shape == (12, 64)
    check(QLinear(qt, strategy=MatmulStrategy.INT8_FAST).forward(x), *mx.product(x.cpu().numpy(), b), 256)
    xq = quantize_rows(GgmlDType.MXFP6X2, x)
    with pytest.raises(QmmError, match="block dots"):
        block_dots(qt, xq, 12)
    with pytest.raises(QmmError, match="Q4_K or Q6_K"):
        matmul_grouped([(qt, 0)], [x[0]])
    with pytest.raises(QmmError, match="share dtype"):
        matmul_multi([qt, q8], x)
    with pytest.raises(QmmError, match="MXFP4 weights"):
        QMatMul(q8).linear(x)
    with pytest.raises(QmmError, match="bias must be"):
        QMatMul(qt).linear(x, torch.zeros(63, device=DEV))
    with pytest.raises(QmmError, match="shape mismatch"):
        QMatMul(qt).linear(x[:, :224])
    with pytest.raises(QmmError, match="input on cpu"):
        QMatMul(qt).linear(x.cpu())
    with pytest.raises(QmmError, match="float32, float16 or bfloat16"):
        QMatMul(qt).linear(x.double())
    L = qmm.lib()
    y = torch.empty(12, 64, device=DEV)
    ws = torch.empty(L.qmm_matmul_workspace_size(qt.handle, 12), dtype=torch.uint8, device=DEV)
    s = qmm._stream(DEV)
    assert L.qmm_matmul(qt.handle, x.data_ptr(), 12, 256, y.data_ptr(), 64, ws.data_ptr(), ws.numel() - 1, s) == 1
    assert L.qmm_matmul(qt.handle, x.data_ptr(), 12, 256, y.data_ptr(), 64, None, 0, s) == 1
    assert L.qmm_matmul(qt.handle, x.data_ptr(), 12, 255, y.data_ptr(), 64, ws.data_ptr(), ws.numel(), s) == 1
    assert L.qmm_matmul(qt.handle, x.data_ptr(), 12, 256, y.data_ptr(), 63, ws.data_ptr(), ws.numel(), s) == 1
    assert L.qmm_linear(qt.handle, x.data_ptr(), 5, 12, 256, None, 0, y.data_ptr(), 0, 64, ws.data_ptr(), ws.numel(), s) == 1
    assert L.qmm_silu_mul_matmul(qt.handle, x.data_ptr(), x.data_ptr(), y.data_ptr(), 0, s) == 4
    assert L.qmm_ffn_workspace_size(qt.handle, q8.handle, qt.handle, 4, 0) == 0
    c = torch.zeros(8, dtype=torch.int32, device=DEV)
    h, yp = (ctypes.c_void_p * 1)(qt.handle.value), (ctypes.c_void_p * 1)(y.data_ptr())
    assert L.qmm_moe_gemv(h, 1, 2, xq.data_ptr(), 4, c.data_ptr(), c.data_ptr(), yp, s) == 4
    torch.cuda.synchronize()


def test_graph_and_streams():
    """Captured and replayed between eager calls on other inputs; two streams at once, each with its own output."""
    for m in (1, 20, 70):
        qt, _ = weight(1, 200, 544)
        lin = QuantizedLinear(QMatMul(qt), torch.ones(200, device=DEV))
        xs = [torch.from_numpy(randn(s, m, 544)).to(DEV) for s in range(4)]
        want = [lin.forward(x) for x in xs]
        x = xs[0].clone()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = lin.forward(x)
        for i in (1, 2, 3, 0):
            x.copy_(xs[i])
            g.replay()
            other = lin.forward(xs[(i + 1) % 4])
            torch.cuda.synchronize()
            assert torch.equal(y, want[i]) and torch.equal(other, want[(i + 1) % 4])
        streams = [torch.cuda.Stream() for _ in range(3)]
        got = []
        for i, st in enumerate(streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(lin.forward(xs[i]))
        torch.cuda.synchronize()
        for i in range(3):
            assert torch.equal(got[i], want[i])


# -- experts ---------------------------------------------------------------------

def expert_call(w, x, counts, offsets, experts, n, ws_extra=0):
    L = qmm.lib()
    p = x.shape[0]
    y = torch.full((p, n), 7.0, device=DEV)
    ws = torch.empty(L.qmm_moe_gemm_workspace_size(w.handle, p) + ws_extra, dtype=torch.uint8, device=DEV)
    h, yp = (ctypes.c_void_p * 1)(w.handle.value), (ctypes.c_void_p * 1)(y.data_ptr())
    qmm._check(L.qmm_moe_gemm(h, 1, experts, x.data_ptr(), p, x.stride(0), max(int(counts.max()), 1), counts.data_ptr(),
                              offsets.data_ptr(), yp, ws.data_ptr(), ws.numel(), qmm._stream(DEV)))
    return y


@pytest.mark.parametrize("cts", [[1], [0, 3, 0, 5], [40, 0, 1, 2, 70], [32, 32], [33, 64, 65, 1], [0] * 70 + [2, 0, 9],
                                 [130, 7, 0, 300]])
@pytest.mark.parametrize("n,k", [(40, 96), (96, 288), (260, 544)])
def test_expert_rows(cts, n, k):
    e, p = len(cts), sum(cts)
    w, b = weight(e + n, e * n, k)
    x = randn(p, p, k)
    counts = torch.tensor(cts, dtype=torch.int32, device=DEV)
    offs = np.concatenate([[0], np.cumsum(cts)])
    y = expert_call(w, torch.from_numpy(x).to(DEV), counts, torch.tensor(offs, dtype=torch.int32, device=DEV), e, n)
    for i, c in enumerate(cts):
        if c:
            s = slice(offs[i], offs[i + 1])
            check(y[s], *mx.product(x[s], b[i * n:(i + 1) * n]), k)


def test_expert_rows_left_alone():
    """Rows that no expert holds keep their values; counts past the rows are cut."""
    n, k = 64, 64
    w, b = weight(1, 3 * n, k)
    x = randn(1, 12, k)
    xd = torch.from_numpy(x).to(DEV)
    y = expert_call(w, xd, torch.tensor([2, 0, 3], dtype=torch.int32, device=DEV),
                    torch.tensor([1, 3, 5, 8], dtype=torch.int32, device=DEV), 3, n)
    check(y[1:3], *mx.product(x[1:3], b[:n]), k)
    check(y[5:8], *mx.product(x[5:8], b[2 * n:]), k)
    rest = torch.ones(12, dtype=torch.bool)
    rest[1:3] = rest[5:8] = False
    assert (y.cpu()[rest] == 7).all()
    L = qmm.lib()
    y = torch.full((12, n), 7.0, device=DEV)
    ws = torch.empty(L.qmm_moe_gemm_workspace_size(w.handle, 12), dtype=torch.uint8, device=DEV)
    h, yp = (ctypes.c_void_p * 1)(w.handle.value), (ctypes.c_void_p * 1)(y.data_ptr())
    big = torch.tensor([4, -3, 1000], dtype=torch.int32, device=DEV)
    off = torch.tensor([0, 4, 8, 12], dtype=torch.int32, device=DEV)
    qmm._check(L.qmm_moe_gemm(h, 1, 3, xd.data_ptr(), 12, k, 12, big.data_ptr(), off.data_ptr(), yp, ws.data_ptr(),
                              ws.numel(), qmm._stream(DEV)))
    check(y[:4], *mx.product(x[:4], b[:n]), k)
    assert (y[4:8] == 7).all()
    check(y[8:], *mx.product(x[8:], b[2 * n:]), k)


def moe_ref(x, experts, weights, bg, bu, bd, e):
    """MoE FFN in 64 bits (the activation's digits included), and its terms' absolute sum."""
    x64 = x.double().cpu().numpy()
    f, h = bg.shape[0] // e, bd.shape[0] // e
    out, mag = np.zeros((len(x64), h)), np.zeros((len(x64), h))
    for i in range(e):
        rows = [t for t, ids in enumerate(experts) if i in ids]
        if not rows:
            continue
        w = np.array([weights[t][experts[t].index(i)] for t in rows])[:, None]
        g, _ = mx.product(x64[rows], bg[i * f:(i + 1) * f])
        u, _ = mx.product(x64[rows], bu[i * f:(i + 1) * f])
        y, m = mx.product(g / (1 + np.exp(-g)) * u, bd[i * h:(i + 1) * h])
        out[rows] += w * y
        mag[rows] += np.abs(w) * m
    return out, mag


@pytest.mark.parametrize("t,e,k", [(1, 8, 2), (3, 4, 4), (20, 16, 3), (40, 5, 1), (90, 8, 2), (200, 64, 6), (17, 300, 12)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_moe_ffn(t, e, k, dtype):
    """The whole expert FFN, routed by sigmoid scores in groups. The digits of silu(g) * u may fall on the other side
    of a border than in 64 bits (by 2^-9 of a block's maximum, for a few values of a row): 2^-9 of the absolute sum
    bounds all of them at once."""
    h, f = 96, 160
    (wg, bg), (wu, bu), (wd, bd) = weight(1, e * f, h), weight(2, e * f, h), weight(3, e * h, f)
    x = torch.from_numpy(randn(t, t, h)).to(dtype)
    lg, bias = randn(4, t, e), randn(5, e, std=0.1)
    groups = 4 if e % 4 == 0 and e // 4 >= 2 else 1
    kw = dict(score="sigmoid", groups=groups, topk_groups=max(1, groups - 1) if k <= e - e // groups else groups, group_top=1)
    experts, weights = mx.route(lg, k, bias=bias, scale=2.5, **kw)
    want, mag = moe_ref(x.float(), experts, weights, bg, bu, bd, e)
    y = moe_ffn(x.to(DEV), torch.from_numpy(lg).to(DEV), wg, wu, wd, k, routed_scaling_factor=2.5,
                bias=torch.from_numpy(bias).to(DEV), out_dtype=dtype, **kw)
    assert y.dtype == dtype and y.shape == (t, h)
    got = y.double().cpu().numpy()
    assert (np.abs(got - want) <= 2.0 ** -9 * mag + torch.finfo(dtype).eps / 2 * np.abs(want) + 1e-7).all()
    # and closer on the whole: the roundings that may fall otherwise are few
    if dtype == torch.float32:
        assert np.linalg.norm(got - want) <= 2.0 ** -10 * np.linalg.norm(want)


@pytest.mark.parametrize("t", [1, 30])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("renorm", [True, False])
def test_moe_ffn_default_routing_and_shared_expert(t, dtype, renorm):
    """Without a score: softmax routing by qmm_moe_route_ex's rule; a shared MXFP4 expert with its gate."""
    e, k, h, f, fs = 8, 2, 64, 96, 160
    (wg, bg), (wu, bu), (wd, bd) = weight(1, e * f, h), weight(2, e * f, h), weight(3, e * h, f)
    (sg, bsg), (su, bsu), (sd, bsd) = weight(4, fs, h), weight(5, fs, h), weight(6, h, fs)
    gate = torch.from_numpy(randn(7, h)).to(DEV)
    x, lg = torch.from_numpy(randn(t, t, h)).to(dtype), randn(4, t, e)
    experts, weights = mx.route(lg, k, renormalize=renorm, scale=1.0 if renorm else 2.0)
    want, mag = moe_ref(x.float(), experts, weights, bg, bu, bd, e)
    ones = [[0]] * t, [[1.0]] * t
    swant, smag = moe_ref(x.float(), *ones, bsg, bsu, bsd, 1)
    s = 1 / (1 + np.exp(-(x.double().numpy() @ gate.double().cpu().numpy())))[:, None]
    y = moe_ffn(x.to(DEV), torch.from_numpy(lg).to(DEV), wg, wu, wd, k, norm_topk_prob=renorm, routed_scaling_factor=2.0,
                shared=(sg, su, sd), shared_gate=gate)
    assert y.dtype == torch.float32
    assert (np.abs(y.double().cpu().numpy() - want - s * swant) <= 2.0 ** -9 * (mag + smag) + 1e-7).all()
    # the f32 entry points that took the other types take this one: the same bits
    if dtype == torch.float32:
        L = qmm.lib()
        xd, ld, out = x.to(DEV), torch.from_numpy(lg).to(DEV), torch.empty(t, h, device=DEV)
        ws = torch.empty(L.qmm_moe_ffn_ex_workspace_size(wg.handle, wd.handle, t, e, k, sg.handle, su.handle, sd.handle),
                         dtype=torch.uint8, device=DEV)
        qmm._check(L.qmm_moe_ffn_ex(xd.data_ptr(), t, h, ld.data_ptr(), e, k, int(renorm), 2.0, wg.handle, wu.handle,
                                    wd.handle, sg.handle, su.handle, sd.handle, gate.data_ptr(), out.data_ptr(), h,
                                    ws.data_ptr(), ws.numel(), qmm._stream(DEV)))
        assert torch.equal(out, y)
        if renorm:
            ws = torch.empty(L.qmm_moe_ffn_workspace_size(wg.handle, wd.handle, t, e, k), dtype=torch.uint8, device=DEV)
            qmm._check(L.qmm_moe_ffn(xd.data_ptr(), t, h, ld.data_ptr(), e, k, wg.handle, wu.handle, wd.handle,
                                     out.data_ptr(), h, ws.data_ptr(), ws.numel(), qmm._stream(DEV)))
            assert (np.abs(out.double().cpu().numpy() - want) <= 2.0 ** -9 * mag + 1e-7).all()


def test_moe_ffn_long_list_in_chunks():
    """More pairs than one chunk (32768): every token's row as in a call of its own part."""
    t, e, k, h, f = 20000, 4, 2, 32, 32
    (wg, _), (wu, _), (wd, _) = weight(1, e * f, h), weight(2, e * f, h), weight(3, e * h, f)
    x, lg = torch.from_numpy(randn(1, t, h)).to(DEV), torch.from_numpy(randn(2, t, e)).to(DEV)
    y = moe_ffn(x, lg, wg, wu, wd, k)
    for a, b in ((0, 500), (16000, 17000), (19990, 20000)):
        assert torch.equal(y[a:b], moe_ffn(x[a:b].contiguous(), lg[a:b].contiguous(), wg, wu, wd, k))


def test_moe_ffn_scored_with_the_other_types():
    """Q4_K experts routed by scores: the routed sum of the plain call where both choose the same experts."""
    e, k, h, f, t = 8, 2, 256, 512, 12
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    q = [QTensor.quantize(torch.randn(s, generator=g, device=DEV) * 0.05, GgmlDType.Q4K)
         for s in ((e * f, h), (e * f, h), (e * h, f))]
    x, lg = torch.randn(t, h, generator=g, device=DEV), torch.randn(t, e, generator=g, device=DEV)
    for tokens in (1, t):
        plain = moe_ffn(x[:tokens], lg[:tokens], *q, k)
        same = moe_ffn(x[:tokens], lg[:tokens], *q, k, score="softmax")
        torch.testing.assert_close(same, plain, rtol=1e-5, atol=1e-5 * float(plain.abs().max()))
        half = moe_ffn(x[:tokens], lg[:tokens], *q, k, score="softmax", routed_scaling_factor=0.5, out_dtype=torch.bfloat16)
        assert half.dtype == torch.bfloat16
        torch.testing.assert_close(half.float(), 0.5 * plain, rtol=2.0 ** -8, atol=1e-5 * float(plain.abs().max()))
    # more tokens than a routing chunk of these types
    xl, ll = torch.randn(4100, h, generator=g, device=DEV), torch.randn(4100, e, generator=g, device=DEV)
    yl = moe_ffn(xl, ll, *q, k, score="sigmoid")
    assert torch.isfinite(yl).all()
    part = moe_ffn(xl[4096:], ll[4096:], *q, k, score="sigmoid")
    torch.testing.assert_close(yl[4096:], part, rtol=1e-4, atol=1e-4 * float(part.abs().max()))


def test_moe_refusals():
    e, h, f = 4, 64, 64
    (wg, _), (wu, _), (wd, _) = weight(1, e * f, h), weight(2, e * f, h), weight(3, e * h, f)
    q8 = QTensor.quantize(torch.randn(e * h, f, device=DEV), GgmlDType.Q8_0)
    x, lg = torch.zeros(3, h, device=DEV), torch.zeros(3, e, device=DEV)
    with pytest.raises(QmmError, match="all three in MXFP4"):
        moe_ffn(x, lg, wg, wu, q8, 2)
    with pytest.raises(QmmError, match="need a score"):
        moe_ffn(x, lg, wg, wu, wd, 2, groups=2)
    with pytest.raises(QmmError, match="experts/topk|routing limits"):
        moe_ffn(x, lg, wg, wu, wd, 5)
    with pytest.raises(QmmError, match="routing bias"):
        moe_ffn(x, lg, wg, wu, wd, 2, score="softmax", bias=torch.zeros(5, device=DEV))
    with pytest.raises(QmmError, match="logits"):
        moe_ffn(x, lg[:2], wg, wu, wd, 2)
    with pytest.raises(QmmError, match="rows on cpu"):
        moe_ffn(x.cpu(), lg, wg, wu, wd, 2)
    with pytest.raises(QmmError, match="float32, float16 or bfloat16"):
        moe_ffn(x, lg, wg, wu, wd, 2, out_dtype=torch.float64)
    with pytest.raises(QmmError, match="out of"):
        moe_ffn(x, lg, wg, wu, wd, 2, score="softmax", groups=4, topk_groups=1)
    assert moe_ffn(x[:0], lg[:0], wg, wu, wd, 2).shape == (0, h)


def test_moe_ffn_graph_and_used_together():
    """A block as a program runs it, captured: a projection, the router's product, routing and the experts."""
    e, k, h, f, t = 16, 4, 128, 96, 24
    (wp, _), (wr, _) = weight(1, h, h), weight(2, e, h)
    (wg, _), (wu, _), (wd, _) = weight(3, e * f, h), weight(4, e * f, h), weight(5, e * h, f)
    proj, router = QuantizedLinear(QMatMul(wp), None), QMatMul(wr)
    bias = torch.from_numpy(randn(6, e, std=0.1)).to(DEV)

    def block(x):
        y = proj.forward(x)
        lg = router.forward(y.float())
        r = moe_route(lg, k, score="sigmoid", bias=bias, groups=4, topk_groups=2, group_top=2)
        return (moe_ffn(y, lg, wg, wu, wd, k, score="sigmoid", bias=bias, groups=4, topk_groups=2, group_top=2,
                        out_dtype=y.dtype), *r)

    xs = [torch.from_numpy(randn(s, t, h)).to(DEV).bfloat16() for s in range(3)]
    want = [block(x) for x in xs]
    x = xs[0].clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = block(x)
    for i in (1, 2, 0):
        x.copy_(xs[i])
        g.replay()
        eager = block(xs[(i + 1) % 3])
        torch.cuda.synchronize()
        for a, b in zip(out, want[i]):
            assert torch.equal(a, b)
        for a, b in zip(eager, want[(i + 1) % 3]):
            assert torch.equal(a, b)
