"""MXFP4 products over the sizes at which their launch changes: waves that split the columns of x, column tiles of a
group, chunks in flight, wide tiles, rows quantized in place or ahead, rows too long for that.

The reference is in 64 bits on the GPU: the weight's values are exact in f32 (dequantize), x's are its digits'
(oracle/mx.py). The tolerance: (k / 32 + 34) 2^-23 of the terms' absolute sum (two additions per 64 columns into a
running f32 sum and at most 32 partial sums, each off by a unit in the last place at most) and one rounding of the
value, half a step of its type.
"""
import ctypes

import numpy as np
import pytest
import torch

from inference_amd import GgmlDType, QMatMul, QmmError, QTensor, QuantizedLinear, moe_ffn, qmm
from oracle import mx

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
MX = GgmlDType.MXFP4


def randn(seed, *shape, std=1.0):
    return (np.random.default_rng(seed).standard_normal(shape) * std).astype(np.float32)


def weight(seed, n, k):
    """Random codes under scales of 2^-12 to 2^-7."""
    rng = np.random.default_rng(seed)
    b = rng.integers(0, 256, (n, k // 32, 17), dtype=np.uint8)
    b[..., 0] = rng.integers(115, 121, b.shape[:2])
    return QTensor.from_ggml(b.reshape(-1), MX, (n, k), device=DEV)


def product(x, w):
    """(x . w^T, the terms' absolute sum) in f64 on the GPU; x as numpy or torch rows, w f32 values."""
    x = x.float().cpu().numpy() if isinstance(x, torch.Tensor) else x
    xv, wv = torch.from_numpy(mx.digit_values(x)).to(DEV), w.double()
    return xv @ wv.t(), xv.abs() @ wv.abs().t()


def check(y, x, w, dtype=torch.float32):
    want, mag = product(x, w)
    tol = (w.shape[1] / 32 + 34) * 2.0 ** -23 * mag + 2.0 ** -24 * want.abs()
    if dtype != torch.float32:
        tol = tol * (1 + 2.0 ** -8) + torch.finfo(dtype).eps / 2 * want.abs() + torch.finfo(dtype).tiny * 2.0 ** -10
    assert y.dtype == dtype and y.shape == want.shape
    bad = (y.double() - want).abs() > tol
    assert not bool(bad.any()), (torch.nonzero(bad)[:4].tolist(), (y.double() - want).abs()[bad][:4], tol[bad][:4])


@pytest.mark.parametrize("m,n,k", [
    (1, 16400, 1056), (2, 16390, 160), (1, 8200, 1312), (2, 8200, 2080), (1, 40, 4096), (2, 100, 4128), (1, 48, 14336),
    (2, 70, 16384)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("pad", [0, 1])
def test_one_and_two_rows(m, n, k, dtype, pad):
    """Quantized by the product itself; with pad, rows that no 16-byte load can read."""
    w = weight(n + k, n, k)
    x = torch.from_numpy(randn(m, m, k + 3 * pad)).to(dtype).to(DEV)[:, pad:k + pad]
    check(QuantizedLinear(QMatMul(w), None).forward(x), x, w.dequantize(), dtype)


@pytest.mark.parametrize("m,n,k", [
    (5, 70, 4064), (16, 100, 2080), (9, 130, 1312), (3, 40, 14336),  # one column tile a group, 16 and 8 waves
    (3, 8200, 96), (16, 8210, 1312), (4, 8200, 2400), (17, 4100, 2400), (64, 1030, 160), (64, 4090, 1056),
    (128, 4090, 288), (128, 260, 4128), (500, 1024, 96), (300, 33, 544), (6, 66000, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_few_rows(m, n, k, dtype):
    w = weight(n + k, n, k)
    x = torch.from_numpy(randn(m, m, k)).to(dtype).to(DEV)
    check(QuantizedLinear(QMatMul(w), None).forward(x), x, w.dequantize(), dtype)


@pytest.mark.parametrize("m,n,k", [
    (129, 4100, 96), (520, 4096, 544),                    # 64 x 128, four ways over the columns of x
    (1000, 4090, 96), (1000, 4090, 800),                  # 128 x 128
    (1000, 8180, 96), (1030, 8150, 544), (2100, 4097, 64)])  # 128 x 256
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_many_rows(m, n, k, dtype):
    w = weight(n + k, n, k)
    x = torch.from_numpy(randn(m, m, k)).to(dtype).to(DEV)
    b = torch.from_numpy(randn(3, n)).to(DEV)
    y = QuantizedLinear(QMatMul(w), None).forward(x)
    check(y, x, w.dequantize(), dtype)
    if dtype == torch.float32:  # the same sums, and the bias added to them in f32
        assert torch.equal(QuantizedLinear(QMatMul(w), b).forward(x), y + b)


@pytest.mark.parametrize("m", [1, 2, 3])
def test_rows_longer_than_a_workgroup_holds(m):
    """More than 16384 values a row: one and two rows take the workspace, too, and are refused without it."""
    n, k = 40, 16640
    w = weight(1, n, k)
    x = torch.from_numpy(randn(m, m, k)).to(DEV)
    L = qmm.lib()
    for dtype in (torch.float32, torch.bfloat16):
        check(QuantizedLinear(QMatMul(w), None).forward(x.to(dtype)), x.to(dtype), w.dequantize(), dtype)
    check(QMatMul(w).forward(x), x, w.dequantize())
    y = torch.empty(m, n, device=DEV)
    assert L.qmm_matmul_workspace_size(w.handle, m) > 0 and L.qmm_linear_workspace_size(w.handle, m) > 0
    s = qmm._stream(DEV)
    assert L.qmm_matmul(w.handle, x.data_ptr(), m, k, y.data_ptr(), n, None, 0, s) == 1
    assert L.qmm_linear(w.handle, x.data_ptr(), 0, m, k, None, 0, y.data_ptr(), 0, n, None, 0, s) == 1
    qmm._check(L.qmm_matmul_noalloc(w.handle, x.data_ptr(), m, k, y.data_ptr(), n, s))
    check(y, x, w.dequantize())
    torch.cuda.synchronize()


@pytest.mark.parametrize("counts,n,k", [
    ([50, 0, 0, 1, 0, 0, 0, 0], 100, 288),       # four row tiles of one expert, one column tile a group
    ([50, 0, 0, 1, 0, 0, 0, 0], 2060, 2400),     # four column tiles, 16 and 8 waves
    ([3, 0, 2], 100, 2400),                      # 16 waves, a chunk each
    ([1] * 8, 1030, 1312),                       # four column tiles, 8 waves
    ([2, 0, 33, 5] * 16, 1040, 1312),            # four waves, two chunks each
    ([100, 0, 250], 500, 352),                   # 64-row tiles
    ([500, 524], 3570, 96),                      # 128 x 128
    ([500, 524], 7100, 160)])                    # 128 x 256
def test_expert_rows(counts, n, k):
    e, p = len(counts), sum(counts)
    w = weight(e + n, e * n, k)
    x = torch.from_numpy(randn(p, p, k)).to(DEV)
    offs = np.concatenate([[0], np.cumsum(counts)])
    L = qmm.lib()
    y = torch.empty(p, n, device=DEV)
    ws = torch.empty(L.qmm_moe_gemm_workspace_size(w.handle, p), dtype=torch.uint8, device=DEV)
    h, yp = (ctypes.c_void_p * 1)(w.handle.value), (ctypes.c_void_p * 1)(y.data_ptr())
    c, o = (torch.tensor(v, dtype=torch.int32, device=DEV) for v in (counts, offs))
    qmm._check(L.qmm_moe_gemm(h, 1, e, x.data_ptr(), p, k, max(counts), c.data_ptr(), o.data_ptr(), yp, ws.data_ptr(),
                              ws.numel(), qmm._stream(DEV)))
    v = w.dequantize()
    for i in range(e):
        if counts[i]:
            check(y[offs[i]:offs[i + 1]], x[offs[i]:offs[i + 1]], v[i * n:(i + 1) * n])


def ffn_reference(x, rows, g, u, d):
    """down(silu(gate(x)) * up(x)) of one expert and its terms' absolute sum, the inner rows as digits."""
    a, b = product(x[rows], g)[0], product(x[rows], u)[0]
    return product((a / (1 + torch.exp(-a)) * b).cpu().numpy(), d)


@pytest.mark.parametrize("t,e,k,h,f", [
    (1, 8, 2, 4128, 160), (2, 4, 2, 2080, 96), (2, 64, 6, 288, 1056), (1, 4, 1, 96, 8224), (1, 2, 2, 16416, 64),
    (1, 2, 1, 16384, 64), (1, 8, 2, 1312, 64),
    (5, 8, 2, 4128, 96), (20, 8, 3, 1312, 288), (9, 8, 2, 544, 4128), (120, 16, 2, 96, 1056), (120, 4, 4, 544, 416),
    (700, 3, 2, 288, 1120)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_moe_ffn(t, e, k, h, f, dtype):
    """Every token through its experts. The digits of silu(g) * u may fall on the other side of a border than in 64
    bits, by 2^-9 of a block's maximum: 2^-9 of the absolute sum bounds all of them at once."""
    wg, wu, wd = weight(1, e * f, h), weight(2, e * f, h), weight(3, e * h, f)
    x = torch.from_numpy(randn(t, t, h)).to(dtype)
    lg = randn(4, t, e)
    experts, weights = mx.route(lg, k, score="sigmoid")
    want, mag = torch.zeros(t, h, device=DEV, dtype=torch.float64), torch.zeros(t, h, device=DEV, dtype=torch.float64)
    vg, vu, vd = wg.dequantize(), wu.dequantize(), wd.dequantize()
    for i in range(e):
        rows = [r for r in range(t) if i in experts[r]]
        if rows:
            c = torch.tensor([weights[r][experts[r].index(i)] for r in rows], device=DEV, dtype=torch.float64)[:, None]
            y, s = ffn_reference(x, rows, vg[i * f:(i + 1) * f], vu[i * f:(i + 1) * f], vd[i * h:(i + 1) * h])
            want[rows] += c * y
            mag[rows] += c * s
    y = moe_ffn(x.to(DEV), torch.from_numpy(lg).to(DEV), wg, wu, wd, k, score="sigmoid", out_dtype=dtype)
    assert y.dtype == dtype
    assert bool(((y.double() - want).abs() <= 2.0 ** -9 * mag + torch.finfo(dtype).eps / 2 * want.abs() + 1e-7).all())


@pytest.mark.parametrize("m,h,f", [(1, 2080, 1056), (2, 4128, 64), (1, 16416, 32), (1, 16384, 32), (7, 1312, 544),
                                   (60, 96, 2080), (300, 160, 2080), (130, 544, 8224)])
def test_ffn(m, h, f):
    """A dense MXFP4 FFN added to the residual, by the same bound as the experts'."""
    wg, wu, wd = weight(1, f, h), weight(2, f, h), weight(3, h, f)
    x = torch.from_numpy(randn(m, m, h))
    want, mag = ffn_reference(x, list(range(m)), wg.dequantize(), wu.dequantize(), wd.dequantize())
    L = qmm.lib()
    xd, y = x.to(DEV), torch.ones(m, h, device=DEV)
    nws = L.qmm_ffn_workspace_size(wg.handle, wu.handle, wd.handle, m, 0)
    ws = torch.empty(nws, dtype=torch.uint8, device=DEV)
    qmm._check(L.qmm_ffn(wg.handle, wu.handle, wd.handle, xd.data_ptr(), m, h, None, 0.0, 1, y.data_ptr(), h,
                         ws.data_ptr(), nws, qmm._stream(DEV)))
    assert bool(((y.double() - 1 - want).abs() <= 2.0 ** -9 * mag + 2.0 ** -23 * (1 + want.abs())).all())


def test_scale_bytes_below_the_least():
    """Rows given as blocks: a scale byte under 4 has no byte 2^4 below it for the second digits, and says NaN."""
    w = weight(1, 33, 64)
    x = torch.from_numpy(randn(2, 6, 64)).to(DEV)
    xq = qmm.quantize_rows(GgmlDType.MXFP6X2, x).view(6, 2, 49)
    xq[3, 1, 0] = 3
    y = qmm.matmul_q(w, xq.view(6, -1), 6)
    nan = torch.isnan(y).all(1).cpu()
    assert nan.tolist() == [False, False, False, True, False, False]
    keep = [0, 1, 2, 4, 5]
    check(y[keep], x[keep], w.dequantize())


def test_one_workspace_for_calls_in_order():
    """Calls of one stream may share a workspace: each is done with it before the next begins."""
    w = weight(1, 300, 544)
    v = w.dequantize()
    L = qmm.lib()
    xs = [torch.from_numpy(randn(s, m, 544)).to(DEV) for s, m in enumerate((40, 3, 300, 16))]
    ws = torch.empty(L.qmm_matmul_workspace_size(w.handle, 300), dtype=torch.uint8, device=DEV)
    ys = [torch.empty(x.shape[0], 300, device=DEV) for x in xs]
    for x, y in zip(xs, ys):
        qmm._check(L.qmm_matmul(w.handle, x.data_ptr(), x.shape[0], 544, y.data_ptr(), 300, ws.data_ptr(), ws.numel(),
                                qmm._stream(DEV)))
    for x, y in zip(xs, ys):
        check(y, x, v)


def test_mixed_types_are_refused():
    w = weight(1, 64, 64)
    with pytest.raises(QmmError):
        QMatMul(w).forward(torch.zeros(2, 64, device=DEV, dtype=torch.float16))


@pytest.mark.parametrize("m", [1, 2, 20])
def test_attention_output_projection(m):
    """qmm_prefill_attention_o with an MXFP4 projection: the attention, then the product added to the residual."""
    heads, kv, hd, max_seq, n = 4, 2, 64, 32, 100
    h = heads * hd
    wo = weight(1, n, h)
    q, kc, vc = (torch.from_numpy(randn(i, *s)).to(DEV) for i, s in enumerate(
        ((m, h), (kv, max_seq, hd), (kv, max_seq, hd))))
    L, s, scale = qmm.lib(), qmm._stream(DEV), ctypes.c_float(0.125)
    att = torch.empty(m, h, device=DEV)
    qmm._check(L.qmm_prefill_attention(q.data_ptr(), h, kc.data_ptr(), vc.data_ptr(), 3, m, att.data_ptr(), h, heads, kv,
                                       hd, max_seq, scale, s))
    res = torch.from_numpy(randn(9, m, n)).to(DEV)
    x = res.clone()
    nws = L.qmm_prefill_attention_o_workspace_size(wo.handle, m)
    ws = torch.empty(nws, dtype=torch.uint8, device=DEV)
    qmm._check(L.qmm_prefill_attention_o(q.data_ptr(), h, kc.data_ptr(), vc.data_ptr(), 3, m, heads, kv, hd, max_seq,
                                         scale, wo.handle, x.data_ptr(), n, ws.data_ptr(), nws, s))
    assert torch.equal(x, QMatMul(wo).forward(att) + res)


def test_cache_warming_refuses_the_type():
    """qmm_decode_rope_attention_warm knows the row bytes of Q4_K and Q6_K only."""
    w = weight(1, 256, 256)
    b = torch.zeros(1 << 16, device=DEV)
    p = [b.data_ptr()] * 5 + [torch.zeros(1, dtype=torch.int32, device=DEV).data_ptr()] + [b.data_ptr()] * 3
    L = qmm.lib()
    ws = torch.empty(L.qmm_decode_attention_workspace_size(4, 2, 64, 32), dtype=torch.uint8, device=DEV)
    assert L.qmm_decode_rope_attention_warm(*p, 4, 2, 64, 32, ctypes.c_float(1), ws.data_ptr(), ws.numel(),
                                            (ctypes.c_void_p * 1)(w.handle.value), (ctypes.c_int * 1)(0), 1,
                                            (ctypes.c_int * 1)(1), qmm._stream(DEV)) == 1
    assert "Q4_K / Q6_K" in qmm.last_error()


def test_unaligned_workspaces_are_refused():
    e, h, f = 4, 64, 96
    wg, wu, wd = weight(1, e * f, h), weight(2, e * f, h), weight(3, e * h, f)
    x, lg, y = torch.zeros(20, h, device=DEV), torch.zeros(20, e, device=DEV), torch.zeros(20, e * f, device=DEV)
    L, s = qmm.lib(), qmm._stream(DEV)
    ws = torch.empty(1 << 20, dtype=torch.uint8, device=DEV)
    c = torch.zeros(256, dtype=torch.int32, device=DEV)
    a, n = ws.data_ptr() + 4, ws.numel() - 4
    hp, yp = (ctypes.c_void_p * 1)(wg.handle.value), (ctypes.c_void_p * 1)(y.data_ptr())
    fg, fu, fd = weight(4, f, h), weight(5, f, h), weight(6, h, f)
    calls = [
        (L.qmm_matmul, wg.handle, x.data_ptr(), 20, h, y.data_ptr(), e * f),
        (L.qmm_linear, wg.handle, x.data_ptr(), 0, 20, h, None, 0, y.data_ptr(), 0, e * f),
        (L.qmm_matmul_q, wg.handle, x.data_ptr(), 20, y.data_ptr(), e * f),
        (L.qmm_ffn, fg.handle, fu.handle, fd.handle, x.data_ptr(), 20, h, None, 0.0, 0, y.data_ptr(), h),
        (L.qmm_moe_gemm, hp, 1, e, x.data_ptr(), 20, h, 20, c.data_ptr(), c.data_ptr(), yp),
        (L.qmm_moe_route_scored, lg.data_ptr(), 20, e, 2, 0, None, 1, 1, 1, 1, 1.0, c.data_ptr(), c.data_ptr(),
         c.data_ptr(), y.data_ptr(), c.data_ptr()),
        (L.qmm_moe_ffn_scored, x.data_ptr(), 0, 20, h, lg.data_ptr(), e, 2, 0, None, 1, 1, 1, 1, 1.0, wg.handle,
         wu.handle, wd.handle, None, None, None, None, y.data_ptr(), 0, h)]
    for fn, *args in calls:
        assert fn(*args, a, n, s) == 1 and "aligned" in qmm.last_error(), (args, qmm.last_error())


def test_gguf_dense_load(tmp_path):
    import gguf_writer as W
    from inference_amd.gguf import GgufFile
    b = mx.to_mxfp4(randn(5, 64, 96))
    p = tmp_path / "w.gguf"
    p.write_bytes(W.build([("general.architecture", W.T_STRING, "llama")], [("w", (64, 96), 39, b.tobytes())]))
    f = GgufFile.open(p)
    got = f.load_dense(f.tensors[0], DEV)
    assert got.shape == (64, 96) and got.dtype == torch.float32
    np.testing.assert_array_equal(got.double().cpu().numpy(), mx.from_mxfp4(b))


@pytest.mark.parametrize("t", [1, 2, 5])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pad", [0, 3, 8])
def test_moe_rows_keep_their_padding(t, dtype, pad):
    """Strided rows in and out of the C call: the Python call's values, nothing written past a row."""
    e, k, h, f = 6, 3, 96, 160
    wg, wu, wd = weight(1, e * f, h), weight(2, e * f, h), weight(3, e * h, f)
    x = torch.from_numpy(randn(t, t, h + pad)).to(dtype).to(DEV)
    lg = torch.from_numpy(randn(4, t, e)).to(DEV)
    want = moe_ffn(x[:, :h], lg, wg, wu, wd, k, score="softmax", out_dtype=dtype)
    L, tag = qmm.lib(), qmm._DENSE[dtype]
    out = torch.full((t, h + pad), 5.0, dtype=dtype, device=DEV)
    ws = torch.empty(L.qmm_moe_ffn_scored_workspace_size(wg.handle, wd.handle, t, e, k, None, None, None),
                     dtype=torch.uint8, device=DEV)
    qmm._check(L.qmm_moe_ffn_scored(x.data_ptr(), tag, t, h + pad, lg.data_ptr(), e, k, 0, None, 1, 1, 1, 1, 1.0,
                                    wg.handle, wu.handle, wd.handle, None, None, None, None, out.data_ptr(), tag, h + pad,
                                    ws.data_ptr(), ws.numel(), qmm._stream(DEV)))
    assert torch.equal(out[:, :h], want) and bool((out[:, h:] == 5).all())


@pytest.mark.parametrize("t", [1, 2])
def test_moe_token_captured_and_on_two_streams(t):
    """The decode form: replayed between eager calls on other inputs, and two calls at once."""
    e, k, h, f = 16, 4, 288, 160
    wg, wu, wd = weight(1, e * f, h), weight(2, e * f, h), weight(3, e * h, f)
    bias = torch.from_numpy(randn(6, e, std=0.1)).to(DEV)
    xs = [torch.from_numpy(randn(s, t, h)).to(DEV).bfloat16() for s in range(3)]
    ls = [torch.from_numpy(randn(s + 9, t, e)).to(DEV) for s in range(3)]

    def call(x, lg):
        return moe_ffn(x, lg, wg, wu, wd, k, score="sigmoid", bias=bias, groups=4, topk_groups=2, group_top=2,
                       out_dtype=torch.bfloat16)

    want = [call(x, lg) for x, lg in zip(xs, ls)]
    x, lg = xs[0].clone(), ls[0].clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = call(x, lg)
    for i in (1, 2, 0, 1):
        x.copy_(xs[i])
        lg.copy_(ls[i])
        g.replay()
        eager = call(xs[(i + 1) % 3], ls[(i + 1) % 3])
        torch.cuda.synchronize()
        assert torch.equal(y, want[i]) and torch.equal(eager, want[(i + 1) % 3])
    got = []
    for i in range(2):
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got.append(call(xs[i], ls[i]))
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_offsets_past_32_bits():
    """A weight of 4.6 GB, products of 2.3 G values and a dense form of 8.6 G: the last rows and columns."""
    n, k, tail = 2100000, 4096, 100
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    b = torch.randint(0, 256, (n, k // 32, 17), dtype=torch.uint8, device=DEV, generator=g)
    b[..., 0] = 118
    w = QTensor.from_ggml(b.reshape(-1), MX, (n, k), device=DEV)
    end = QTensor.from_ggml(b[-tail:].contiguous().reshape(-1), MX, (tail, k), device=DEV)
    del b
    v = end.dequantize()
    assert torch.equal(w.dequantize(torch.bfloat16)[-tail:].float(), v)
    for m in (1, 5, 20, 1100):
        x = torch.from_numpy(randn(m, m, k)).to(DEV)
        y = QMatMul(w).forward(x)
        check(y[-3:, -tail:], x[-3:], v)
        del y
    torch.cuda.empty_cache()
