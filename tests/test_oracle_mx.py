"""The 64-bit restatement of the microscaled types against their definitions (no GPU), and the refusals of the
new entry points that are decided on the host."""
import ctypes
import itertools
import math

import numpy as np
import pytest

from oracle import mx


def test_grids_are_the_formats():
    """E2M1 / E2M3: sign, two exponent bits (bias 1), one / three mantissa bits, exponent 0 without the leading 1."""
    for grid, bits in ((mx.E2M1, 1), (mx.E2M3, 3)):
        assert len(grid) == 4 << bits
        for c, v in enumerate(grid):
            e, m = c >> bits, c % (1 << bits) / (1 << bits)
            assert v == (m if e == 0 else 2.0 ** (e - 1) * (1 + m))


def test_nearest_is_the_nearest_code():
    for grid in (mx.E2M1, mx.E2M3):
        t = np.linspace(-9, 9, 4 * 16 * 18 + 1)
        got = mx.nearest(t, grid)
        for v, c in zip(np.abs(t), got):
            d = np.abs(grid - min(v, grid[-1] + 100))
            best = np.flatnonzero(d == d.min())
            assert c in best and (len(best) == 1 or c % 2 == 0)


@pytest.mark.parametrize("grid,least", [(mx.E2M1, 0), (mx.E2M3, 4)])
def test_scale_is_the_smallest_that_does_not_round_past_the_top(grid, least):
    top, step = grid[-1], grid[-1] - grid[-2]
    longer = np.concatenate([grid, [top + step, top + 2 * step]])  # where rounding would go next
    for p, f in itertools.product((-126, -20, 0, 3, 100), (1, 1.2, 1.5, 1.74, 1.75, 1.76, 1.93, 1.9375, 1.94, 1.99)):
        v = float(np.float32(f)) * 2.0 ** p
        e = int(mx.scale_byte(np.array([v]), grid, least)[0])
        assert longer[mx.nearest(v / 2.0 ** (e - 127), longer)] <= top
        assert e == least or longer[mx.nearest(v / 2.0 ** (e - 1 - 127), longer)] > top
    assert mx.scale_byte(np.array([0.0, math.inf]), grid, least).tolist() == [least, 255]


def test_digits_leave_at_most_a_512th_of_the_block_maximum():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((64, 256)) * np.exp2(rng.integers(-20, 20, (64, 1)))
    err = np.abs(mx.digit_values(x) - x).reshape(64, 8, 32)
    assert (err <= np.abs(x).reshape(64, 8, 32).max(-1, keepdims=True) / 512).all()
    assert np.linalg.norm(err) <= 2e-3 * np.linalg.norm(x)


def test_packing():
    w = np.zeros((1, 32), np.float32)
    w[0, 0], w[0, 16], w[0, 31] = 6.0, -0.5, 3.0
    b = mx.to_mxfp4(w)[0, 0]
    assert b[0] == 127 and b[1] == (7 | (8 + 1) << 4) and b[16] == 5 << 4
    assert np.array_equal(mx.from_mxfp4(mx.to_mxfp4(w)), w)
    x = np.zeros((1, 32), np.float32)
    x[0, 1] = -7.5
    q = mx.to_mxfp6x2(x)[0, 0]
    assert q[0] == 127 and int.from_bytes(q[1:25].tobytes(), "little") == 63 << 6


# ---------------------------------------------------------------------------
# refusals decided on the host
# ---------------------------------------------------------------------------

@pytest.fixture(scope="module")
def L():
    from inference_amd import qmm
    return qmm.lib()


def test_geometry(L):
    assert (L.qmm_block_size(39), L.qmm_type_size(39), L.qmm_vec_dot_type(39)) == (32, 17, 256)
    assert (L.qmm_block_size(256), L.qmm_type_size(256), L.qmm_vec_dot_type(256)) == (32, 49, -1)


def test_weight_refusals(L):
    h = ctypes.c_void_p()
    buf = (ctypes.c_uint8 * 64)()
    for args in ((39, 1, 33, buf, 0), (39, 0, 32, buf, 0), (39, 1, 0, buf, 0), (256, 1, 32, buf, 0), (39, 1, 32, None, 0),
                 (39, 2 ** 31 - 1, 2 ** 31 - 32, buf, 0)):
        assert L.qmm_qtensor_from_ggml(*args[:3], args[3], args[4], None, ctypes.byref(h)) == 1 and h.value is None
    assert L.qmm_qtensor_quantize_from(39, 1, 32, buf, 2, None, ctypes.byref(h)) == 1  # no such input type
    assert L.qmm_qtensor_quantize_from(12, 1, 256, buf, 30, None, ctypes.byref(h)) == 4  # bf16 into Q4_K
    assert L.qmm_qtensor_quantize_from(39, 1, 32, None, 0, None, ctypes.byref(h)) == 1
    assert L.qmm_quantize_rows(256, buf, 1, 48, 48, buf, None) == 1  # k % 32
    assert L.qmm_quantize_rows(256, buf, 1, 64, 32, buf, None) == 1  # ldx < k
    assert L.qmm_quantize_rows(39, buf, 1, 32, 32, buf, None) == 1   # a weight type
    assert L.qmm_linear(None, buf, 0, 1, 32, None, 0, buf, 0, 32, None, 0, None) == 1
    assert L.qmm_linear_workspace_size(None, 1) == 0


GOOD = dict(tokens=4, experts=16, topk=4, score=1, groups=4, topk_groups=2, group_top=2, scale=1.0)


@pytest.mark.parametrize("bad", [dict(tokens=0), dict(tokens=65537), dict(experts=0), dict(experts=1025, groups=1,
                                 topk_groups=1), dict(topk=0), dict(topk=9), dict(topk=33, experts=64, topk_groups=4),
                                 dict(score=2), dict(score=-1), dict(groups=3), dict(groups=0), dict(topk_groups=0),
                                 dict(topk_groups=5), dict(group_top=0), dict(group_top=3),
                                 dict(groups=16, topk_groups=8), dict(scale=math.nan), dict(experts=130, groups=65,
                                 topk_groups=65)])
def test_route_refusals(L, bad):
    a = {**GOOD, **bad}
    buf = (ctypes.c_uint8 * 64)()
    rc = L.qmm_moe_route_scored(buf, a["tokens"], a["experts"], a["topk"], a["score"], None, a["groups"],
                                a["topk_groups"], a["group_top"], 1, a["scale"], buf, buf, buf, buf, buf, None, 0, None)
    assert rc == 1 and L.qmm_last_error()


def test_route_workspace(L):
    buf = (ctypes.c_uint8 * 64)()
    assert L.qmm_moe_route_scored_workspace_size(4, 256, 8) == 0 and L.qmm_moe_route_scored_workspace_size(16, 64, 8) == 0
    need = L.qmm_moe_route_scored_workspace_size(17, 256, 8)
    assert need >= 17 * 8 * 6 and L.qmm_moe_route_scored_workspace_size(1, 257, 8) > 0
    assert L.qmm_moe_route_scored_workspace_size(0, 256, 8) == 0
    for ws, n in ((None, 0), (buf, need - 1)):
        assert L.qmm_moe_route_scored(buf, 17, 256, 8, 0, None, 1, 1, 1, 1, 1.0, buf, buf, buf, buf, buf, ws, n, None) == 1
    assert L.qmm_moe_route_scored(buf, 1, 8, 2, 0, None, 1, 1, 1, 1, 1.0, None, buf, buf, buf, buf, None, 0, None) == 1


def test_python_refusals():
    import torch
    from inference_amd import GgmlDType, QmmError, QTensor, moe_route
    with pytest.raises(QmmError, match="need a score"):
        moe_route(torch.zeros(2, 8), 2, groups=2)
    with pytest.raises(QmmError, match="need a score"):
        moe_route(torch.zeros(2, 8), 2, bias=torch.zeros(8))
    with pytest.raises(QmmError, match="tokens, experts"):
        moe_route(torch.zeros(8), 2, score="softmax")
    with pytest.raises(QmmError, match="activation-only"):
        QTensor.from_ggml(bytes(49), GgmlDType.MXFP6X2, (1, 32))
    with pytest.raises(QmmError, match="activation-only"):
        QTensor.quantize(torch.zeros(1, 32), GgmlDType.MXFP6X2)
    with pytest.raises(QmmError, match="GPU"):
        QTensor.quantize(torch.zeros(1, 32), GgmlDType.MXFP4)
