"""moe_ffn refuses operands that its kernels would read past, before any call of the library: fewer rows of logits than
tokens, rows of another width than the experts', a shared expert's gate of another length or device."""
from types import SimpleNamespace

import pytest
import torch

from inference_amd import GgmlDType, QmmError, moe_ffn, qmm

T, H, E, F = 5, 256, 4, 512


def stack(dtype, n, k):
    return SimpleNamespace(shape=(n, k), device=torch.device("cpu"), handle=1, _dtype=dtype, dtype=lambda: dtype)


@pytest.mark.parametrize("dtype", [GgmlDType.Q4K, GgmlDType.Q8_0, GgmlDType.MXFP4])
@pytest.mark.parametrize("score", [None, "sigmoid"])
@pytest.mark.parametrize("case,match", [
    (dict(x=(T, H + 256)), "rows"), (dict(x=(T, H - 32)), "rows"), (dict(x=(H,)), "rows"), (dict(logits=(T - 1, E)), "logits"),
    (dict(logits=(T * E,)), "logits"), (dict(logits_device="meta"), "logits on meta"), (dict(gate=(H - 1,)), "gate must"),
    (dict(gate=(H + 1,)), "gate must"), (dict(gate=(0,)), "gate must"), (dict(gate=(H,), gate_device="meta"), "gate must")])
def test_refused_on_the_host(monkeypatch, dtype, score, case, match):
    def lib():
        raise AssertionError("a call of the library")

    monkeypatch.setattr(qmm, "lib", lib)
    w = [stack(dtype, E * F, H), stack(dtype, E * F, H), stack(dtype, E * H, F)]
    shared = [stack(dtype, F, H), stack(dtype, F, H), stack(dtype, H, F)]
    x = torch.zeros(case.get("x", (T, H)))
    lg = torch.zeros(case.get("logits", (T, E)), device=case.get("logits_device", "cpu"))
    kw = {}
    if "gate" in case:
        kw = dict(shared=tuple(shared), shared_gate=torch.zeros(case["gate"], device=case.get("gate_device", "cpu")))
    with pytest.raises(QmmError, match=match) as err:
        moe_ffn(x, lg, *w, 2, score=score, **kw)
    assert err.value.status == qmm.QMM_ERR_INVALID
