"""QMatMul's work around the C call, followed on the host: which calls query and allocate a workspace."""
from types import SimpleNamespace

import pytest
import torch

from inference_amd import GgmlDType, QMatMul, qmm


@pytest.fixture
def calls(monkeypatch):
    """The names of the library's calls, none of which does anything."""
    seen = []

    def entry(name, value):
        return lambda *a: (seen.append(name), value)[1]

    fake = SimpleNamespace(qmm_matmul_workspace_size=entry("size", 256), qmm_matmul=entry("matmul", 0),
                           qmm_linear_workspace_size=entry("size", 256), qmm_linear=entry("linear", 0))
    monkeypatch.setattr(qmm, "lib", lambda: fake)
    monkeypatch.setattr(qmm, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)
    return seen


@pytest.mark.parametrize("dtype", [GgmlDType.Q4K, GgmlDType.Q6K, GgmlDType.Q8_0, GgmlDType.MXFP4])
@pytest.mark.parametrize("m,k", [(1, 4096), (2, 16384), (1, 16640), (2, 28672), (3, 256), (3, 16640)])
def test_rows_that_ask_for_a_workspace(calls, dtype, m, k):
    """Above two rows; of an MXFP4 weight also one and two rows too long for its kernel."""
    qt = SimpleNamespace(shape=(8, k), device=torch.device("cpu"), handle=1, _dtype=dtype, dtype=lambda: dtype)
    x = torch.zeros(m, k)
    wants = ["size"] if m > 2 or (dtype == GgmlDType.MXFP4 and k > 16384) else []
    assert QMatMul(qt).forward(x).shape == (m, 8)
    assert calls == wants + ["matmul"]
    if dtype == GgmlDType.MXFP4:
        calls.clear()
        assert QMatMul(qt).linear(x.bfloat16()).shape == (m, 8)
        assert calls == wants + ["linear"]
