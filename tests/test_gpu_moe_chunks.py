"""Expert FFNs with a shared expert over more tokens than one chunk, where the last chunk's shared expert needs more
workspace than a whole chunk's (its products split K): every token's row as in a call of its own part, and nothing
written past the workspace that the query names."""
import pytest
import torch

from inference_amd import GgmlDType, QTensor, moe_ffn, qmm

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
GUARD = 32 << 20


def experts(dtypes, e, h, f, fs, shared_dtypes):
    g = torch.Generator(device=DEV)
    g.manual_seed(e + h)

    def q(n, k, dt):
        return QTensor.quantize(torch.randn(n, k, generator=g, device=DEV) * 0.02, dt)

    return ([q(e * f, h, dtypes[0]), q(e * f, h, dtypes[0]), q(e * h, f, dtypes[1])],
            [q(fs, h, shared_dtypes[0]), q(fs, h, shared_dtypes[0]), q(h, fs, shared_dtypes[1])], g)


def guarded_call(x, lg, k, w, shared, score):
    """The call through the C entry, with a guard behind a workspace of exactly the queried size."""
    L, (t, h), e = qmm.lib(), x.shape, lg.shape[1]
    hw, hs = [v.handle for v in w], [v.handle for v in shared]
    size = L.qmm_moe_ffn_scored_workspace_size if score else L.qmm_moe_ffn_ex_workspace_size
    n = size(hw[0], hw[2], t, e, k, *hs)
    ws = torch.empty(n + GUARD, dtype=torch.uint8, device=DEV)
    ws[n:] = 0xA5
    out = torch.empty(t, h, device=DEV)
    s = qmm._stream(DEV)
    if score:
        rc = L.qmm_moe_ffn_scored(x.data_ptr(), 0, t, h, lg.data_ptr(), e, k, 1, None, 1, 1, 1, 1, 1.0, *hw, *hs, None,
                                  out.data_ptr(), 0, h, ws.data_ptr(), n, s)
    else:
        rc = L.qmm_moe_ffn_ex(x.data_ptr(), t, h, lg.data_ptr(), e, k, 1, 1.0, *hw, *hs, None, out.data_ptr(), h,
                              ws.data_ptr(), n, s)
    qmm._check(rc)
    assert bool((ws[n:] == 0xA5).all())
    return out


def test_mxfp4_experts_and_a_q4k_shared_expert():
    e, k, h, f, fs, chunk, rest = 16, 16, 2048, 32, 1024, 2048, 976
    mx = (GgmlDType.MXFP4, GgmlDType.MXFP4)
    w, shared, g = experts(mx, e, h, f, fs, (GgmlDType.Q4K, GgmlDType.Q6K))
    L, hs = qmm.lib(), [v.handle for v in shared]
    # (the sizes that this is about; no launch before they are seen to be covered)
    assert L.qmm_ffn_workspace_size(*hs, rest, 0) > L.qmm_ffn_workspace_size(*hs, chunk, 0)
    t = chunk + rest
    total, routed = (L.qmm_moe_ffn_scored_workspace_size(w[0].handle, w[2].handle, t, e, k, *s) for s in (hs, (None,) * 3))
    assert total >= routed + 4 * chunk * h + L.qmm_ffn_workspace_size(*hs, rest, 0)
    x, lg = torch.randn(t, h, generator=g, device=DEV), torch.randn(t, e, generator=g, device=DEV)
    for score in (False, True):
        y = guarded_call(x, lg, k, w, shared, score)
        for a, b in ((0, chunk), (chunk, t)):
            part = moe_ffn(x[a:b], lg[a:b], *w, k, shared=tuple(shared), score="sigmoid" if score else None)
            assert torch.equal(y[a:b], part)


@pytest.mark.parametrize("score", [False, True])
def test_q4k_experts_and_a_wide_shared_expert(score):
    e, k, h, f, fs, chunk, rest = 8, 1, 512, 256, 8192, 4096, 3584
    q = (GgmlDType.Q4K, GgmlDType.Q6K)
    w, shared, g = experts(q, e, h, f, fs, q)
    L, hs = qmm.lib(), [v.handle for v in shared]
    size = [L.qmm_moe_ffn_ex_workspace_size(w[0].handle, w[2].handle, t, e, k, *hs) for t in (chunk, rest, chunk + rest)]
    assert size[1] > size[0] and size[2] == size[1]
    t = chunk + rest
    x, lg = torch.randn(t, h, generator=g, device=DEV), torch.randn(t, e, generator=g, device=DEV)
    y = guarded_call(x, lg, k, w, shared, score)
    for a, b in ((0, chunk), (chunk, t)):
        assert torch.equal(y[a:b], moe_ffn(x[a:b], lg[a:b], *w, k, shared=tuple(shared), score="sigmoid" if score else None))
