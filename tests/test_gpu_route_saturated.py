"""Scored routing where scores in 64 bits are equal though the logits are not: the lower expert goes first.

1 / (1 + exp(-l)) rounds to 1 where exp(-l) < 2^-53, from l = 53 ln 2 = 36.74 on (at 38: exp(-38) = 3.1e-17 against
1.1e-16), and to 0 where exp(-l) overflows, from l = -709.8 down. Softmax scores are not near a constant there: their
order is the logits'."""
import numpy as np
import pytest
import torch

from inference_amd import moe_route
from oracle import mx

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def selections(lg, k, **kw):
    counts, offsets, ptok, pw, tp = (v.cpu().numpy() for v in moe_route(torch.from_numpy(lg).to(DEV), k, **kw))
    ids = np.searchsorted(offsets, tp, side="right") - 1
    return ids.reshape(len(lg), k), pw[tp].reshape(len(lg), k)


@pytest.mark.parametrize("t", [1, 5, 40])
@pytest.mark.parametrize("n", [8, 130, 520])
def test_saturated_sigmoid_scores_tie(t, n):
    rng = np.random.default_rng(n + t)
    high = np.stack([rng.permutation(n) for _ in range(t)]).astype(np.float32) + 38
    low = -high - 700
    for lg, score in ((high, 1.0), (low, 0.0)):
        ids, w = selections(lg, 4, score="sigmoid", renormalize=False)
        np.testing.assert_array_equal(ids, np.tile(np.arange(4), (t, 1)))
        np.testing.assert_array_equal(w, np.float32(score))
        want, _ = mx.route(lg, 4, score="sigmoid")
        np.testing.assert_array_equal(ids, want)
    # one below the others stays behind; a bias decides between equal scores
    lg = high.copy()
    lg[:, 0] = 30
    assert (selections(lg, 4, score="sigmoid")[0] == np.arange(1, 5)).all()
    bias = torch.zeros(n, device=DEV)
    bias[n - 4:] = 2.0 ** -20
    assert (selections(high, 4, score="sigmoid", bias=bias)[0] == np.arange(n - 4, n)).all()
    # by softmax the same logits are ordered
    want = np.sort(np.argsort(-high, axis=1)[:, :4], axis=1)
    np.testing.assert_array_equal(selections(high, 4, score="softmax")[0], want)
