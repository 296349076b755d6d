"""Upstream gradients that are not finite (a scaled loss that overflowed): padded rows, and rows
whose own gradients are 0, get zeros all the same, and their logits are not read."""

import numpy as np
import pytest

from test_gpu_token_logp import logits_of

pytestmark = pytest.mark.gpu

UPSTREAMS = [float("inf"), float("-inf"), float("nan")]


@pytest.mark.parametrize("up", UPSTREAMS)
@pytest.mark.parametrize("c", [7, 300, 5003, 70001])
def test_backward(hip, c, up):
    x = logits_of(6, c, 91)
    ids = np.array([0, -1, c - 1, c // 2, 1, 2], np.int64)
    D = hip.DeviceArray.from_numpy
    di = D(ids)
    _, _, saved = hip.token_logp_fwd(D(x), di)
    x[[1, 3]] = np.nan  # not read
    gl = np.array([1.0, 2.0, -0.5, 0.0, 0.0, 1.0], np.float32)
    gh = np.array([0.5, 1.0, 0.0, 0.0, 1.0, 0.0], np.float32)
    gloss = D(np.array([up], np.float32))
    for a, b in ((gl, None), (gl, gh), (None, gh)):
        got = hip.token_logp_bwd(D(x), di, saved, None if a is None else D(a), None if b is None else D(b), gloss).numpy()
        zero = (ids < 0) | ((a is None) | (gl == 0)) & ((b is None) | (gh == 0))
        assert zero[[1, 3]].all() and not zero.all()
        assert (got[zero] == 0).all(), "rows that do not count"
        assert not np.isfinite(got[~zero]).any(), "the others go with the upstream"


@pytest.mark.parametrize("up", UPSTREAMS)
def test_losses(hip, up):
    """Rows of weight 0, clipped ones, and rows behind the last sequence."""
    import oxitorch_amd as ox
    from oxitorch_amd.nn import functional as F

    x = logits_of(6, 500, 93)
    ids = x.argmax(1).astype(np.int64)
    t = ox.from_numpy(x, True)
    w = np.array([1, 1, 0, 1, 1, 0], np.float32)
    adv = np.array([1, 0, 1, -1, 2, 1], np.float32)
    (F.policy_loss(t, ids, adv, weights=w) * up).backward()
    g = t.grad.numpy()
    assert (g[[1, 2, 5]] == 0).all() and not np.isfinite(g[[0, 3, 4]]).any()
    t.zero_grad()
    (F.preference_loss(t, ids, [[2, 2]]) * up).backward()
    g = t.grad.numpy()
    assert (g[4:] == 0).all() and not np.isfinite(g[:4]).any()
