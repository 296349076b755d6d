"""The policy loss over rows that hold no distribution (all classes at -inf, NaN, +inf): NaN
in that row's loss and in its gradient, by either way to the gradient, and in no other row."""

import numpy as np
import pytest

from test_gpu_token_logp import logits_of
from token_oracle import Rows

pytestmark = pytest.mark.gpu

BAD = np.array([False, True, True, True, False])


@pytest.mark.parametrize("with_old", [False, True])
@pytest.mark.parametrize("ent", [0.0, 0.01])
@pytest.mark.parametrize("advantage", [0.0, 1.0, -2.0])
@pytest.mark.parametrize("c", [5, 40, 300, 5003, 32000, 50257, 530001])
def test_rows_without_a_distribution(hip, c, advantage, ent, with_old):
    x = logits_of(5, c, 81)
    ids = np.full(5, 1, np.int64)
    old = (Rows(x, ids).logp - 0.05).astype(np.float32)
    x[1] = -np.inf
    x[2, c // 2] = np.nan
    x[3, c - 1] = np.inf
    D = hip.DeviceArray.from_numpy
    dx, di = D(x), D(ids)
    adv = D(np.full(5, advantage, np.float32))
    out, rows, logp, coef, saved, d = hip.policy_loss_fwd(dx, di, adv, D(old) if with_old else None, entropy_coef=ent,
                                                          divisor=5.0, need_grad=True)
    assert np.array_equal(np.isnan(rows.numpy()[0]), BAD) and np.array_equal(np.isnan(logp.numpy()), BAD)
    assert np.isnan(out.numpy()[0])
    assert np.array_equal(np.isnan(coef.numpy()[0]), BAD)
    back = hip.token_logp_bwd(dx, di, saved, D(coef.numpy()[0].copy()), D(coef.numpy()[1].copy()) if ent else None)
    for got, what in ((d.numpy(), "one pass"), (back.numpy(), "backward")):
        assert np.isnan(got[BAD]).all(), what
        assert np.isfinite(got[~BAD]).all(), what
    again = hip.policy_loss_fwd(dx, di, adv, D(old) if with_old else None, entropy_coef=ent, divisor=5.0)
    assert np.array_equal(again[1].numpy(), rows.numpy(), equal_nan=True)


def test_a_zero_advantage_bounds_an_infinite_ratio(hip):
    """exp(logp - old) may be infinite where the row has a distribution: nothing is gained there."""
    x = logits_of(3, 100, 83)
    ids = x.argmax(1).astype(np.int64)
    old = np.array([-np.inf, -2000.0, 0.0], np.float32)
    D = hip.DeviceArray.from_numpy
    for high in (0.2, float("inf")):
        out, rows, logp, coef, saved, d = hip.policy_loss_fwd(D(x), D(ids), D(np.zeros(3, np.float32)), D(old),
                                                              clip=(0.2, high), need_grad=True)
        assert (rows.numpy()[0] == 0).all() and (coef.numpy() == 0).all() and (d.numpy() == 0).all()
