"""The preference loss over rows with masked classes, against float64 with the bounds of token_oracle.py."""

import numpy as np
import pytest

from conftest import rng
from test_gpu_preference_loss import check, pairs_of
from token_oracle import Rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("level", [0.0, -120.0])
@pytest.mark.parametrize("lowest", [-np.inf, np.finfo(np.float32).min])
@pytest.mark.parametrize("c", [6, 40, 300, 5003, 32000, 50257, 140001])
def test_masked_classes(hip, c, lowest, level):
    """Classes masked here and there, one half of the row, all but the chosen one; what is left lies around `level`."""
    x, ids, starts, _ = pairs_of([4, 3, 5, 2], c, 121)
    x += np.float32(level)
    keep = rng(122).random(x.shape) < 0.3
    keep[1] = False
    keep[5, :c // 2] = False
    keep[8, c // 2:] = False
    on = ids >= 0
    keep[np.flatnonzero(on), ids[on]] = True
    x = np.where(keep, x, np.float32(lowest))
    ref = (Rows(x, ids).logp + 0.3 * rng(123).standard_normal(len(ids))).astype(np.float32)
    for kw in (dict(beta=0.1), dict(kind="ipo", average=True, beta=0.5)):
        check(hip, x, ids, starts, ref, what=f"c={c} {lowest} {level}", **kw)


@pytest.mark.parametrize("c", [40, 32000, 50257])
def test_a_chosen_class_that_is_masked(hip, c):
    """A sequence with a token that its policy excludes has S = -inf: the pair's loss is infinite where that is the chosen
    one, and 0 where it is the rejected one, whose gradient is 0 then. The other pair keeps its own."""
    x, ids, _, _ = pairs_of([2, 2, 2, 2, 2, 2], c, 125, prompt=0.0)
    starts = np.array([0, 2, 4, 6, 8, 10, 12], np.int64)
    x[0, ids[0]] = -np.inf  # pair 0, chosen
    x[6, ids[6]] = -np.inf  # pair 1, rejected
    D = hip.DeviceArray.from_numpy
    loss, pair, S, coef, saved, dx = hip.preference_loss_fwd(D(x), D(ids), D(starts), beta=0.5, need_grad=True)
    pair, S, coef, dx = (v.numpy() for v in (pair, S, coef, dx))
    assert S[0] == -np.inf and S[3] == -np.inf and np.isfinite(np.delete(S, [0, 3])).all()
    assert pair[0] == np.inf and pair[1] == 0 and np.isfinite(pair[2]) and loss.numpy()[0] == np.inf
    assert np.isfinite(coef).all() and np.isfinite(dx).all()
    assert (coef[4:8] == 0).all() and (dx[4:8] == 0).all()
    assert (coef[:2] == np.float32(-0.5 / 3)).all() and (coef[2:4] == np.float32(0.5 / 3)).all()
