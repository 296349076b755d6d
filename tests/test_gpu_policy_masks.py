"""The policy loss over rows with masked classes, against float64 with the bounds of
token_oracle.py: a masked class has probability 0 and no gradient wherever it lies, and
whatever the size of the logits that are left."""

import numpy as np
import pytest

from conftest import rng
from test_gpu_policy_loss import check
from test_gpu_token_logp import logits_of
from token_oracle import Rows

pytestmark = pytest.mark.gpu

CLIP = dict(clip=(0.2, 0.28), clip_max=3.0)


def check_rows(hip, x, ids, T, ent, seed, what):
    """Old and reference log-probabilities around the rows' own, off the clipping's edges; row 0 is clipped."""
    n = len(x)
    r, q = Rows(x, ids, T), rng(seed)
    adv = q.standard_normal(n).astype(np.float32)
    step = 0.2 * q.standard_normal(n)
    adv[0], step[0] = 1.5, 0.5
    for edge in (0.8, 1.28, 3.0):
        step = np.where(np.abs(np.exp(step) - edge) < 1e-3, step + 5e-3, step)
    old = (r.logp - step).astype(np.float32)
    ref = (r.logp + 0.3 * q.standard_normal(n)).astype(np.float32)
    w = check(hip, x, ids, adv, old, ref, T=T, ent=ent, kl=0.04, divisor=float(n), what=what, **CLIP)
    assert w["rows"][3][0] == 1
    w = check(hip, x, ids, adv, old, T=T, ent=ent, divisor=float(n), what=f"{what}, no KL", **CLIP)
    assert w["cl"][0] == 0


@pytest.mark.parametrize("ent", [0.0, 0.01])
@pytest.mark.parametrize("T", [1.0, 0.1])
@pytest.mark.parametrize("level", [-100.0, -20.0, 0.0, 100.0])
@pytest.mark.parametrize("c", [32801, 50257, 131072])
def test_few_classes_left(hip, c, level, T, ent):
    """All but a few classes at -inf: at the row's beginning, at its end, the chosen one far from the others, the
    chosen one alone. The logits that are left lie around `level`, far below 0 too."""
    q = rng(c)
    x = np.full((6, c), -np.inf, np.float32)
    few = lambda: (level + q.standard_normal(9)).astype(np.float32)  # noqa: E731
    x[0, 3:12] = few()
    x[1, 40:49] = few()
    x[2, c - 9:] = few()
    x[3, 100:109] = few()
    x[3, c - 5] = level
    x[4, c - 20:c - 11] = few()
    x[4, 5] = level
    x[5, c // 2] = level
    ids = np.array([4, 44, c - 1, c - 5, 5, c // 2], np.int64)
    check_rows(hip, x, ids, T, ent, 71, f"{level} of {c}, T={T}")


@pytest.mark.parametrize("ent", [0.0, 0.01])
@pytest.mark.parametrize("lowest", [-np.inf, np.finfo(np.float32).min])
@pytest.mark.parametrize("c", [6, 40, 300, 1003, 5003, 12289, 32000, 50257, 131072, 530001])
def test_masked_classes(hip, c, lowest, ent):
    x = logits_of(6, c, 73)
    ids = x.argmax(1).astype(np.int64)
    ids[4] = (ids[4] + 1) % c
    keep = rng(74).random((6, c)) < 0.3
    keep[1] = False  # the chosen class alone
    keep[2, :c // 2] = False
    keep[3, c // 2:] = False
    keep[np.arange(6), ids] = True
    x = np.where(keep, x, np.float32(lowest))
    for T in (1.0, 0.5):
        check_rows(hip, x, ids, T, ent, 75, f"masked with {lowest}, c={c}, T={T}")
