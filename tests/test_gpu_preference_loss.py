"""The preference loss of pairs (oxi_preference_loss_fwd) and its gradient against
float64; the bounds are derived in token_oracle.py."""

import numpy as np
import pytest

from conftest import rng
from test_gpu_token_logp import chosen, logits_of
from token_oracle import Rows, near, preference

pytestmark = pytest.mark.gpu


def check(hip, x, ids, starts, ref=None, what="", up=-0.75, **kw):
    D = lambda a: None if a is None else hip.DeviceArray.from_numpy(a)  # noqa: E731
    n, c = x.shape
    at = np.arange(n)
    on = (ids >= 0) & (ids < c) & (at >= starts[0]) & (at < starts[-1])
    r = Rows(x, ids, 1.0, on)
    w = preference(r, starts, ref, **kw)
    args = (D(x), D(ids), D(np.asarray(starts, np.int64)), D(ref))
    loss, pair, S, coef, saved, dx = hip.preference_loss_fwd(*args, **kw, need_grad=True)
    near(S.numpy(), w["S"], w["bS"], f"{what} sequences")
    near(pair.numpy(), w["pair"], w["bpair"], f"{what} pairs")
    near(loss.numpy(), [w["loss"]], w["bloss"], f"{what} loss")
    near(coef.numpy(), w["coef"], w["bcoef"], f"{what} coefficients")
    near(dx.numpy(), *r.gradient(w["coef"], None, w["bcoef"]), f"{what} gradient")
    again = hip.preference_loss_fwd(*args, **kw)
    assert again[5] is None
    for p, q in zip((loss, pair, S, coef), again):
        assert np.array_equal(p.numpy(), q.numpy(), equal_nan=True), "the gradient changes the loss"
    back = hip.token_logp_bwd(args[0], args[1], again[4], again[3], None, D(np.array([up], np.float32))).numpy()
    near(back, *r.gradient(w["coef"] * up, None, w["bcoef"] * abs(up)), f"{what} backward")
    return w


def pairs_of(lengths, c, seed, prompt=0.25):
    """Logits and ids of sequences back to back, the first share of each being the prompt's; reference values."""
    n = sum(lengths)
    x = logits_of(n, c, seed)
    ids = chosen(x, seed + 1)
    starts = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)
    for a, l in zip(starts, lengths):
        ids[a:a + min(l - 1, int(l * prompt))] = -1
    ref = (Rows(x, ids).logp + 0.3 * rng(seed + 2).standard_normal(n)).astype(np.float32)
    return x, ids, starts, ref


KINDS = [dict(kind="sigmoid", beta=0.1), dict(kind="sigmoid", beta=0.5, smoothing=0.1, margin=0.3),
         dict(kind="sigmoid", average=True, beta=2.0, margin=0.5), dict(kind="hinge", beta=0.05),
         dict(kind="ipo", beta=0.2), dict(kind="ipo", average=True, beta=0.5)]


@pytest.mark.parametrize("kw", KINDS, ids=lambda k: "-".join(str(v) for v in k.values()))
@pytest.mark.parametrize("c", [3, 40, 1003, 32000])
def test_kinds(hip, kw, c):
    x, ids, starts, ref = pairs_of([7, 3, 1, 5, 12, 12], c, c + 1)
    check(hip, x, ids, starts, ref, what="with a reference", **kw)
    check(hip, x, ids, starts, None, what="without", **kw)


@pytest.mark.parametrize("lengths,c", [([300, 260], 257), ([1, 1] * 60, 65), ([40, 30, 25, 50], 8195), ([9, 8], 70001),
                                       ([3, 2], 131075), ([700, 1], 40)])
def test_lengths(hip, lengths, c):
    x, ids, starts, ref = pairs_of(lengths, c, 61)
    check(hip, x, ids, starts, ref, beta=0.1, what=str(lengths))


def test_pairs_that_are_decided(hip):
    """Log-ratios so far apart that a sigmoid in 32 bits is 0 or 1: the loss and its slope keep their digits."""
    c = 50
    x = logits_of(8, c, 63)
    ids = x.argmin(1).astype(np.int64)
    starts = np.array([0, 2, 4, 6, 8], np.int64)
    ref = np.array([0, 0, -30, -30, -40, -40, 0, 0], np.float32)
    for kw in (dict(beta=1.0), dict(beta=0.2), dict(kind="hinge", beta=1.0), dict(beta=1.0, smoothing=0.25)):
        check(hip, x, ids, starts, ref, **kw)


def test_empty_sequences_and_prompts_alone(hip):
    """Sequences of no rows or of the prompt alone have S = 0."""
    c = 77
    x = logits_of(9, c, 65)
    ids = chosen(x, 66)
    ids[3:6] = -1
    for average in (False, True):
        w = check(hip, x, ids, np.array([0, 3, 6, 6, 9], np.int64), None, average=average)
        assert w["S"][1] == 0 and w["S"][2] == 0
    w = check(hip, x, np.full(9, -1, np.int64), np.array([0, 3, 9], np.int64), None)
    assert abs(w["loss"] - np.log(2)) < 1e-12


def test_rows_outside_the_sequences(hip):
    """Rows before the first and behind the last sequence are padding, and are not read."""
    c = 300
    x = logits_of(12, c, 67)
    ids = chosen(x, 68)
    starts = np.array([2, 5, 9], np.int64)
    x[:2] = np.nan
    x[9:] = np.nan
    D = hip.DeviceArray.from_numpy
    loss, pair, S, coef, saved, dx = hip.preference_loss_fwd(D(x), D(ids), D(starts), need_grad=True)
    for v in (loss, pair, S, coef, dx):
        assert np.isfinite(v.numpy()).all()
    assert (dx.numpy()[:2] == 0).all() and (dx.numpy()[9:] == 0).all()
    x[:2] = x[9:] = 0.0
    check(hip, x, ids, starts)


def test_bounds_that_are_wrong_raise_the_guard(hip):
    x = logits_of(6, 40, 69)
    ids = chosen(x, 70)
    D = hip.DeviceArray.from_numpy
    hip.sync()
    for starts in ([0, 3, 7], [0, 4, 2], [-1, 2, 4]):
        got = hip.preference_loss_fwd(D(x), D(ids), D(np.array(starts, np.int64)), need_grad=True)
        with pytest.raises(RuntimeError):
            hip.sync()
        assert np.isfinite(got[5].numpy()).all()


def test_no_pairs_and_no_rows(hip):
    x = logits_of(3, 20, 71)
    ids = chosen(x, 72)
    D = hip.DeviceArray.from_numpy
    loss, pair, S, coef, saved, dx = hip.preference_loss_fwd(D(x), D(ids), D(np.zeros(1, np.int64)), need_grad=True)
    assert loss.numpy()[0] == 0 and (dx.numpy() == 0).all() and (coef.numpy() == 0).all()
    loss, pair, S, *_ = hip.preference_loss_fwd(hip.DeviceArray((0, 20)), hip.DeviceArray((0,), np.int64),
                                                D(np.zeros(5, np.int64)), margin=0.5)
    assert np.allclose(pair.numpy(), np.log1p(np.exp(0.5)), rtol=1e-6) and (S.numpy() == 0).all()


@pytest.mark.parametrize("c", [30, 5003, 32000, 70001])
def test_padded_rows_are_not_read(hip, c):
    x, ids, starts, ref = pairs_of([6, 5], c, 73)
    x[ids < 0] = np.nan
    ref[ids < 0] = np.nan
    D = hip.DeviceArray.from_numpy
    got = hip.preference_loss_fwd(D(x), D(ids), D(starts), D(ref), need_grad=True)
    for v in (got[0], got[1], got[2], got[3], got[5]):
        assert np.isfinite(v.numpy()).all()
    x[ids < 0] = 0.0
    ref[ids < 0] = 0.0
    check(hip, x, ids, starts, ref)


def test_one_pair_that_is_nan(hip):
    """A row of NaN spoils its own pair; the others' gradients stay."""
    x, ids, starts, ref = pairs_of([4, 4, 4, 4], 90, 75)
    row = int(np.flatnonzero(ids[4:8] >= 0)[0]) + 4
    x[row, 3] = np.nan
    D = hip.DeviceArray.from_numpy
    loss, pair, S, coef, saved, dx = hip.preference_loss_fwd(D(x), D(ids), D(starts), D(ref), need_grad=True)
    assert np.isnan(loss.numpy()[0]) and np.isnan(pair.numpy()[0]) and np.isfinite(pair.numpy()[1])
    assert np.isfinite(dx.numpy()[8:]).all()


def test_workspace_of_the_caller(hip):
    x, ids, starts, ref = pairs_of([30, 20], 9001, 77)
    a = [hip.DeviceArray.from_numpy(v) for v in (x, ids, starts, ref)]
    ws = hip.DeviceArray((hip.preference_loss_workspace(50, 9001),), np.uint8)
    for p, q in zip(hip.preference_loss_fwd(*a, need_grad=True), hip.preference_loss_fwd(*a, need_grad=True, workspace=ws)):
        assert np.array_equal(p.numpy(), q.numpy())
