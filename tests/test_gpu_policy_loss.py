"""The clipped policy loss (oxi_policy_loss_fwd) and its gradient against float64;
the bounds are derived in token_oracle.py."""

import numpy as np
import pytest

from conftest import rng
from test_gpu_token_logp import chosen, logits_of
from token_oracle import Rows, near, policy

pytestmark = pytest.mark.gpu


def case(n, c, seed, pad=0.2, moved=0.2, T=1.0, clip=(0.2, 0.28), clip_max=3.0):
    """Logits, ids, advantages, old and reference log-probabilities; no ratio on an edge of the clipping."""
    r = rng(seed)
    x = logits_of(n, c, seed)
    ids = chosen(x, seed + 1, pad)
    rows = Rows(x, ids, T)
    adv = (r.standard_normal(n) * (r.random(n) > 0.1)).astype(np.float32)
    step = moved * r.standard_normal(n)
    for edge in (1 - clip[0], 1 + clip[1], clip_max):
        step = np.where(np.abs(np.exp(step) - edge) < 1e-3, step + 5e-3, step)
    old = (rows.logp - step).astype(np.float32)
    ref = (rows.logp + 0.3 * r.standard_normal(n)).astype(np.float32)
    return x, ids, adv, old, ref


def check(hip, x, ids, adv, old=None, ref=None, weights=None, T=1.0, what="", **kw):
    D = lambda a: None if a is None else hip.DeviceArray.from_numpy(a)  # noqa: E731
    n, c = x.shape
    on = (ids >= 0) & (ids < c)
    if weights is not None:
        on &= weights != 0
    r = Rows(x, ids, T, on)
    w = policy(r, adv, old, ref, weights, **kw)
    args = (D(x), D(ids), D(adv), D(old), D(ref), D(weights), T)
    names = dict(clip=kw.get("clip", (0.2, 0.2)), clip_max=kw.get("clip_max", 0.0), kl_coef=kw.get("kl", 0.0),
                 entropy_coef=kw.get("ent", 0.0), divisor=kw.get("divisor", 1.0))
    out, rows, logp, coef, saved, dx = hip.policy_loss_fwd(*args, **names, need_grad=True)
    near(rows.numpy(), w["rows"], w["brows"], f"{what} rows")
    near(out.numpy(), w["out"], w["bout"], f"{what} out")
    near(logp.numpy(), r.logp, r.b_logp, f"{what} logp")
    near(coef.numpy()[0], w["cl"], w["bcl"], f"{what} coefficient of logp")
    near(coef.numpy()[1], w["ch"], w["bch"], f"{what} coefficient of the entropy")
    ent = kw.get("ent", 0.0) != 0
    near(dx.numpy(), *r.gradient(w["cl"], w["ch"] if ent else None, w["bcl"], w["bch"] if ent else 0.0), f"{what} gradient")
    # without the gradient the same numbers; the backward for another upstream
    again = hip.policy_loss_fwd(*args, **names)
    assert again[5] is None
    for p, q in zip((out, rows, logp, coef), again):
        assert np.array_equal(p.numpy(), q.numpy(), equal_nan=True), "the gradient changes the loss"
    up = np.array([-0.625], np.float32)
    co = coef.numpy()
    gl, gh = D(co[0].copy()), D(co[1].copy()) if ent else None
    back = hip.token_logp_bwd(args[0], args[1], again[4], gl, gh, D(up), T).numpy()
    f = float(up[0])
    near(back, *r.gradient(w["cl"] * f, w["ch"] * f if ent else None, w["bcl"] * abs(f), w["bch"] * abs(f) if ent else 0.0),
         f"{what} backward")
    return w


@pytest.mark.parametrize("c", [1, 2, 5, 8, 33, 64, 257, 1000, 1003, 2051, 4096, 8195, 12289, 16411, 20000, 32000, 32801,
                               50257, 65536, 65571, 131072, 150001])
def test_widths(hip, c):
    x, ids, adv, old, ref = case(7, c, c)
    check(hip, x, ids, adv, old, ref, clip=(0.2, 0.28), clip_max=3.0, kl=0.04, ent=0.01, divisor=5.0, what=f"c={c}")
    check(hip, x, ids, adv, old, divisor=5.0, what=f"c={c}, no KL")


@pytest.mark.parametrize("n,c", [(700, 1003), (3000, 65), (300, 32000), (900, 8195)])
@pytest.mark.parametrize("ent", [0.0, 0.003])
def test_many_rows(hip, n, c, ent):
    x, ids, adv, old, ref = case(n, c, 41)
    w = rng(42).random(n).astype(np.float32)
    w[::7] = 0.0
    got = check(hip, x, ids, adv, old, ref, w, clip=(0.2, 0.28), clip_max=3.0, kl=0.04, ent=ent, divisor=64.0,
                what=f"{(n, c)}")
    assert 0 < got["rows"][3].sum() < n


@pytest.mark.parametrize("T", [0.5, 1.7])
def test_temperatures(hip, T):
    x, ids, adv, old, ref = case(20, 3001, 43, T=T)
    check(hip, x, ids, adv, old, ref, T=T, clip=(0.2, 0.28), clip_max=3.0, kl=0.1, ent=0.02, divisor=20.0, what=f"T={T}")


def test_the_policy_that_sampled(hip):
    """Without old log-probabilities the ratio is 1: nothing is clipped, the gradient is the plain policy gradient."""
    x, ids, adv, _, ref = case(30, 777, 45)
    w = check(hip, x, ids, adv, divisor=30.0)
    assert (w["rows"][3] == 0).all()
    check(hip, x, ids, adv, ref=ref, kl=0.2, divisor=30.0)


def test_each_side_of_the_clipping(hip):
    """Every sign of the advantage with the ratio below, between, above, and past clip_max; its gradient is 0 where
    the bound is met."""
    x = logits_of(12, 300, 47)
    ids = x.argmax(1).astype(np.int64)
    lp = Rows(x, ids).logp
    ratio = np.array([0.5, 1.0, 1.5, 5.0] * 3)
    adv = np.repeat([1.5, 0.0, -1.5], 4).astype(np.float32)
    old = (lp - np.log(ratio)).astype(np.float32)
    w = check(hip, x, ids, adv, old, clip=(0.2, 0.28), clip_max=3.0)
    assert w["rows"][3].tolist() == [0, 0, 1, 1, 0, 0, 0, 0, 1, 0, 0, 1]
    w = check(hip, x, ids, adv, old, clip=(0.2, float("inf")))
    assert w["rows"][3].tolist() == [0, 0, 0, 0, 0, 0, 0, 0, 1, 0, 0, 0]
    w = check(hip, x, ids, adv, old, clip=(1.0, 0.0))  # ratios down to 0, none above 1
    assert np.delete(w["rows"][3], 1).tolist() == [0, 1, 1, 0, 0, 0, 0, 0, 0, 0, 0]  # row 1 lies on the edge itself


def test_reference_that_is_near_or_far(hip):
    """k of a policy next to its reference is d^2/2, not a difference of rounded terms; far ones keep theirs."""
    x = logits_of(8, 2000, 49)
    ids = x.argmax(1).astype(np.int64)
    lp = Rows(x, ids).logp
    ref = (lp + np.array([1e-3, -1e-3, 0.4999, 0.5001, -0.5, 20.0, -30.0, -80.0])).astype(np.float32)
    adv = np.ones(8, np.float32)
    check(hip, x, ids, adv, ref=ref, kl=0.5, divisor=8.0)
    check(hip, x, ids, adv, ref=ref, kl=0.0, divisor=8.0, what="reported only")


def test_masked_reference_and_old(hip):
    """A reference or an old policy that excluded the token: the definition's infinities, in that row alone."""
    x = logits_of(5, 100, 51)
    ids = x.argmax(1).astype(np.int64)
    adv = np.ones(5, np.float32)
    ref = np.zeros(5, np.float32)
    ref[1] = -np.inf
    D = hip.DeviceArray.from_numpy
    out, rows, logp, coef, saved, dx = hip.policy_loss_fwd(D(x), D(ids), D(adv), None, D(ref), None, 1.0, kl_coef=0.5,
                                                           divisor=5.0, need_grad=True)
    k = rows.numpy()[1]
    assert k[1] == np.inf and np.isfinite(np.delete(k, 1)).all()
    assert np.isfinite(dx.numpy()).all() and np.isfinite(coef.numpy()).all()
    old = np.zeros(5, np.float32)
    old[2] = -np.inf  # the ratio is infinite: with A > 0 the clipping bounds it
    out, rows, logp, coef, saved, dx = hip.policy_loss_fwd(D(x), D(ids), D(adv), D(old), None, None, 1.0, divisor=5.0,
                                                           need_grad=True)
    assert np.isfinite(rows.numpy()).all() and rows.numpy()[3][2] == 1 and np.isfinite(dx.numpy()).all()


@pytest.mark.parametrize("c", [40, 5003, 32000, 70001])
def test_padded_and_weightless_rows_are_not_read(hip, c):
    """NaN anywhere in rows that do not count changes nothing."""
    x, ids, adv, old, ref = case(9, c, 53, pad=0.0)
    w = np.ones(9, np.float32)
    ids[2], ids[5], w[7] = -1, -9, 0.0
    kw = dict(clip=(0.2, 0.28), clip_max=3.0, kl=0.05, ent=0.01, divisor=6.0)
    off = np.array([2, 5, 7])
    for a in (x, adv, old, ref):
        a[off] = np.nan
    w[[2, 5]] = np.nan  # of padded rows
    D = hip.DeviceArray.from_numpy
    out, rows, logp, coef, saved, dx = hip.policy_loss_fwd(D(x), D(ids), D(adv), D(old), D(ref), D(w), 1.0, (0.2, 0.28),
                                                           3.0, 0.05, 0.01, 6.0, need_grad=True)
    for v in (out, rows, logp, coef, dx):
        assert np.isfinite(v.numpy()).all()
    assert (dx.numpy()[off] == 0).all() and (rows.numpy()[:, off] == 0).all() and (coef.numpy()[:, off] == 0).all()
    for a in (x, adv, old, ref):
        a[off] = 0.0
    w[[2, 5]] = 1.0
    check(hip, x, ids, adv, old, ref, w, what="cleared", **kw)


def test_all_rows_padded_and_none(hip):
    x = logits_of(4, 60, 55)
    ids = np.full(4, -1, np.int64)
    adv = np.ones(4, np.float32)
    w = check(hip, x, ids, adv, divisor=1.0)
    assert (w["out"] == 0).all()
    out = hip.DeviceArray.from_numpy(np.full(4, 5.0, np.float32))
    hip.call("oxi_policy_loss_fwd", *[None] * 6, out.ptr, *[None] * 6, 0, 60, 1.0, 0.2, 0.2, 0.0, 0.0, 0.0, 1.0)
    assert (out.numpy() == 0).all()


def test_workspace_of_the_caller(hip):
    x, ids, adv, old, ref = case(12, 9001, 57)
    D = hip.DeviceArray.from_numpy
    a = [D(v) for v in (x, ids, adv, old, ref)]
    ws = hip.DeviceArray((max(1, hip.policy_loss_workspace(12, 9001)),), np.uint8)
    for p, q in zip(hip.policy_loss_fwd(*a, kl_coef=0.1, need_grad=True), hip.policy_loss_fwd(*a, kl_coef=0.1, need_grad=True,
                                                                                              workspace=ws)):
        assert np.array_equal(p.numpy(), q.numpy())
