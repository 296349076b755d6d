"""The rest's term of the distillation loss where the classes that are not listed
lie far below the listed ones, or carry nothing: log-sum-exps of their own in
float64, never 1 less the listed.

Tolerances, u = 2^-24, as in test_gpu_distill: an exponential of (z - m) is off,
relatively, by u (3 |z - m| + 6); a sum adds c/64 + 24 steps. `s` is the softmax
over the classes not listed, by its own maximum; the student's mass there is qr.
The row's loss is formed from masses that balance, so that an error d of a log
enters times |q - p| and squared."""

import numpy as np
import pytest

from conftest import rng
from test_gpu_distill import student_and_teacher, teacher_lse

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def near_one(lse):
    """What a log-sum-exp worked out in float32 may lack of the teacher's whole mass."""
    return 2.0 ** -22 * (1 + abs(float(lse)))


def tail64(x, ids, top, T, lse, divisor):
    n, c = x.shape
    T = float(np.float32(T))
    rows, brow = np.zeros(n), np.zeros(n)
    grads, bgrad = np.zeros((n, c)), np.zeros((n, c))
    seq = (c / 64 + 24) * U
    eps = lambda d: U * (3 * np.minimum(np.abs(d), 110.0) + 6)  # noqa: E731
    for r in range(n):
        z = x[r].astype(np.float64) / T
        keep = [j for j in range(ids.shape[1]) if 0 <= ids[r, j] < c and top[r, j] != -np.inf]
        if not keep:
            continue
        at = ids[r, keep]
        out = np.ones(c, bool)
        out[at] = False
        m = z.max()
        e = np.exp(z - m)
        lq = z - m - np.log(e.sum())
        q = np.exp(lq)
        lp = top[r, keep].astype(np.float64) / T - float(lse[r])
        p = np.exp(lp)
        given = np.zeros(c)
        np.add.at(given, at, p)
        pr = max(1.0 - p.sum(), 0.0)
        empty = not np.isfinite(z[out]).any()
        if empty:
            s, lr, dS = np.zeros(out.sum()), -np.inf, 0.0
        else:
            mr = z[out].max()
            s = np.exp(z[out] - mr)
            lr = mr + np.log(s.sum()) - m - np.log(e.sum())
            s /= s.sum()
            with np.errstate(invalid="ignore"):
                dS = np.where(s > 0, s * eps(z[out] - mr), 0.0).sum() + seq + 2 * U
        qr = np.exp(lr)
        if qr < 2.0 ** -126 and pr <= near_one(lse[r]):
            pr = 0.0
        with np.errstate(invalid="ignore"):
            dT = np.where(~out & (q > 0), q * eps(z - m), 0.0).sum() + seq + 4 * U
        if not empty:
            dT += qr * (dS + eps(mr - m))
        with np.errstate(invalid="ignore"):
            rows[r] = np.where(p > 0, p * (lp - lq[at]), 0.0).sum() + (pr * (np.log(pr) - lr) if pr > 0 else 0.0)
        gap = np.abs(q - given)[~out].sum()
        brow[r] = T * T * (gap * dT + abs(qr - pr) * (dS + dT) + 8 * (dS + dT) ** 2 + 4 * U * abs(rows[r]) + 1e-12)
        rows[r] *= T * T
        brow[r] += U * abs(rows[r])
        g = q - given
        b = np.zeros(c)
        with np.errstate(invalid="ignore"):
            b[~out] = (q * np.where(q > 0, eps(z - m) + 2 * dT + 6 * U, 0.0) + 2 * U * np.abs(g) + U * given)[~out]
        if empty:
            g[out] = 0.0
        else:
            coef = qr - pr
            g[out] = s * coef
            mass = (p.sum() + q[~out].sum()) if p.sum() < 0.5 else qr + pr
            with np.errstate(invalid="ignore"):
                b[out] = s * (abs(coef) * (np.where(s > 0, eps(z[out] - mr), 0.0) + dS + 8 * U) + mass * (dS + 2 * dT + 6 * U))
        grads[r] = g * T / divisor
        bgrad[r] = b * T / divisor + 2e-38 * (1 + T / divisor)
    return rows, brow, grads, bgrad


def run(hip, x, ids, top, T, lse):
    D = hip.DeviceArray.from_numpy
    n = x.shape[0]
    a = (D(x), D(ids), D(top))
    loss, row, slse, rest, grad = hip.distill_fwd(*a, T, D(lse), need_grad=True)
    loss2, row2, _, rest2, _ = hip.distill_fwd(*a, T, D(lse))
    assert np.array_equal(row.numpy(), row2.numpy()) and np.array_equal(rest.numpy(), rest2.numpy())
    back = hip.distill_bwd(*a, slse, rest, D(np.ones(1, np.float32)), T, D(lse))
    return loss.numpy()[0], row.numpy(), rest.numpy(), grad.numpy(), back.numpy()


def check(hip, x, ids, top, T, lse, what=""):
    rows, brow, grads, bgrad = tail64(x, ids, top, T, lse, float(len(x)))
    loss, row, rest, grad, back = run(hip, x, ids, top, T, lse)
    for name, got, want, bound in (("row", row, rows, brow), ("gradient", grad, grads, bgrad), ("backward", back, grads, bgrad)):
        with np.errstate(invalid="ignore"):
            ok = (got == want) | (np.abs(got - want) <= bound)
        assert ok.all(), (what, name, np.argwhere(~ok)[0], got[~ok][0], want[~ok][0], np.broadcast_to(bound, got.shape)[~ok][0])
    with np.errstate(invalid="ignore"):
        mean = rows.sum() / len(x)
        assert loss == mean or abs(loss - mean) <= (brow.sum() / len(x) + 2 * U * abs(mean)), what
    return rows, rest


@pytest.mark.parametrize("c,k", [(7, 3), (40, 4), (515, 8), (1020, 200), (5001, 5), (32000, 6), (70001, 5), (300005, 4)])
@pytest.mark.parametrize("T", [1.0, 0.2, 4.0])
@pytest.mark.parametrize("gaps", [(3, 40, 70), (86, 87.5, 88.2), (88.6, 90, 104), (120, 800, 30000)])
def test_listed_classes_far_above_the_others(hip, c, k, T, gaps):
    """Every mass of the classes not listed from a large one to far below the smallest float. The second row's listed
    classes are all alike, the third's teacher gives them little, the fourth has no entry."""
    print("[case] distill far", c, k, T, gaps, flush=True)
    r = rng(c + k)
    for gap in gaps:
        n = 4
        x = (T * r.standard_normal((n, c))).astype(np.float32)
        ids = np.argsort(r.random((n, c)), 1)[:, :k].astype(np.int64)
        up = (T * (gap + r.standard_normal((n, k)))).astype(np.float32)
        up[1] = np.float32(T * gap)
        np.put_along_axis(x, ids, up, 1)
        top = (T * r.standard_normal((n, k))).astype(np.float32)
        z = top.astype(np.float64) / float(np.float32(T))
        share = np.array([0.7, 0.999, 0.2, 0.5])
        lse = (np.log(np.exp(z).sum(1)) - np.log(share)).astype(np.float32)
        ids[3] = -1
        rows, rest = check(hip, x, ids, top, T, lse, (c, k, T, gap))
        assert np.isfinite(rows).all()
        assert np.isfinite(rest).all()


@pytest.mark.parametrize("n,c,T", [(16, 3, 0.7), (16, 7, 1.0), (64, 24, 1.0), (64, 24, 0.7), (8, 600, 3.0), (4, 1000, 1.0)])
def test_every_class_listed_and_the_sum_as_rounded(hip, n, c, T):
    """k == c: what the rounding of the teacher's log-sum-exp leaves over is compared with nothing."""
    x, ids, top, teacher = student_and_teacher(n, c, c, c)
    lse = teacher_lse(teacher, T)
    p = np.exp(teacher.astype(np.float64) / float(np.float32(T)) - lse.astype(np.float64)[:, None]).sum(1)
    assert (p < 1).any() and (1 - p <= [near_one(v) for v in lse]).all()
    rows, _ = check(hip, x, ids, top, T, lse)
    assert np.isfinite(rows).all()


@pytest.mark.parametrize("c,k", [(7, 3), (40, 4), (515, 8), (5001, 5), (40000, 9), (70001, 5), (300005, 4)])
def test_other_classes_masked(hip, c, k):
    """Logits of -inf (and of the lowest float) at every class not listed. With a teacher that is masked as well the
    loss is that of the listed ones; one with mass there is infinitely far, with a gradient at the listed ones only."""
    r = rng(c)
    n, T = 6, 1.3
    ids = np.argsort(r.random((n, c)), 1)[:, :k].astype(np.int64)
    listed = (2 * r.standard_normal((n, k))).astype(np.float32)
    top = (2 * r.standard_normal((n, k))).astype(np.float32)
    z = top.astype(np.float64) / float(np.float32(T))
    lse = np.log(np.exp(z).sum(1)).astype(np.float32)
    x = np.full((n, c), -np.inf, np.float32)
    np.put_along_axis(x, ids, listed, 1)
    rows, rest = check(hip, x, ids, top, T, lse)
    assert np.isfinite(rows).all() and (rest == -np.inf).all()
    rows, rest = check(hip, x, ids, top, T, (lse + np.float32(0.5)))
    assert (rows == np.inf).all()
    _, _, _, grad, back = run(hip, x, ids, top, T, lse + np.float32(0.5))
    out = np.ones((n, c), bool)
    np.put_along_axis(out, ids, False, 1)
    for g in (grad, back):
        assert np.isfinite(g).all() and (g[out] == 0).all()
    # the lowest float is a number: a rest that is finite, and far
    low = np.where(x == -np.inf, np.finfo(np.float32).min, x)
    masked, _ = check(hip, low, ids, top, T, lse)
    assert np.allclose(masked, tail64(x, ids, top, T, lse, 6.0)[0], rtol=1e-5, atol=1e-5)
    for mask in (-1e4, -1e9):
        check(hip, np.where(x == -np.inf, np.float32(mask), x), ids, top, T, lse)
    rows, rest = check(hip, low, ids, top, T, (lse + np.float32(0.5)))
    assert np.isfinite(rows).all() and (rest < -1e37).all()


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("c", [6, 40, 5001])
def test_gradient_against_differences_of_the_row_losses(hip, c, tail):
    """Central differences of the device's own row losses. A row's loss is off by at most `brow`, so a difference over
    2 h by brow/h; a log-sum-exp's third derivative is below 0.1, and the row holds two at most, each T^2 times one of
    z = x/T."""
    from test_gpu_distill import oracle

    k, T, h = 4, 1.5, 2.0 ** -4
    x, ids, top, teacher = student_and_teacher(1, c, k, c + 5)
    lse = teacher_lse(teacher, T) if tail else None
    D = hip.DeviceArray.from_numpy
    dl = D(lse) if tail else None
    g = hip.distill_fwd(D(x), D(ids), D(top), T, dl, 1.0, need_grad=True)[4].numpy()[0]
    bound = oracle(x, ids, top, T, lse, 1.0)["brow"][0] * 2  # the moved rows' are no larger than twice it
    for i in [int(v) for v in ids[0]] + [int(v) for v in np.argsort(-x[0])[:3]]:
        up, down = x.copy(), x.copy()
        up[0, i] += np.float32(h)
        down[0, i] -= np.float32(h)
        f = [float(hip.distill_fwd(D(v), D(ids), D(top), T, dl, 1.0)[1].numpy()[0]) for v in (up, down)]
        width = float(up[0, i]) - float(down[0, i])
        assert abs((f[0] - f[1]) / width - g[i]) <= 2 * bound / width + h * h / 6 * 0.2 / T + U * abs(g[i]) + 1e-7, (c, tail, i)
