"""Distillation from a teacher's top logits (oxi_distill_*) against float64.

Tolerances, u = 2^-24: an exponential of (x - m)/T is off, relatively, by a u for
each of the difference and the product, times the argument's size, and by at most
2 steps (4 u) of its own; a row's sum adds at most c/64 + 24 of them in sequence
in float32 on any path. `Errors` propagates these through the formulas, per row.
"""

import numpy as np
import pytest

from conftest import rng

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def oracle(x, ids, top, T, lse=None, divisor=None):
    """float64: loss, row losses, lse, log rest, gradient, and the bounds of the rows' losses and the gradient."""
    n, c = x.shape
    divisor = float(divisor or max(1, n))
    T = float(np.float32(T))
    z = x.astype(np.float64) / T
    rows, grads = np.zeros(n), np.zeros((n, c))
    brow, bgrad = np.zeros(n), np.zeros((n, c))
    lses, rests = np.zeros(n), np.zeros(n)
    for r in range(n):
        with np.errstate(all="ignore"):
            m = z[r].max()
            e = np.exp(z[r] - m)
            lq = z[r] - m - np.log(e.sum())
        q = np.exp(lq)
        lses[r] = m + np.log(e.sum())
        eps = U * (3 * np.minimum(np.abs(z[r] - m), 110.0) + 6)  # of each exponential; beyond 110 it is 0
        seq = (c / 64 + 24) * U
        dl = (q * eps).sum() + seq + 2 * U  # of the sum, and so of lse
        keep = [j for j in range(ids.shape[1]) if 0 <= ids[r, j] < c and top[r, j] != -np.inf]
        seen = sorted({int(ids[r, j]) for j in keep})
        rest = np.delete(e, seen).sum() / e.sum() if lse is not None else 1.0
        with np.errstate(divide="ignore"):
            rests[r] = np.log(rest) if lse is not None else 0.0
        if not keep:
            continue
        t = np.array([float(top[r, j]) for j in keep]) / T
        lp = t - (np.log(np.exp(t - t.max()).sum()) + t.max()) if lse is None else t - float(lse[r])
        p = np.exp(lp)
        at = [int(ids[r, j]) for j in keep]
        with np.errstate(invalid="ignore"):
            rows[r] = np.where(p > 0, p * (lp - lq[at]), 0.0).sum()
        given = np.zeros(c)
        np.add.at(given, at, p)
        factor = np.ones(c)
        bf = 0.0
        if lse is not None:
            pr = max(1.0 - p.sum(), 0.0)
            if pr > 0:
                rows[r] += pr * (np.log(pr) - rests[r])
            out = np.ones(c, bool)
            out[seen] = False
            if rest > 0:
                factor[out] = 1 - pr / rest
                dr = 2 * dl / max(1e-30, 1.0)  # both sums' relative errors
                bf = dr * pr / rest + 4 * U + 4 * 2.0 ** -52 * (1 + pr / rest)
            # masses balance, so lse enters times sum |q - p|, and squared
            gap = sum(abs(q[i] - given[i]) for i in seen) + abs(rest - pr)
            brow[r] = 2 * dl * gap + 8 * dl * dl + 4 * U * rows[r] + 1e-13
        else:
            brow[r] = dl + 2 * 2.0 ** -50 * np.abs(t).max() + 4 * U * abs(rows[r]) + 1e-13
        q_all = q * factor
        grads[r] = (q_all - given) * T / divisor
        bgrad[r] = T / divisor * (q * np.abs(factor) * (eps + dl + 6 * U) + q * bf + given * 4 * U + U * np.abs(q_all - given)
                                  ) + 1e-38
    rows *= T * T
    brow = brow * T * T + U * np.abs(rows)
    loss = rows.sum() / divisor
    return dict(loss=loss, rows=rows, lse=lses, rest=rests, grad=grads, brow=brow, bgrad=bgrad,
                bloss=brow.sum() / divisor + 2 * U * abs(loss))


def student_and_teacher(n, c, k, seed, near=1.0, spread=2.0):
    r = rng(seed)
    teacher = (spread * r.standard_normal((n, c))).astype(np.float32)
    x = (0.8 * teacher + near * r.standard_normal((n, c))).astype(np.float32)
    ids = np.argsort(-teacher, axis=1, kind="stable")[:, :k].astype(np.int64)
    return x, ids, np.take_along_axis(teacher, ids, 1), teacher


def teacher_lse(teacher, T):
    t = teacher.astype(np.float64) / float(np.float32(T))
    m = t.max(1, keepdims=True)
    return (m[:, 0] + np.log(np.exp(t - m).sum(1))).astype(np.float32)


def check(hip, x, ids, top, T, lse=None, divisor=None, what=""):
    D = hip.DeviceArray.from_numpy
    n, c = x.shape
    w = oracle(x, ids, top, T, lse, divisor)
    dx, di, dt, dl = D(x), D(ids), D(top), D(lse) if lse is not None else None
    loss, row, slse, rest, grad = hip.distill_fwd(dx, di, dt, T, dl, divisor, need_grad=True)
    loss2, row2, slse2, rest2, none = hip.distill_fwd(dx, di, dt, T, dl, divisor)
    assert none is None
    for a, b in ((loss, loss2), (row, row2), (slse, slse2), (rest, rest2)):
        assert np.array_equal(a.numpy(), b.numpy(), equal_nan=True), "the gradient changes the loss"

    def near(got, want, bound, name):
        got = got.astype(np.float64)
        same = (got == want) | (np.isnan(got) & np.isnan(want))
        with np.errstate(invalid="ignore"):
            bad = ~same & ~(np.abs(got - want) <= bound)
        assert not bad.any(), (f"{what} {name}: {bad.sum()} of {bad.size} outside; first {np.argwhere(bad)[0]}: "
                               f"{got[bad][0]!r} for {want[bad][0]!r}, bound {np.broadcast_to(bound, got.shape)[bad][0]!r}")

    near(row.numpy(), w["rows"], w["brow"], "row_loss")
    near(loss.numpy(), np.array([w["loss"]]), w["bloss"], "loss")
    near(slse.numpy(), w["lse"], 1e-6 * np.abs(w["lse"]) + (c / 64 + 40) * U, "lse")
    near(grad.numpy(), w["grad"], w["bgrad"], "gradient")
    g = np.array([-0.37], np.float32)
    back = hip.distill_bwd(dx, di, dt, slse, rest, D(g), T, dl, divisor).numpy()
    # exp(x/T - lse) in float32: the quotient's and lse's own rounding, relative to their size; a rest of a few
    # steps is known to its logarithm's
    size = 3 * np.abs(w["lse"][:, None]) + 3 * np.abs(x / np.float32(T)) + 12
    T32 = float(np.float32(T))
    dv = float(divisor or max(1, n))
    some = np.abs(w["grad"]).sum(1, keepdims=True) > 0
    z = x.astype(np.float64) / T32
    q = np.exp(z - w["lse"][:, None])
    ratio = 0.0
    if lse is not None:
        ratio = 1.0 + np.abs(np.where(q > 0, w["grad"] * dv / T32 / np.maximum(q, 1e-300), 0.0))
        ratio = ratio * (4 + np.abs(w["rest"][:, None]))
    extra = np.where(some, T32 / dv * q * U * (size + ratio * 4), 0.0)
    near(back, w["grad"] * float(g[0]), (w["bgrad"] + extra) * abs(float(g[0])) + 1e-38, "gradient for an upstream")
    return w


@pytest.mark.parametrize("n,c,k", [
    (1, 1, 1), (2, 2, 1), (3, 3, 3), (5, 7, 2), (4, 31, 8), (6, 64, 5), (3, 255, 200), (9, 256, 8), (2, 1000, 64), (5, 1003, 50),
    (3, 4096, 100), (2, 4097, 256), (3, 16385, 8), (2, 32000, 64), (3, 32001, 7), (2, 50257, 50), (2, 65536, 16), (2, 65537, 3),
    (1, 70001, 1024), (2, 131072, 64), (1, 200003, 33), (1, 300001, 5), (1, 310003, 1024), (300, 515, 4), (1100, 96, 6), (40, 9, 8), (7, 600, 300),
    (3, 2050, 1000), (4, 1500, 150), (3, 3100, 40), (3, 3100, 60), (5, 1020, 223), (5, 1020, 224),
    (2, 5003, 9), (3, 7001, 40), (2, 12001, 8), (2, 13002, 20), (2, 18003, 6), (2, 22001, 5), (3, 26002, 7)])
@pytest.mark.parametrize("T,tail", [(1.0, False), (2.0, True), (0.7, True), (4.0, False)])
def test_loss_and_gradient(hip, n, c, k, T, tail):
    print("[case] distill", n, c, k, T, tail, flush=True)
    x, ids, top, teacher = student_and_teacher(n, c, k, n + c + k)
    check(hip, x, ids, top, T, teacher_lse(teacher, T) if tail else None)


def test_a_student_near_its_teacher(hip):
    """A small loss of large terms keeps its relative accuracy (1e-5) when the rest counts."""
    for c in (300, 5001, 32000):
        x, ids, top, teacher = student_and_teacher(4, c, 1, c, near=0.05)
        x = (teacher + 0.05 * rng(1).standard_normal(teacher.shape)).astype(np.float32)
        w = oracle(x, ids, top, 1.0, teacher_lse(teacher, 1.0))
        D = hip.DeviceArray.from_numpy
        row = hip.distill_fwd(D(x), D(ids), D(top), 1.0, D(teacher_lse(teacher, 1.0)))[1].numpy()
        assert (w["rows"] < 0.01).all()
        assert (np.abs(row - w["rows"]) <= w["brow"]).all()
        check(hip, x, ids, top, 1.0, teacher_lse(teacher, 1.0))


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("c", [40, 515, 4096, 70000])
def test_padding_duplicates_and_empty_rows(hip, c, tail):
    n, k = 9, 12
    x, ids, top, teacher = student_and_teacher(n, c, k, c)
    ids[1, 5:] = -1
    ids[2, ::2] = -7
    ids[3] = -1  # nothing
    top[4, 3] = -np.inf
    top[5] = -np.inf  # nothing
    ids[6, 7] = ids[6, 2]
    ids[6, 11] = ids[6, 2]
    top[6, 11] = top[6, 2]
    ids[7, 0] = -1  # the first entry is padding
    lse = teacher_lse(teacher, 1.5) + (np.float32(0.5) if tail else 0)
    w = check(hip, x, ids, top, 1.5, lse if tail else None, divisor=7.0)
    assert w["rows"][3] == 0 and w["rows"][5] == 0 and (w["grad"][3] == 0).all() and (w["grad"][5] == 0).all()
    D = hip.DeviceArray.from_numpy
    grad = hip.distill_fwd(D(x), D(ids), D(top), 1.5, D(lse) if tail else None, 7.0, need_grad=True)[4].numpy()
    assert (grad[3] == 0).all() and (grad[5] == 0).all()


def test_every_class_listed(hip):
    """k == c with the teacher's lse: nothing is left over on either side."""
    x, ids, top, teacher = student_and_teacher(6, 24, 24, 3)
    T = 1.0
    lse = teacher_lse(teacher, T) - np.float32(1e-3)  # the p sum to a little over 1: pr is 0
    check(hip, x, ids, top, T, lse)


def test_special_logits(hip):
    """-inf at a class that is not listed costs nothing; at a listed one the loss is inf; NaN stays in its row."""
    D = hip.DeviceArray.from_numpy
    for c in (520, 1003, 70000):
        x, ids, top, teacher = student_and_teacher(5, c, 4, c)
        out = [i for i in range(c) if i not in ids[1]][:3]
        x[1, out] = -np.inf
        x[2, ids[2, 1]] = -np.inf
        x[3, 17] = np.nan
        want = oracle(x[[0, 1, 4]], ids[[0, 1, 4]], top[[0, 1, 4]], 1.0, divisor=5.0)
        loss, row, _, _, grad = (a.numpy() for a in hip.distill_fwd(D(x), D(ids), D(top), 1.0, None, 5.0, need_grad=True))
        assert np.isinf(row[2]) and row[2] > 0 and np.isnan(row[3]) and np.isnan(grad[3]).all() and np.isnan(loss[0])
        assert (np.abs(row[[0, 1, 4]] - want["rows"]) <= want["brow"]).all()
        assert (np.abs(grad[[0, 1, 4]] - want["grad"]) <= want["bgrad"]).all()
        assert (grad[1, out] == 0).all() and np.isfinite(grad[2]).all()


def test_wide_logits(hip):
    """Logits of +-1e4 and a teacher as wide: exponentials underflow to 0, sums stay finite."""
    r = rng(5)
    for c in (64, 5001):
        teacher = (1e4 * r.standard_normal((4, c))).astype(np.float32)
        x = (1e4 * r.standard_normal((4, c))).astype(np.float32)
        ids = np.argsort(-teacher, 1)[:, :6].astype(np.int64)
        check(hip, x, ids, np.take_along_axis(teacher, ids, 1), 1.0)


def test_gradient_against_differences(hip):
    """Central differences of the device's own row losses (float64 of the oracle agrees with both)."""
    n, c, k, T = 3, 40, 5, 1.5
    x, ids, top, teacher = student_and_teacher(n, c, k, 8)
    lse = teacher_lse(teacher, T)
    D = hip.DeviceArray.from_numpy
    for tail in (None, lse):
        g = hip.distill_fwd(D(x), D(ids), D(top), T, D(tail) if tail is not None else None, 1.0, need_grad=True)[4].numpy()
        step = 2.0 ** -6
        for i in list(ids[0]) + [0, 1, 20, 39]:
            up, down = x.copy(), x.copy()
            up[0, i] += np.float32(step)
            down[0, i] -= np.float32(step)
            d = oracle(up, ids, top, T, tail, 1.0)["loss"] - oracle(down, ids, top, T, tail, 1.0)["loss"]
            width = float(up[0, i]) - float(down[0, i])
            # the third derivative of a log-sum-exp is at most 1 (over T here)
            assert abs(d / width - g[0, i]) <= step * step / 6 * 2 + 1e-5


def test_id_outside_the_classes_is_reported(hip):
    x, ids, top, _ = student_and_teacher(3, 50, 4, 1)
    bad = ids.copy()
    bad[1, 2] = 50
    D = hip.DeviceArray.from_numpy
    _, row, _, _, grad = hip.distill_fwd(D(x), D(bad), D(top), 1.0, need_grad=True)
    with pytest.raises(RuntimeError):
        hip.sync()
    skip = ids.copy()
    skip[1, 2] = -1
    w = oracle(x, skip, top, 1.0)
    assert (np.abs(row.numpy() - w["rows"]) <= w["brow"]).all()
    assert (np.abs(grad.numpy() - w["grad"]) <= w["bgrad"]).all()
    hip.sync()  # reported once


def test_no_rows(hip):
    loss = hip.DeviceArray.from_numpy(np.ones(1, np.float32))
    hip.call("oxi_distill_fwd", None, None, None, None, loss.ptr, None, None, None, None, 0, 50, 4, 1.0, 1.0)
    assert loss.numpy()[0] == 0


@pytest.mark.parametrize("shift,to", [(1, 1), (2, 2), (3, 3), (0, 1), (2, 0), (1, 3)])
@pytest.mark.parametrize("c", [6, 64, 515, 4096, 70000])
def test_buffers_at_any_float(hip, shift, to, c):
    """Logits and gradient `shift` and `to` floats past a 16-byte address."""
    n, k = 3, 5
    x, ids, top, _ = student_and_teacher(n, c, k, c)
    D = hip.DeviceArray.from_numpy
    src = D(np.concatenate([np.zeros(shift, np.float32), x.ravel()]))
    dst, dst2 = (D(np.full(n * c + 8, 7, np.float32)) for _ in range(2))
    di, dt, one = D(ids), D(top), D(np.ones(1, np.float32))
    loss, row, lse, rest = (hip.DeviceArray((m,)) for m in (1, n, n, n))
    hip.call("oxi_distill_fwd", src.ptr + 4 * shift, di.ptr, dt.ptr, None, loss.ptr, row.ptr, lse.ptr, rest.ptr,
             dst.ptr + 4 * to, n, c, k, 1.0, float(n))
    hip.call("oxi_distill_bwd", src.ptr + 4 * shift, di.ptr, dt.ptr, None, lse.ptr, rest.ptr, one.ptr, dst2.ptr + 4 * to, n,
             c, k, 1.0, float(n))
    w = oracle(x, ids, top, 1.0)
    assert (np.abs(row.numpy() - w["rows"]) <= w["brow"]).all()
    q = np.exp(x - w["lse"][:, None])
    # the backward's exponent: the logit's and lse's own float32 steps
    more = q / n * U * (3 * np.abs(w["lse"][:, None]) + 3 * np.abs(x) + 16)
    for buf, extra in ((dst, 0.0), (dst2, more)):
        got = buf.numpy()
        assert (got[:to] == 7).all() and (got[to + n * c:] == 7).all()
        assert (np.abs(got[to:to + n * c].reshape(n, c) - w["grad"]) <= w["bgrad"] + extra).all()


@pytest.mark.parametrize("c", [300, 5001, 70001])
def test_gradient_where_nearly_everything_is_left_over(hip, c):
    """A few entries of small mass: q (1 - pr/qr) at the other classes is a small part of q, known to the accuracy of
    the masses listed (psum and ql), not of 1 less them."""
    T = 4.0
    x, ids, top, teacher = student_and_teacher(4, c, 3, c)
    lse = teacher_lse(teacher, T)
    D = hip.DeviceArray.from_numpy
    _, _, slse, rest, d = hip.distill_fwd(D(x), D(ids), D(top), T, D(lse), need_grad=True)
    back = hip.distill_bwd(D(x), D(ids), D(top), slse, rest, D(np.ones(1, np.float32)), T, D(lse)).numpy()
    d = d.numpy()
    z = x.astype(np.float64) / T
    for r in range(4):
        lq = z[r] - z[r].max() - np.log(np.exp(z[r] - z[r].max()).sum())
        q = np.exp(lq)
        eps = U * (3 * np.abs(z[r] - z[r].max()) + 6)
        dl = (q * eps).sum() + (c / 64 + 26) * U
        p = np.exp(top[r].astype(np.float64) / T - float(lse[r]))
        psum, ql = p.sum(), q[ids[r]].sum()
        assert psum < 0.25
        out = np.ones(c, bool)
        out[ids[r]] = False
        want = T / 4 * q * (psum - ql) / (1 - ql)
        # the masses' errors, then the product's; the backward has lse and the logits at float32's steps too
        for got, more in ((d[r], 0.0), (back[r], U * (3 * np.abs(z[r]).max() + 3 * abs(float(slse.numpy()[r]))))):
            bound = T / 4 * q * ((dl + more + 8 * U) * (psum + ql) / (1 - ql) + np.abs(psum - ql) * (eps + dl + more + 8 * U))
            assert (np.abs(got - want)[out] <= bound[out]).all()
