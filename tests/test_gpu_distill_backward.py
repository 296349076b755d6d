"""The distillation backward against the gradient that the forward's own pass
writes, at logits far from zero too: no probability goes by a log-sum-exp that is
rounded to a float. Rows whose sums the backward forms again have the forward's
bits, scaled exactly by an upstream gradient that is a power of two (no element
here comes near the smallest floats)."""

import numpy as np
import pytest

from conftest import rng
from test_gpu_distill import U, check, oracle, student_and_teacher, teacher_lse

pytestmark = pytest.mark.gpu

SHAPES = [(3, 5, 2), (4, 40, 6), (9, 512, 8), (5, 1003, 300), (6, 2047, 20), (4, 5001, 64), (3, 9000, 9), (3, 14001, 30),
          (2, 20001, 5), (3, 32000, 64), (2, 50257, 50), (2, 65536, 8), (2, 70001, 16), (1, 300005, 9)]


@pytest.mark.parametrize("n,c,k", SHAPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("shift", [0.0, 2.0 ** 13])
def test_an_upstream_scales_the_forwards_gradient(hip, n, c, k, tail, shift):
    """Logits as they are and all of a row moved by the same number, which changes no probability."""
    print("[case] distill backward", n, c, k, tail, shift, flush=True)
    T = 2.0
    x, ids, top, teacher = student_and_teacher(n, c, k, n + c)
    x = np.float32(x + np.float32(shift))
    if n > 2:
        ids[1, k // 2:] = -1
        ids[2] = -1
    D = hip.DeviceArray.from_numpy
    a = (D(x), D(ids), D(top))
    lse = D(teacher_lse(teacher, T)) if tail else None
    _, _, slse, rest, grad = hip.distill_fwd(*a, T, lse, need_grad=True)
    grad = grad.numpy()
    assert np.abs(grad).max() > 0
    bound = 0.0
    if 65536 < c <= 300000:
        # each within its bound of the same value; the backward's log-sum-exp is off by at most 2^-21 besides
        w = oracle(x, ids, top, T, teacher_lse(teacher, T) if tail else None)
        z = x.astype(np.float64) / T
        bound = 2 * w["bgrad"] + 16 * U * np.exp(z - w["lse"][:, None]) * T / n
    for up in (1.0, -0.5, 8.0):
        back = hip.distill_bwd(*a, slse, rest, D(np.array([up], np.float32)), T, lse).numpy().astype(np.float64)
        assert (np.abs(back - grad * np.float32(up)) <= bound * abs(up)).all(), (up, np.abs(back - grad * np.float32(up)).max())


@pytest.mark.parametrize("c", [40, 5001, 70001])
def test_far_from_zero(hip, c):
    """The forward's gradient itself, of logits near 8192: within the bounds that go by the distance from the maximum."""
    x, ids, top, teacher = student_and_teacher(4, c, 6, c)
    x = np.float32(x + np.float32(8192))
    check(hip, x, ids, top, 1.0)
    check(hip, x, ids, top, 2.0, teacher_lse(teacher, 2.0))


def test_no_rows_and_no_gradient_of_the_upstream(hip):
    """An upstream of 0 gives zeros, also where rows hold no entry."""
    x, ids, top, _ = student_and_teacher(3, 700, 4, 1)
    ids[1] = -1
    D = hip.DeviceArray.from_numpy
    _, _, slse, rest, _ = hip.distill_fwd(D(x), D(ids), D(top))
    assert (hip.distill_bwd(D(x), D(ids), D(top), slse, rest, D(np.zeros(1, np.float32))).numpy() == 0).all()
    hip.call("oxi_distill_bwd", None, None, None, None, None, None, None, None, 0, 50, 4, 1.0, 1.0)


def test_graph_node_of_a_scaled_loss(hip):
    import oxitorch_amd as ox
    from oxitorch_amd.nn import functional as F

    x, ids, top, _ = student_and_teacher(5, 300, 7, 3)
    x = np.float32(x + np.float32(8192))
    got = []
    for scale in (None, 0.5):
        t = ox.from_numpy(x, True)
        loss = F.distillation_loss(t, ids, top, 1.5)
        (loss if scale is None else loss * scale).backward()
        got.append(t.grad.numpy())
    assert np.array_equal(got[1], got[0] * np.float32(0.5)) and np.abs(got[0]).max() > 0
