"""The joint gradient norm and clipping (oxi_grad_norm, oxi_grad_clip) against float64.

The norm is summed in 64 bits: each of n terms adds at most 2^-53 of the sum, each
squaring none (24-bit factors), the root 2^-53: n 2^-53 bounds it. A clipped element
takes two roundings, of the factor and of the product: 2 * 2^-24 relatively.
"""

import numpy as np
import pytest

from conftest import rng

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def grads_of(sizes, seed):
    r = rng(seed)
    return [(10.0 ** r.uniform(-4, 2) * r.standard_normal(s)).astype(np.float32) for s in sizes]


def norm_of(grads, p=2.0):
    v = np.concatenate([np.abs(g.astype(np.float64)).ravel() for g in grads] + [np.zeros(0)])
    if p == np.inf:
        return v.max() if v.size else -np.inf
    return float(np.sqrt(np.sum(v.astype(np.longdouble) ** 2))) if p == 2 else float(np.sum(v.astype(np.longdouble)))


def check(hip, grads, most, p=2.0, in_place=False):
    D = [hip.DeviceArray.from_numpy(g) for g in grads]
    n = sum(g.size for g in grads)
    want = norm_of(grads, p)
    total = hip.grad_norm(D, p)
    got = float(total.numpy()[0])
    assert got == want or abs(got - want) <= (n + 4) * 2.0 ** -53 * abs(want), (got, want)
    outs = hip.grad_clip(D, total, most, D if in_place else None)
    factor = most / (want + 1e-6)
    for g, o in zip(grads, outs):
        o = o.numpy()
        if not factor < 1:
            assert np.array_equal(o, g, equal_nan=True)
        else:
            w = g.astype(np.float64) * factor
            assert (np.abs(o - w) <= 2.01 * U * np.abs(w) + 2.0 ** -149).all()


@pytest.mark.parametrize("p", [1.0, 2.0, float("inf")])
@pytest.mark.parametrize("sizes", [[1], [5], [4096], [4097], [16385, 3], [100003], [1, 2, 3, 4, 5, 6, 7, 8, 9],
                                   [64] * 200, [1000003, 17, 262144, 1]], ids=lambda s: f"{len(s)}x{s[0]}")
def test_sizes(hip, sizes, p):
    grads = grads_of(sizes, len(sizes) + sizes[0])
    for most in (0.5, 1e9):
        check(hip, grads, most, p)
        check(hip, grads, most, p, in_place=True)


def test_empty_ones_and_none(hip):
    check(hip, grads_of([0, 7, 0, 9, 0], 3), 0.1)
    total = hip.grad_norm([], 2.0)
    assert total.numpy()[0] == 0.0
    assert hip.grad_norm([hip.DeviceArray((0,))], 1.0).numpy()[0] == 0.0
    hip.grad_clip([], total, 1.0)
    hip.sync()


def test_squares_that_32_bits_cannot_hold(hip):
    check(hip, [np.array([3e30, -4e30], np.float32)], 1.0)
    check(hip, [np.full(5000, 1e-30, np.float32)], 1e-32)


def test_a_long_sum_keeps_its_digits(hip):
    """2^24 ones after a large term: a 32-bit sum would not move."""
    g = np.ones(1 << 24, np.float32)
    g[0] = 4096.0
    check(hip, [g], 1.0)
    check(hip, [g], 1.0, 1.0)


def test_infinities_and_nan(hip):
    D = hip.DeviceArray.from_numpy
    g = np.array([1.0, -np.inf, 2.0], np.float32)
    t = hip.grad_norm([D(g)])
    assert t.numpy()[0] == np.inf
    o = hip.grad_clip([D(g)], t, 1.0)[0].numpy()  # the factor is 0
    assert o[0] == 0 and np.isnan(o[1]) and o[2] == 0
    g = np.array([1.0, np.nan, 2.0], np.float32)
    for p in (1.0, 2.0):
        t = hip.grad_norm([D(g), D(np.ones(3, np.float32))], p)
        assert np.isnan(t.numpy()[0])
        assert np.array_equal(hip.grad_clip([D(g)], t, 1.0)[0].numpy(), g, equal_nan=True)  # as they were
    assert hip.grad_norm([D(g)], float("inf")).numpy()[0] == 2.0
    assert hip.grad_norm([D(np.full(3, np.nan, np.float32))], float("inf")).numpy()[0] == -np.inf


def test_views_at_any_float(hip):
    """Slices back to back in one buffer, none at a float4's address; what lies between stays."""
    r = rng(9)
    buf = r.standard_normal(60000).astype(np.float32)
    spans = [(1, 5), (7, 4099), (4107, 1), (4110, 33333), (37450, 20001)]
    b = hip.DeviceArray.from_numpy(buf)
    o = hip.DeviceArray.from_numpy(np.full(60000, 7.0, np.float32))
    for shift in (0, 1, 3):
        rows = [(b.ptr + 4 * a, o.ptr + 4 * (a + shift), n) for a, n in spans]
        s = hip.slice_array(hip.GradSlice, rows)
        total = hip.DeviceArray((1,), np.float64)
        hip.call("oxi_grad_norm", s, len(spans), 2.0, total.ptr, None)
        want = norm_of([buf[a:a + n] for a, n in spans])
        assert abs(total.numpy()[0] - want) <= 60004 * 2.0 ** -53 * want
        hip.call("oxi_fill", o.ptr, 60000, 7.0)
        hip.call("oxi_grad_clip", s, len(spans), total.ptr, 1.0)
        got = o.numpy()
        for a, n in spans:
            w = buf[a:a + n].astype(np.float64) * (1.0 / (want + 1e-6))
            assert (np.abs(got[a + shift:a + shift + n] - w) <= 2.01 * U * np.abs(w)).all()
            got[a + shift:a + shift + n] = 7.0
        assert (got == 7.0).all()


def test_workspace_of_the_caller_and_the_same_bits(hip):
    D = [hip.DeviceArray.from_numpy(g) for g in grads_of([50001, 333, 70000], 11)]
    ws = hip.DeviceArray((max(1, hip.grad_norm_workspace(D)),), np.uint8)
    a = hip.grad_norm(D).numpy()
    for _ in range(3):
        assert np.array_equal(hip.grad_norm(D, workspace=ws).numpy(), a)
