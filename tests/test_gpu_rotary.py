"""Rotary positions (oxi_rotary) against float64.

Tolerance, u = 2^-24: a cosine or sine is off by at most 3 steps of float32 below
1 (6 u; an angle of 64 bits adds nothing at these positions), its product with
the scale, the two products and their sum by a u each: 9 u (|u| + |v|) scale.
"""

import numpy as np
import pytest

from conftest import rng

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def frequencies(rot, base=10000.0):
    half = rot // 2
    return base ** (-np.arange(half, dtype=np.float64) / max(1, half))


def turn64(x, pos, freq, layout, inverse=False, scale=1.0):
    """x (B, T, H, D) and each value's size for its error."""
    rot = 2 * len(freq)
    a = (pos.astype(np.float64)[..., None] * freq)[:, :, None, :]
    c, s = np.cos(a) * scale, np.sin(a) * scale * (-1 if inverse else 1)
    y, size = x.astype(np.float64).copy(), np.zeros(x.shape)
    i0, i1 = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    u, v = x[..., i0].astype(np.float64), x[..., i1].astype(np.float64)
    y[..., i0], y[..., i1] = u * c - v * s, v * c + u * s
    size[..., i0] = size[..., i1] = (np.abs(u) + np.abs(v)) * abs(scale)
    return y, size


def check(got, x, pos, freq, layout, inverse=False, scale=1.0):
    y, size = turn64(x, pos, freq, layout, inverse, scale)
    err = np.abs(got.astype(np.float64) - y)
    assert (err <= 9 * U * size).all(), f"worst {np.max(err / np.maximum(size, 1e-30)) / U:.3g} u"


CASES = [  # batch, tokens, heads, dim, rot
    (1, 1, 1, 2, 2), (1, 1, 1, 1, 0), (2, 3, 1, 6, 2), (1, 5, 3, 8, 8), (2, 7, 5, 20, 10), (3, 1, 40, 128, 128), (64, 1, 8, 64, 64),
    (2, 33, 12, 64, 32), (1, 300, 4, 128, 128), (2, 17, 3, 80, 20), (1, 9, 2, 96, 48), (1, 4, 2, 256, 64), (1, 3, 1, 258, 258),
    (2, 5, 7, 130, 66), (1, 2, 65, 36, 36), (1, 2, 3, 12, 6), (5, 11, 2, 40, 40)]


@pytest.mark.parametrize("B,T,H,D,rot", CASES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_forward_and_inverse(hip, B, T, H, D, rot, layout):
    print("[case] rotary", B, T, H, D, rot, layout, flush=True)
    r = rng(B * T + D)
    x = r.standard_normal((B, T, H, D)).astype(np.float32)
    pos = r.integers(0, 200000, (B, T)).astype(np.int64)
    f = frequencies(rot)
    dev = hip.DeviceArray.from_numpy
    dx, dp, df = dev(x), dev(pos), dev(f) if rot else hip.DeviceArray((0,), np.float64)
    for inverse, scale in ((False, 1.0), (True, 1.0), (False, 1.25), (True, 0.75)):
        y = hip.rotary(dx, df, dp, layout=layout, inverse=inverse, scale=scale).numpy()
        check(y, x, pos, f, layout, inverse, scale)
        assert np.array_equal(y[..., rot:], x[..., rot:])


def test_positions(hip):
    """Shared positions, an offset, none given, negative ones, far ones, one per sequence."""
    r = rng(2)
    x = r.standard_normal((3, 9, 2, 64)).astype(np.float32)
    f = frequencies(64)
    dev = hip.DeviceArray.from_numpy
    dx, df = dev(x), dev(f)
    steps = np.broadcast_to(np.arange(9), (3, 9))
    check(hip.rotary(dx, df).numpy(), x, steps, f, "half")
    check(hip.rotary(dx, df, offset=12345).numpy(), x, steps + 12345, f, "half")
    shared = r.integers(-5000, 5000, 9).astype(np.int64)
    check(hip.rotary(dx, df, dev(shared), offset=7).numpy(), x, np.broadcast_to(shared + 7, (3, 9)), f, "half")
    each = r.integers(0, 1 << 20, 3).astype(np.int64)
    check(hip.rotary(dx, df, dev(each), pos_strides=(1, 0)).numpy(), x, np.broadcast_to(each[:, None], (3, 9)), f, "half")
    far = (1 << 20) + steps.astype(np.int64) * 99991
    check(hip.rotary(dx, df, dev(np.ascontiguousarray(far))).numpy(), x, far, f, "half")


def test_angles_that_pass_32_bits(hip):
    """Positions past 2^31: the angle's own rounding in 64 bits (2^-53 of it) joins the tolerance."""
    r = rng(4)
    x = r.standard_normal((1, 6, 2, 8)).astype(np.float32)
    f = frequencies(8)
    pos = (np.arange(6, dtype=np.int64) * 7 + (1 << 33))[None]
    dev = hip.DeviceArray.from_numpy
    y = hip.rotary(dev(x), dev(f), dev(pos)).numpy()
    want, size = turn64(x, pos, f, "half")
    angle = 2 * float(pos.max()) * 2.0 ** -53
    assert (np.abs(y - want) <= (9 * U + angle) * size).all()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_strided(hip, layout):
    """Heads before tokens, query and key heads inside a wider buffer, a strided element, and in place."""
    B, H, T, D = 2, 6, 13, 64
    r = rng(6)
    f = frequencies(32)
    pos = r.integers(0, 9000, (B, T)).astype(np.int64)
    dev = hip.DeviceArray.from_numpy
    df, dp = dev(f), dev(pos)
    x = r.standard_normal((B, H, T, D)).astype(np.float32)  # as (B, T, H, D): strides below
    st = (H * T * D, D, T * D, 1)
    xt = x.transpose(0, 2, 1, 3)
    y = hip.rotary(dev(x), df, dp, layout=layout, x_strides=st, shape=(B, T, H, D)).numpy()
    check(y, xt, pos, f, layout)
    y = hip.rotary(dev(x), df, dp, layout=layout, x_strides=st, out_strides=st, shape=(B, T, H, D)).numpy()
    check(y.reshape(B, H, T, D).transpose(0, 2, 1, 3), xt, pos, f, layout)
    # 8 heads of a buffer of 11, in place: the other heads stay
    w = r.standard_normal((B, T, 11, D)).astype(np.float32)
    b = dev(w)
    hip.rotary(b, df, dp, layout=layout, out=b, x_strides=(T * 11 * D, 11 * D, D, 1), out_strides=(T * 11 * D, 11 * D, D, 1),
               shape=(B, T, 8, D))
    got = b.numpy()
    assert np.array_equal(got[:, :, 8:], w[:, :, 8:])
    check(got[:, :, :8], w[:, :, :8], pos, f, layout)
    # every second float of a wider element dim
    z = r.standard_normal((B, T, H, 2 * D)).astype(np.float32)
    y = hip.rotary(dev(z), df, dp, layout=layout, x_strides=(T * H * 2 * D, H * 2 * D, 2 * D, 2), shape=(B, T, H, D)).numpy()
    check(y, z[..., ::2], pos, f, layout)
    # one sequence broadcast over the batch
    y = hip.rotary(dev(w[:1]), df, dp, layout=layout, x_strides=(0, 11 * D, D, 1), shape=(B, T, 11, D)).numpy()
    check(y, np.broadcast_to(w[:1], w.shape), pos, f, layout)


@pytest.mark.parametrize("shift", [1, 2, 3])
def test_buffers_at_any_float(hip, shift):
    B, T, H, D = 1, 5, 3, 64
    r = rng(shift)
    x = r.standard_normal((B, T, H, D)).astype(np.float32)
    f, pos = frequencies(64), np.arange(5, dtype=np.int64)[None] * 1000
    dev = hip.DeviceArray.from_numpy
    n = x.size
    src = dev(np.concatenate([np.zeros(shift, np.float32), x.ravel()]))
    dst = dev(np.full(n + 8, 7, np.float32))
    df, dp = dev(f), dev(pos)
    st = hip._i64arr(hip.row_major_strides(x.shape))
    hip.call("oxi_rotary", src.ptr + 4 * shift, st, dst.ptr + 4 * shift, st, hip._i64arr(x.shape), dp.ptr,
             hip._i64arr((5, 1)), 0, df.ptr, 64, 0, 0, 1.0)
    got = dst.numpy()
    assert (got[:shift] == 7).all() and (got[shift + n:] == 7).all()
    check(got[shift:shift + n].reshape(x.shape), x, pos, f, "half")


def test_vjp_is_the_transpose(hip):
    """<g, R x> = <R' g, x> and R' (R x) = scale^2 x."""
    r = rng(9)
    x, g = (r.standard_normal((2, 31, 4, 48)).astype(np.float32) for _ in range(2))
    f = frequencies(36)
    dev = hip.DeviceArray.from_numpy
    df = dev(f)
    for layout in ("half", "interleaved"):
        y = hip.rotary(dev(x), df, layout=layout, scale=1.5)
        back = hip.rotary(dev(g), df, layout=layout, scale=1.5, inverse=True).numpy().astype(np.float64)
        a, b = (g.astype(np.float64) * y.numpy()).sum(), (back * x).sum()
        assert abs(a - b) <= 20 * U * 1.5 * (np.abs(g).sum() * np.abs(x).max())
        twice = hip.rotary(y, df, layout=layout, scale=1.5, inverse=True).numpy()
        assert np.allclose(twice[..., :36], 2.25 * x[..., :36], rtol=0, atol=40 * U * 2.25 * np.abs(x).max())


def test_empty(hip):
    df = hip.DeviceArray.from_numpy(frequencies(8))
    for shape in ((0, 3, 2, 8), (2, 0, 2, 8), (2, 3, 0, 8)):
        assert hip.rotary(hip.DeviceArray(shape), df).numpy().shape == shape
