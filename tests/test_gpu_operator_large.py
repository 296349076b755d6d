"""Offsets past 2^31 elements and 2^32 bytes: the last rows of buffers that
large give the bits that the same rows give in small ones."""

import numpy as np
import pytest

from conftest import rng

pytestmark = pytest.mark.gpu


def put(hip, ptr, a):
    a = np.ascontiguousarray(a)
    hip.check(hip.lib.oxi_hip_memcpy_h2d(ptr, a.ctypes.data, a.nbytes))


def take(hip, ptr, shape, dtype=np.float32):
    a = np.empty(shape, dtype)
    hip.check(hip.lib.oxi_hip_memcpy_d2h(a.ctypes.data, ptr, a.nbytes))
    return a


def test_add_rms_norm(hip):
    cols, rows = 8192, (1 << 18) + 300  # 2.15e9 elements, 8.6 GB each; dx over gh, h over r
    print("[case] large add_rms_norm", rows, cols, flush=True)
    n = rows * cols
    assert n > 1 << 31
    r = rng(1)
    A, D = hip.DeviceArray, hip.DeviceArray.from_numpy
    small = [r.standard_normal((4, cols)).astype(np.float32) for _ in range(4)]
    w = D((1 + 0.1 * r.standard_normal(cols)).astype(np.float32))
    x, res, y, rstd, q, scale = A((n,)), A((n,)), A((n,)), A((rows,)), A((n,), np.uint8), A((rows, 64))
    for b in (x, res):
        hip.call("oxi_fill", b.ptr, n, 0.5)
    at = (n - 4 * cols) * 4
    put(hip, x.ptr + at, small[0])
    put(hip, res.ptr + at, small[1])
    hip.call("oxi_add_rms_norm_e4m3_fwd", x.ptr, res.ptr, w.ptr, y.ptr, q.ptr, scale.ptr, rows, cols, 128, 1e-6)
    h8, q8, s8 = (a.numpy() for a in hip.add_rms_norm_e4m3_fwd(D(small[0]), D(small[1]), w, 128))
    assert np.array_equal(take(hip, y.ptr + at, (4, cols)), h8)
    assert np.array_equal(take(hip, q.ptr + n - 4 * cols, (4, cols), np.uint8), q8)
    assert np.array_equal(take(hip, scale.ptr + (rows - 4) * 256, (4, 64)), s8)
    hip.call("oxi_add_rms_norm_fwd", x.ptr, res.ptr, w.ptr, res.ptr, y.ptr, rstd.ptr, rows, cols, 1e-6)
    h, yy, rs = hip.add_rms_norm_fwd(D(small[0]), D(small[1]), w)
    assert np.array_equal(take(hip, res.ptr + at, (4, cols)), h.numpy())
    assert np.array_equal(take(hip, y.ptr + at, (4, cols)), yy.numpy())
    # the VJP: gy in x, gh in y, which dx replaces
    for b in (x, y):
        hip.call("oxi_fill", b.ptr, n, 0.25)
    put(hip, x.ptr + at, small[2])
    put(hip, y.ptr + at, small[3])
    dw = A((cols,))
    hip.call("oxi_add_rms_norm_bwd", res.ptr, w.ptr, rstd.ptr, x.ptr, y.ptr, y.ptr, dw.ptr, None, rows, cols, 1)
    dx, _ = hip.add_rms_norm_bwd(h, w, rs, D(small[2]), D(small[3]), mode="exact")
    assert np.array_equal(take(hip, y.ptr + at, (4, cols)), dx.numpy())
    assert np.isfinite(dw.numpy()).all()


def test_rotary(hip):
    B, T, H, D_ = 3, 90000, 64, 128  # 2.2e9 elements
    print("[case] large rotary", B, T, H, D_, flush=True)
    n = B * T * H * D_
    assert n > 1 << 31
    r = rng(2)
    A, D = hip.DeviceArray, hip.DeviceArray.from_numpy
    x = A((n,))
    hip.call("oxi_fill", x.ptr, n, 1.0)
    tail = r.standard_normal((1, 3, H, D_)).astype(np.float32)
    at = (n - 3 * H * D_) * 4
    put(hip, x.ptr + at, tail)
    freq = D(10000.0 ** (-np.arange(64, dtype=np.float64) / 64))
    hip.rotary(x, freq, out=x, shape=(B, T, H, D_), offset=5)  # in place
    want = hip.rotary(D(tail), freq, offset=5 + T - 3).numpy()
    assert np.array_equal(take(hip, x.ptr + at, tail.shape), want)
    assert np.array_equal(take(hip, x.ptr, (1, 1, H, D_)),
                          hip.rotary(D(np.ones((1, 1, H, D_), np.float32)), freq, offset=5).numpy())


@pytest.mark.parametrize("n,c", [(33000, 65536), (11000, 200001)])
def test_distill(hip, n, c):
    print("[case] large distill", n, c, flush=True)
    assert n * c > 1 << 31
    r = rng(3)
    A, D = hip.DeviceArray, hip.DeviceArray.from_numpy
    x, d = A((n * c,)), A((n * c,))
    hip.call("oxi_fill", x.ptr, n * c, 0.0)
    tail = (2 * r.standard_normal((3, c))).astype(np.float32)
    put(hip, x.ptr + (n - 3) * c * 4, tail)
    ids = np.zeros((n, 5), np.int64) + np.arange(5)
    ids[n - 3:] = np.argsort(-tail, 1)[:, :5]
    top = np.zeros((n, 5), np.float32)
    top[n - 3:] = r.standard_normal((3, 5))
    di, dt, one = D(ids), D(top), D(np.ones(1, np.float32))
    loss, row, lse, rest = (A((m,)) for m in (1, n, n, n))
    hip.call("oxi_distill_fwd", x.ptr, di.ptr, dt.ptr, None, loss.ptr, row.ptr, lse.ptr, rest.ptr, d.ptr, n, c, 5, 1.0, 3.0)
    # the same rows by themselves, at the same place in their 16 bytes: which classes share a float4, and so the
    # order of a row's sums, goes by it
    phase = (n - 3) * c % 4
    sd, sg = D(np.concatenate([np.zeros(phase, np.float32), tail.ravel()])), A((phase + 3 * c,))
    si, st, sl, srow, slse, srest = D(ids[n - 3:]), D(top[n - 3:]), A((1,)), A((3,)), A((3,)), A((3,))
    at = 4 * phase
    hip.call("oxi_distill_fwd", sd.ptr + at, si.ptr, st.ptr, None, sl.ptr, srow.ptr, slse.ptr, srest.ptr, sg.ptr + at, 3, c, 5,
             1.0, 3.0)
    assert np.array_equal(row.numpy()[n - 3:], srow.numpy())
    assert np.array_equal(take(hip, d.ptr + (n - 3) * c * 4, (3, c)), take(hip, sg.ptr + at, (3, c)))
    hip.call("oxi_distill_bwd", x.ptr, di.ptr, dt.ptr, None, lse.ptr, rest.ptr, one.ptr, d.ptr, n, c, 5, 1.0, 3.0)
    hip.call("oxi_distill_bwd", sd.ptr + at, si.ptr, st.ptr, None, slse.ptr, srest.ptr, one.ptr, sg.ptr + at, 3, c, 5, 1.0, 3.0)
    assert np.array_equal(take(hip, d.ptr + (n - 3) * c * 4, (3, c)), take(hip, sg.ptr + at, (3, c)))


def test_verify(hip):
    from test_gpu_verify import make, oracle

    b, k, v = 5, 70, 6 << 20  # 2.2e9 target probabilities
    print("[case] large verify", b, k, v, flush=True)
    assert b * (k + 1) * v > 1 << 31
    A, D = hip.DeviceArray, hip.DeviceArray.from_numpy
    target = A((b * (k + 1) * v,))
    draft = A((b * k * v,))
    for t in (target, draft):
        hip.call("oxi_fill", t.ptr, t.size, 0.0)
    tokens = np.full((b, k), 7, np.int64)
    u = np.zeros((b, k + 1), np.float32)
    one = np.ones(1, np.float32)
    for s in range(b):
        for i in range(k):  # target 1 at the token: every draft is kept
            put(hip, target.ptr + ((s * (k + 1) + i) * v + 7) * 4, one)
    # the last sequence: its last draft is judged by real rows, far into both buffers
    tg, dr, tk, uu = make(1, 1, v, 4, scale=1.0)
    put(hip, target.ptr + ((b - 1) * (k + 1) + k - 1) * v * 4, tg[0])
    put(hip, draft.ptr + ((b - 1) * k + k - 1) * v * 4, dr[0])
    put(hip, target.ptr + ((b - 1) * (k + 1) + k) * v * 4, tg[0, 1])
    tokens[b - 1, k - 1] = tk[0, 0]
    for draw in (0.1, 0.999):
        u[b - 1, k - 1:] = draw
        acc, out = A((b,), np.int64), A((b, k + 1), np.int64)
        dt, du = D(tokens), D(u)
        hip.call("oxi_verify_drafts", target.ptr, draft.ptr, dt.ptr, None, du.ptr, acc.ptr, out.ptr, None, b, k, v)
        wa, wo, margin = oracle(tg, dr, tk, np.full((1, 2), draw, np.float32))
        assert (margin > 1e-12).all()
        a, o = acc.numpy(), out.numpy()
        assert (a[:b - 1] == k).all() and (o[:b - 1, k] == -1).all() and (o[:, :k - 1] == 7).all()
        assert a[b - 1] == k - 1 + wa[0]
        assert np.array_equal(o[b - 1, k - 1:], wo[0])
