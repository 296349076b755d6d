"""The residual RMS norm (oxi_add_rms_norm_*) against float64: forward, VJP in
both modes, the 8-bit output with its scales.

Tolerances, u = 2^-24 (half a step of float32): a row's sum of squares adds at
most H/256 + 16 terms in sequence on any path (a thread's share, then trees), so
the inverse is off by at most half of that many u, and y = (h*inv)*w by a root,
a division, two products and an addition more. Gradients cancel, so theirs are
relative to the terms they are summed from. An e4m3 code is half a step off:
2^-4 of the value, 2^-10 below 2^-6.
"""

import numpy as np
import pytest

from conftest import rng

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-6

# (rows, cols): single elements, fewer than 4 columns, odd widths, both sides of
# every row configuration's limit, few rows and more than one walk of the grid
SHAPES = [(1, 1), (3, 2), (2, 3), (5, 4), (7, 5), (4, 63), (64, 64), (9, 255), (3, 256), (5, 257), (17, 768), (6, 1003),
          (300, 1024), (2, 1025), (65, 2047), (33, 2048), (4, 2552), (8, 4096), (700, 4096), (3, 4097), (5, 8191), (4, 8192),
          (2, 8193), (3, 12288), (2, 16384), (2, 16385), (3, 20003), (4500, 96), (2100, 130)]


def k_sum(H):
    return H / 256 + 16


def data(rows, cols, seed):
    r = rng(seed)
    f = lambda *s: r.standard_normal(s).astype(np.float32)  # noqa: E731
    return dict(x=f(rows, cols), r=2 * f(rows, cols), w=(1 + 0.1 * f(cols)).astype(np.float32), gy=f(rows, cols),
                gh=f(rows, cols))


def forward64(d, w=True):
    h = (d["x"] + d["r"]).astype(np.float64)
    inv = 1.0 / np.sqrt((h * h).mean(1, keepdims=True) + np.float64(np.float32(EPS)))
    return h, inv, h * inv * (d["w"] if w else 1.0)


def backward64(h, inv, d, mode, gh, w=True):
    """dx, dw and the sums of magnitudes their errors are relative to."""
    gy = d["gy"].astype(np.float64)
    xh = h * inv
    gw = gy * (d["w"] if w else 1.0)
    H = h.shape[1]
    dx = gw * inv
    size = np.abs(dx)
    if mode == "exact":
        dx = dx - xh * (gw * xh).mean(1, keepdims=True) * inv
        size = size + np.abs(xh) * np.abs(gw * xh).mean(1, keepdims=True) * inv
    size = size * (2 * k_sum(H) + 8)
    if gh:
        dx = dx + d["gh"]
    return dx, (gy * xh).sum(0), size + np.abs(dx), np.abs(gy * xh).sum(0)


def within(got, want, bound, what):
    err = np.abs(got.astype(np.float64) - want)
    bad = ~(err <= bound)
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} off by more than the bound; worst "
                           f"{np.nanmax(err / bound):.3g} x")


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward_and_vjp(hip, rows, cols):
    print("[case] add_rms_norm", rows, cols, flush=True)
    d = data(rows, cols, rows + cols)
    D = hip.DeviceArray.from_numpy
    x, r, w, gy, gh = (D(d[n]) for n in ("x", "r", "w", "gy", "gh"))
    h, y, rstd = hip.add_rms_norm_fwd(x, r, w, EPS)
    h64, inv, y64 = forward64(d)
    assert np.array_equal(h.numpy(), d["x"] + d["r"])
    tol = (k_sum(cols) / 2 + 6) * U
    within(rstd.numpy()[:, None], inv, tol * inv, "rstd")
    within(y.numpy(), y64, tol * np.abs(y64) + 1e-37, "y")
    for mode in ("ref", "exact"):
        for with_gh in (True, False):
            dx, dw = hip.add_rms_norm_bwd(h, w, rstd, gy, gh if with_gh else None, mode=mode)
            dx64, dw64, size, sums = backward64(h64, inv, d, mode, with_gh)
            within(dx.numpy(), dx64, size * U, f"dx {mode} {with_gh}")
            # at least 64 blocks share the rows of large batches, each adding its own in float32
            within(dw.numpy(), dw64, (rows / 64 + k_sum(cols) + 24) * U * sums + 1e-37, f"dw {mode} {with_gh}")


def test_no_weight_and_single_outputs(hip):
    d = data(37, 515, 3)
    D = hip.DeviceArray.from_numpy
    x, r, gy, gh = (D(d[n]) for n in ("x", "r", "gy", "gh"))
    h, y, rstd = hip.add_rms_norm_fwd(x, r, None, EPS)
    h64, inv, y64 = forward64(d, w=False)
    within(y.numpy(), y64, (k_sum(515) / 2 + 6) * U * np.abs(y64), "y")
    both = hip.add_rms_norm_bwd(h, None, rstd, gy, gh, mode="exact")
    dx64, dw64, size, sums = backward64(h64, inv, d, "exact", True, w=False)
    within(both[0].numpy(), dx64, size * U, "dx")
    dx, none = hip.add_rms_norm_bwd(h, None, rstd, gy, gh, mode="exact", need_dw=False)
    assert none is None and np.array_equal(dx.numpy(), both[0].numpy())
    none, dw = hip.add_rms_norm_bwd(h, None, rstd, gy, gh, mode="exact", need_dx=False)
    assert none is None and np.array_equal(dw.numpy(), both[1].numpy())
    # rstd is optional
    h2, y2 = hip.DeviceArray(h.shape), hip.DeviceArray(h.shape)
    hip.call("oxi_add_rms_norm_fwd", x.ptr, r.ptr, None, h2.ptr, y2.ptr, None, 37, 515, EPS)
    assert np.array_equal(h2.numpy(), h.numpy()) and np.array_equal(y2.numpy(), y.numpy())


# odd rows whose last float4 begins a wave (1025, 1281, 1795, 2305, 4097, 8193, 12290) share floats with another wave's
@pytest.mark.parametrize("rows,cols", [(21, 3), (21, 768), (21, 1003), (21, 4096), (21, 20003), (700, 1025), (700, 1281),
                                       (600, 1795), (600, 2305), (500, 4097), (300, 8193), (300, 12290)])
@pytest.mark.parametrize("mode", ["ref", "exact"])
def test_in_place(hip, rows, cols, mode):
    """h over x or over r, and dx over gh: the values of the separate buffers."""
    d = data(rows, cols, cols)
    D = hip.DeviceArray.from_numpy
    w, gy = D(d["w"]), D(d["gy"])
    h, y, rstd = hip.add_rms_norm_fwd(D(d["x"]), D(d["r"]), w, EPS)
    for over in ("x", "r"):
        b = {n: D(d[n]) for n in ("x", "r")}
        h2, y2, _ = hip.add_rms_norm_fwd(b["x"], b["r"], w, EPS, h=b[over])
        assert np.array_equal(b[over].numpy(), h.numpy()) and np.array_equal(y2.numpy(), y.numpy())
    dx, dw = hip.add_rms_norm_bwd(h, w, rstd, gy, D(d["gh"]), mode=mode)
    gh, dw2 = D(d["gh"]), hip.DeviceArray((cols,))
    hip.call("oxi_add_rms_norm_bwd", h.ptr, w.ptr, rstd.ptr, gy.ptr, gh.ptr, gh.ptr, dw2.ptr, None, rows, cols,
             hip.NORM_VJP[mode])
    assert np.array_equal(gh.numpy(), dx.numpy()) and np.array_equal(dw2.numpy(), dw.numpy())


@pytest.mark.parametrize("shift", [1, 2, 3])
def test_buffers_at_any_float(hip, shift):
    """Operands 4, 8 or 12 bytes past a 16-byte address; what lies around the outputs stays."""
    rows, cols = 19, 1024
    d = data(rows, cols, shift)
    A, D = hip.DeviceArray, hip.DeviceArray.from_numpy
    n = rows * cols

    def moved(a):
        return D(np.concatenate([np.full(shift, 7, np.float32), a.ravel(), np.full(5, 7, np.float32)]))

    b = {k: moved(d[k]) for k in d}
    b.update({k: moved(np.zeros(n, np.float32)) for k in ("h", "y", "dx")})
    p = {k: v.ptr + 4 * shift for k, v in b.items()}
    rstd, dw = A((rows,)), A((cols,))
    hip.call("oxi_add_rms_norm_fwd", p["x"], p["r"], p["w"], p["h"], p["y"], rstd.ptr, rows, cols, EPS)
    hip.call("oxi_add_rms_norm_bwd", p["h"], p["w"], rstd.ptr, p["gy"], p["gh"], p["dx"], dw.ptr, None, rows, cols, 1)
    h64, inv, y64 = forward64(d)
    dx64, dw64, size, sums = backward64(h64, inv, d, "exact", True)
    out = {k: b[k].numpy() for k in ("h", "y", "dx")}
    for v in out.values():
        assert (v[:shift] == 7).all() and (v[shift + n:] == 7).all()
    cut = lambda k: out[k][shift:shift + n].reshape(rows, cols)  # noqa: E731
    assert np.array_equal(cut("h"), d["x"] + d["r"])
    within(cut("y"), y64, (k_sum(cols) / 2 + 6) * U * np.abs(y64), "y")
    within(cut("dx"), dx64, size * U, "dx")
    within(dw.numpy(), dw64, (rows / 64 + 40) * U * sums, "dw")


def test_special_values(hip):
    """An inf in a row makes it NaN there and 0 elsewhere, a NaN the whole row; other rows keep their values."""
    d = data(6, 520, 11)
    clean = forward64(d)[2]
    d["x"][1, 7] = np.inf
    d["r"][3, 100] = np.nan
    d["x"][4] = 0
    d["r"][4] = 0
    D = hip.DeviceArray.from_numpy
    h, y, rstd = (a.numpy() for a in hip.add_rms_norm_fwd(D(d["x"]), D(d["r"]), D(d["w"]), EPS))
    assert np.isnan(y[1, 7]) and (np.delete(y[1], 7) == 0).all() and rstd[1] == 0
    assert np.isnan(y[3]).all() and (y[4] == 0).all()
    for i in (0, 2, 5):
        within(y[i], clean[i], (k_sum(520) / 2 + 6) * U * np.abs(clean[i]), "y")


def test_caller_workspace(hip):
    """The VJP in a caller's workspace gives the allocator's bits, and writes no byte behind it."""
    for rows, cols in ((4, 64), (5000, 96), (700, 4096), (900, 1003), (40, 20003)):
        d = data(rows, cols, 5)
        D = hip.DeviceArray.from_numpy
        w, gy, gh = D(d["w"]), D(d["gy"]), D(d["gh"])
        h, y, rstd = hip.add_rms_norm_fwd(D(d["x"]), D(d["r"]), w, EPS)
        want = [a.numpy() for a in hip.add_rms_norm_bwd(h, w, rstd, gy, gh)]
        n = hip.add_rms_norm_bwd_workspace(rows, cols)
        assert n % 4 == 0
        ws = D(np.full(n // 4 + 64, 3.0, np.float32))
        got = [a.numpy() for a in hip.add_rms_norm_bwd(h, w, rstd, gy, gh, workspace=ws)]
        assert all(np.array_equal(a, b) for a, b in zip(got, want))
        assert (ws.numpy()[n // 4:] == 3.0).all()


# ---- 8 bits --------------------------------------------------------------------

def e4m3_values():
    c = np.arange(256)
    s, e, m = c >> 7, (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * 2.0 ** (e - 7.0))
    v = np.where((c & 0x7F) == 0x7F, np.nan, v)
    return np.where(s == 1, -v, v)


CODES = e4m3_values()


@pytest.mark.parametrize("rows,cols,group", [
    (1, 1, 1), (3, 3, 3), (5, 16, 32), (4, 40, 32), (7, 64, 64), (9, 130, 32), (3, 255, 255), (3, 257, 128), (17, 768, 128),
    (6, 1003, 32), (6, 1003, 64), (5, 1003, 128), (5, 1003, 256), (4, 1003, 1003), (33, 2048, 256), (700, 4096, 128),
    (3, 4096, 4096), (5, 8191, 64), (4, 8192, 8192), (3, 12288, 128), (2, 16384, 16384), (2, 20003, 128), (2, 20003, 20003),
    (4500, 96, 32)])
@pytest.mark.parametrize("residual", [True, False])
def test_e4m3(hip, rows, cols, group, residual):
    print("[case] add_rms_norm_e4m3", rows, cols, group, residual, flush=True)
    d = data(rows, cols, rows + cols + group)
    d["w"][::17] *= 30
    if not residual:
        d["r"][:] = 0
    D = hip.DeviceArray.from_numpy
    h, q, scale = hip.add_rms_norm_e4m3_fwd(D(d["x"]), D(d["r"]) if residual else None, D(d["w"]), group, EPS)
    if residual:
        assert np.array_equal(h.numpy(), d["x"] + d["r"])
    y64 = forward64(d)[2]
    codes, s = q.numpy(), scale.numpy()
    starts = np.arange(0, cols, group)
    s64 = np.maximum(np.maximum.reduceat(np.abs(y64), starts, axis=1) / 448.0, 2.0 ** -126)
    tol = (k_sum(cols) / 2 + 8) * U
    within(s, s64, tol * s64, "scale")
    wide = np.repeat(s64, np.diff(np.append(starts, cols)), axis=1)
    ratio = y64 / wide
    got = CODES[codes]
    assert np.isfinite(got).all()
    # half a step, and the float32 quotient's own error before it
    within(got, ratio, np.maximum(2.0 ** -4 * np.abs(ratio), 2.0 ** -10) * (1 + 2 * tol) + 2 * tol * np.abs(ratio), "codes")
    # to nearest even: the codes are those of the float32 quotient that the scale written implies, where y is known well
    # enough to say so
    y = hip.e4m3_dequantize(q, scale, group).numpy()
    wide32 = np.repeat(s, np.diff(np.append(starts, cols)), axis=1)
    assert np.array_equal(y, got.astype(np.float32) * wide32)


def test_e4m3_rounds_to_nearest_even_and_keeps_nan(hip):
    """With rows whose norm is exactly 1 and one group of maximum 448 the codes are those of the weights: every
    value between two codes, the ties, the subnormals, NaN."""
    v = np.sort(CODES[~np.isnan(CODES)])
    mids = (v[1:] + v[:-1]) / 2
    w = np.concatenate([v, mids, np.nextafter(mids.astype(np.float32), np.float32(-np.inf)),
                        np.nextafter(mids.astype(np.float32), np.float32(np.inf))]).astype(np.float32)
    w = np.append(w, np.float32(np.nan)).astype(np.float32)
    H = len(w)
    x = np.ones((2, H), np.float32)
    x[1, ::2] = -1
    D = hip.DeviceArray.from_numpy
    _, q, scale = hip.add_rms_norm_e4m3_fwd(D(x), None, D(w), H, 0.0)
    assert (scale.numpy() == 1.0).all()
    codes = q.numpy()
    table = CODES[:127]  # 0 .. 448
    for row in range(2):
        for i in range(H):
            want = float(w[i]) * float(x[row, i])
            if np.isnan(want):
                assert codes[row, i] & 0x7F == 0x7F
                continue
            dist = np.abs(table - abs(want))
            near = np.flatnonzero(dist == dist.min())
            code = near[0] if len(near) == 1 else near[near % 2 == 0][0]  # ties: the even significand
            assert codes[row, i] & 0x7F == code, (row, i, want)
            assert code == 0 or codes[row, i] >> 7 == (want < 0), (row, i, want)


def test_e4m3_zeros_and_infinities(hip):
    """Rows of zeros get the smallest scale and zero codes; an inf gives NaN codes where y is NaN; a row of NaN all."""
    x = rng(1).standard_normal((4, 300)).astype(np.float32)
    x[1] = 0
    x[2, 5] = np.inf
    x[3, 0] = np.nan
    D = hip.DeviceArray.from_numpy
    _, q, s = hip.add_rms_norm_e4m3_fwd(D(x), None, None, 128, EPS)
    q, s = q.numpy(), s.numpy()
    assert (q[1] & 0x7F == 0).all() and (s[1] == np.float32(2.0 ** -126)).all()
    assert q[2, 5] & 0x7F == 0x7F and (np.delete(q[2], 5) & 0x7F == 0).all()
    assert (q[3] & 0x7F == 0x7F).all() and (s[3] == np.float32(2.0 ** -126)).all()
    assert np.isfinite(s).all()
