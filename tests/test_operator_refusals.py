"""What the residual norm, rotary, distillation and draft verification entry
points refuse, no GPU: arguments are checked before any device use."""

import numpy as np
import pytest

N = 1 << 40


@pytest.fixture(scope="module")
def capi():
    from oxitorch_amd import capi

    return capi


P = 1 << 20  # a non-NULL address that no refused call touches


def test_add_rms_norm(capi):
    call = capi.call
    fwd, bwd, q8 = "oxi_add_rms_norm_fwd", "oxi_add_rms_norm_bwd", "oxi_add_rms_norm_e4m3_fwd"
    with pytest.raises(ValueError, match="negative size"):
        call(fwd, P, P, P, P, P, P, -1, 4, 1e-6)
    with pytest.raises(ValueError, match="exceeds the kernel limits"):
        call(fwd, P, P, P, P, P, P, 1 << 31, 4, 1e-6)
    with pytest.raises(ValueError, match="exceeds the kernel limits"):
        call(fwd, P, P, P, P, P, P, 1, N, 1e-6)
    with pytest.raises(ValueError, match="zero-length last dim"):
        call(fwd, P, P, P, P, P, P, 2, 0, 1e-6)
    for i in (0, 1, 3, 4):
        a = [P, P + 64, P + 128, P + 192, P + 256, P + 320]
        a[i] = None
        with pytest.raises(ValueError, match="NULL tensor"):
            call(fwd, *a, 2, 4, 1e-6)
    with pytest.raises(ValueError, match="y must not be"):
        call(fwd, P, P + 64, P, P + 128, P, P, 2, 4, 1e-6)
    with pytest.raises(ValueError, match="unknown VJP mode"):
        call(bwd, P, P, P, P, P, P, P, None, 2, 4, 7)
    with pytest.raises(ValueError, match="NULL tensor"):
        call(bwd, P, P, None, P, P, P, P, None, 2, 4, 0)
    with pytest.raises(ValueError, match="dx must not be"):
        call(bwd, P, P, P, P + 64, P, P, P, None, 2, 4, 0)
    with pytest.raises(ValueError, match="8-byte aligned"):
        call(bwd, P, P, P, P, P, P + 64, P, P + 4, 2, 4, 0)
    for g in (0, -1, 1, 16, 96, 512, 5000):
        with pytest.raises(ValueError, match="groups of"):
            call(q8, P, P, P, P, P, P, 2, 4096, g, 1e-6)
    with pytest.raises(ValueError, match="NULL tensor"):
        call(q8, P, P, P, None, P, P, 2, 4096, 128, 1e-6)  # a residual without h
    with pytest.raises(ValueError, match="NULL tensor"):
        call("oxi_e4m3_dequantize", P, None, P, 2, 64, 32)
    with pytest.raises(ValueError, match="groups of"):
        call("oxi_e4m3_dequantize", P, P, P, 2, 64, 48)
    with pytest.raises(ValueError, match="NULL result"):
        call("oxi_add_rms_norm_bwd_workspace", 2, 64, None)


def test_rotary(capi):
    i64 = capi._i64arr
    sh, st = i64((2, 3, 4, 8)), i64((96, 32, 8, 1))

    def rotary(x=P, xs=st, y=2 * P, ys=st, shape=sh, pos=P, ps=i64((3, 1)), freq=P, rot=8, layout=0):
        capi.call("oxi_rotary", x, xs, y, ys, shape, pos, ps, 0, freq, rot, layout, 0, 1.0)

    with pytest.raises(ValueError, match="negative size"):
        rotary(shape=i64((2, -3, 4, 8)))
    with pytest.raises(ValueError, match="exceeds the kernel limits"):
        rotary(shape=i64((N, N, 4, 8)))
    for rot in (-2, 3, 10):
        with pytest.raises(ValueError, match="an even number"):
            rotary(rot=rot)
    with pytest.raises(ValueError, match="unknown layout"):
        rotary(layout=2)
    with pytest.raises(ValueError, match="without strides"):
        rotary(ps=None)
    with pytest.raises(ValueError, match="NULL shape"):
        rotary(xs=None)
    for name in ("x", "y", "freq"):
        with pytest.raises(ValueError, match="NULL tensor"):
            rotary(**{name: None})
    with pytest.raises(ValueError, match="broadcast"):
        rotary(ys=i64((0, 32, 8, 1)))
    with pytest.raises(ValueError, match="in place"):
        rotary(y=P, xs=i64((96, 8, 24, 1)))


def test_distill(capi):
    def fwd(n=2, c=50, k=4, T=1.0, div=2.0, drop=None):
        a = [P] * 9
        if drop is not None:
            a[drop] = None
        capi.call("oxi_distill_fwd", *a, n, c, k, T, div)

    with pytest.raises(ValueError, match="negative size"):
        fwd(n=-1)
    with pytest.raises(ValueError, match="kernel limits"):
        fwd(c=1 << 31)
    with pytest.raises(ValueError, match="kernel limits"):
        fwd(n=1 << 24)
    for k in (0, 1025):
        with pytest.raises(ValueError, match="teacher entries"):
            fwd(k=k)
    for T in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="temperature"):
            fwd(T=T)
        with pytest.raises(ValueError, match="divisor"):
            fwd(div=T)
    with pytest.raises(ValueError, match="zero classes"):
        fwd(c=0)
    for i in (0, 1, 2, 4, 5, 6, 7):
        with pytest.raises(ValueError, match="NULL"):
            fwd(drop=i)
    with pytest.raises(ValueError, match="NULL tensor"):
        capi.call("oxi_distill_bwd", P, P, P, None, P, P, None, P, 2, 50, 4, 1.0, 2.0)


def test_verify(capi):
    def verify(batch=2, drafts=3, vocab=50, drop=None, ws=None):
        a = [P] * 7 + [ws]
        if drop is not None:
            a[drop] = None
        capi.call("oxi_verify_drafts", *a, batch, drafts, vocab)

    for kw in ({"batch": -1}, {"drafts": -1}, {"vocab": -1}):
        with pytest.raises(ValueError, match="negative size"):
            verify(**kw)
    for kw in ({"batch": N}, {"drafts": N}, {"vocab": N}):
        with pytest.raises(ValueError, match="kernel limits"):
            verify(**kw)
    with pytest.raises(ValueError, match="zero classes"):
        verify(vocab=0)
    for i in (0, 2, 4, 5, 6):
        with pytest.raises(ValueError, match="NULL tensor"):
            verify(drop=i)
    with pytest.raises(ValueError, match="8-byte aligned"):
        verify(ws=P + 4)
    with pytest.raises(ValueError, match="NULL result"):
        capi.call("oxi_verify_drafts_workspace", 2, 50, None)
    assert capi.verify_drafts_workspace(0, 50) == 0
