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
    with pytest.raises(ValueError, match="16-byte aligned"):
        call(bwd, P, P, P, P, P, P + 64, P, P + 8, 2, 4, 0)
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
    with pytest.raises(ValueError, match="32-bit reciprocal"):
        fwd(T=1e-40)
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


# ---- the Python surface, on host tensors ----------------------------------------------

def test_rotary_frequencies():
    from oxitorch_amd.nn import functional as F

    inv, scale = F.rotary_frequencies(64)
    assert scale == 1.0 and inv.dtype == np.float64
    assert np.allclose(inv, [10000.0 ** (-2 * i / 64) for i in range(32)], rtol=1e-15)
    lin, _ = F.rotary_frequencies(64, scaling={"type": "linear", "factor": 8})
    assert np.array_equal(lin, inv / 8)
    # the slowest pair is divided by the factor, the fastest kept
    ntk, _ = F.rotary_frequencies(64, scaling={"type": "ntk", "factor": 8.0})
    assert ntk[0] == 1.0 and np.isclose(ntk[-1], inv[-1] / 8, rtol=1e-12)
    assert (ntk <= inv).all() and (ntk >= inv / 8 * (1 - 1e-12)).all()
    yarn, m = F.rotary_frequencies(64, scaling={"type": "yarn", "factor": 8.0, "original_length": 4096})
    turns = 4096 * inv / (2 * np.pi)
    assert np.allclose(yarn[turns >= 32], inv[turns >= 32]) and np.allclose(yarn[turns <= 1], inv[turns <= 1] / 8)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and (yarn[mid] < inv[mid]).all() and (yarn[mid] > inv[mid] / 8).all()
    assert np.isclose(m, 0.1 * np.log(8) + 1)
    assert F.rotary_frequencies(64, scaling={"type": "yarn", "factor": 8.0, "original_length": 4096, "scale": 1.0})[1] == 1.0
    assert F.rotary_frequencies(2, scaling={"type": "ntk", "factor": 8.0})[0].tolist() == [1.0]
    assert F.rotary_frequencies(0)[0].size == 0


def test_python_refusals():
    import oxitorch_amd as ox
    from oxitorch_amd import nn
    from oxitorch_amd.nn import functional as F

    for dim in (3, -2):
        with pytest.raises(ValueError, match="even number"):
            F.rotary_frequencies(dim)
    for base in (0, -1, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="base"):
            F.rotary_frequencies(8, base)
    for kw in ({"type": "linear", "factor": 0}, {"type": "ntk", "factor": -1}):
        with pytest.raises(ValueError, match="factor"):
            F.rotary_frequencies(8, scaling=kw)
    with pytest.raises(ValueError, match="unknown rotary scaling"):
        F.rotary_frequencies(8, scaling={"type": "cubic", "factor": 2})
    with pytest.raises(ValueError, match="above slow"):
        F.rotary_frequencies(8, scaling={"type": "yarn", "factor": 2, "original_length": 64, "slow": 4, "fast": 2})
    with pytest.raises(KeyError):
        F.rotary_frequencies(8, scaling={"type": "yarn", "factor": 2})
    with pytest.raises(ValueError, match="layout"):
        nn.RotaryEmbedding(8, layout="both")
    cpu = lambda *s: ox.from_numpy(np.zeros(s, np.float32), device="cpu")  # noqa: E731
    ids = np.zeros((3, 2), np.int64)
    with pytest.raises(ValueError, match="teacher_ids"):
        F.distillation_loss(cpu(3, 8), ids[0], cpu(3, 2))
    with pytest.raises(IndexError, match="index 8 is out of bounds"):
        F.distillation_loss(cpu(3, 8), ids + 8, cpu(3, 2))
    with pytest.raises(TypeError, match="integers"):
        F.distillation_loss(cpu(3, 8), ids * 1.0, cpu(3, 2))
    with pytest.raises(ValueError, match="teacher_logits"):
        F.distillation_loss(cpu(3, 8), ids, cpu(3, 3))
    with pytest.raises(NotImplementedError):  # host tensors do not reach device compute
        F.distillation_loss(cpu(3, 8), ids, cpu(3, 2))
    with pytest.raises(ValueError, match="draft_tokens"):
        F.verify_drafts(ids, None, cpu(3, 2, 8), cpu(3, 2))
    with pytest.raises(TypeError, match="integers"):
        F.verify_drafts(ids * 1.0, None, cpu(3, 3, 8), cpu(3, 3))
    with pytest.raises(ValueError, match="shape mismatch"):
        F.verify_drafts(ids, None, cpu(3, 3, 8), cpu(3, 2))
    with pytest.raises(ValueError, match="a length of 3 of 2"):
        F.verify_drafts(ids, None, cpu(3, 3, 8), cpu(3, 3), [0, 3, 0])
    with pytest.raises(ValueError, match="2 lengths for batch of 3"):
        F.verify_drafts(ids, None, cpu(3, 3, 8), cpu(3, 3), [0, 1])
    with pytest.raises(RuntimeError, match="index 8 is out of bounds"):
        F.verify_drafts(ids + 8, None, cpu(3, 3, 8), cpu(3, 3))
    with pytest.raises(NotImplementedError):
        F.verify_drafts(ids, None, cpu(3, 3, 8), cpu(3, 3))


def test_host_operands_of_the_norm():
    import oxitorch_amd as ox
    from oxitorch_amd.nn import functional as F

    x, r, w = (ox.from_numpy(np.zeros(s, np.float32), device="cpu") for s in ((3, 8), (3, 8), (8,)))
    with pytest.raises(NotImplementedError, match="add_rms_norm"):
        F.add_rms_norm(x, r, w)
    for residual in (r, None):
        with pytest.raises(NotImplementedError, match="add_rms_norm_e4m3"):
            F.add_rms_norm_e4m3(x, residual, w)


def test_integers_past_int64():
    """As elsewhere, no wrapping: 2^64 - 1 would become -1, which is padding."""
    import oxitorch_amd as ox
    from oxitorch_amd.nn import functional as F

    cpu = lambda *s: ox.from_numpy(np.zeros(s, np.float32), device="cpu")  # noqa: E731
    ids = np.full((3, 2), 2 ** 64 - 1, np.uint64)
    with pytest.raises(OverflowError, match="teacher_ids"):
        F.distillation_loss(cpu(3, 8), ids, cpu(3, 2))
    with pytest.raises(OverflowError, match="draft_tokens"):
        F.verify_drafts(ids, None, cpu(3, 3, 8), cpu(3, 3))
    with pytest.raises(OverflowError, match="lengths"):
        F.verify_drafts(np.zeros((3, 2), np.uint64), None, cpu(3, 3, 8), cpu(3, 3), ids[:, 0])
    with pytest.raises(OverflowError, match="positions"):
        F.rotary_embedding(cpu(2, 3, 4), [1.0], ids[0])
