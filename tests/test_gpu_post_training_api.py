"""Token log-probabilities, the policy and preference losses and gradient clipping
through the Python surface: graph nodes, other upstreams, views, a run of them
together, and graph capture of their C-ABI calls. The bounds are derived in
token_oracle.py."""

import ctypes

import numpy as np
import pytest

from conftest import rng
from test_gpu_token_logp import chosen, logits_of
from token_oracle import Rows, U, near, policy, preference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ox(hip):
    import oxitorch_amd

    return oxitorch_amd


@pytest.fixture(scope="module")
def F(ox):
    return ox.nn.functional


def test_token_log_probs(ox, F):
    x = logits_of(7, 501, 1)
    ids = chosen(x, 2, pad=0.3)
    t = ox.from_numpy(x, True)
    lp, H = F.token_log_probs(t, ids, temperature=0.8, entropy=True)
    r = Rows(x, ids, 0.8)
    near(lp.numpy(), r.logp, r.b_logp, "logp")
    near(H.numpy(), r.entropy, r.b_entropy, "entropy")
    g = rng(3).standard_normal((2, 7)).astype(np.float32)
    ((lp * ox.from_numpy(g[0])).sum() + (H * ox.from_numpy(g[1])).sum()).backward()
    near(t.grad.numpy(), *r.gradient(g[0], g[1]), "gradient of both")
    t.zero_grad()
    only = F.token_log_probs(t, list(int(i) for i in ids), temperature=0.8)
    assert np.array_equal(only.numpy(), lp.numpy()) and only.shape == [7]
    only.sum().backward()
    near(t.grad.numpy(), *r.gradient(np.ones(7)), "gradient of the sum")
    t.zero_grad()
    _, H = F.token_log_probs(t, ids, 0.8, True)
    H.sum().backward()
    near(t.grad.numpy(), *r.gradient(np.zeros(7), np.ones(7)), "gradient of the entropy alone")
    with ox.no_grad():
        free = F.token_log_probs(t, ids, 0.8)
    assert not free.requires_grad and np.array_equal(free.numpy(), lp.numpy())


def test_token_log_probs_of_a_view(ox, F):
    x = logits_of(40, 9, 5)
    ids = chosen(x, 6)
    t = ox.from_numpy(np.ascontiguousarray(x.T), True)
    F.token_log_probs(t.transpose(), ids).sum().backward()
    r = Rows(x, ids)
    want, bound = r.gradient(np.ones(40))
    near(t.grad.numpy(), want.T, bound.T, "through a transposed view")


@pytest.mark.parametrize("one_pass", [True, False])
def test_policy_loss(ox, F, one_pass):
    from oxitorch_amd import _native

    x = logits_of(12, 700, 7)
    ids = chosen(x, 8, pad=0.25)
    r = Rows(x, ids, 1.2)
    q = rng(9)
    adv = q.standard_normal(12).astype(np.float32)
    old = (r.logp - 0.1 * q.choice([-1, 1], 12)).astype(np.float32)
    ref = (r.logp + 0.2 * q.standard_normal(12)).astype(np.float32)
    n = float((ids >= 0).sum())
    w = policy(r, adv, old, ref, clip=(0.05, 0.3), clip_max=2.0, kl=0.1, ent=0.01, divisor=n)
    kw = dict(clip=(0.05, 0.3), clip_max=2.0, kl=0.1, entropy=0.01, temperature=1.2)
    was = _native.set_ce_one_pass(one_pass)
    try:
        t = ox.from_numpy(x, True)
        loss, more = F.policy_loss(t, ids, adv, ox.from_numpy(old), ref, stats=True, **kw)
        near([loss.item(), *more.numpy()], w["out"], w["bout"], "loss and stats")
        loss.backward(retain_graph=True)
        want, bound = r.gradient(w["cl"], w["ch"], w["bcl"], w["bch"])
        near(t.grad.numpy(), want, bound, "gradient")
        t.zero_grad()
        loss.backward()  # the second backward is a pass of its own
        near(t.grad.numpy(), want, bound, "second backward")
        t.zero_grad()
        (F.policy_loss(t, ids, adv, old, ref, **kw) * -3.0).backward()
        near(t.grad.numpy(), *r.gradient(-3 * w["cl"], -3 * w["ch"], 3 * w["bcl"], 3 * w["bch"]), "another upstream")
    finally:
        _native.set_ce_one_pass(was)
    with ox.no_grad():
        assert not F.policy_loss(t, ids, adv, old, ref, **kw).requires_grad


def test_policy_loss_weights(ox, F):
    """Each sequence's mean counts alike; a weight of 0 is padding."""
    x = logits_of(6, 50, 11)
    x[5] = np.nan
    ids = chosen(logits_of(6, 50, 11), 12)
    adv = np.array([1, -1, 2, 0.5, 1, np.nan], np.float32)
    weights = np.array([1 / 6, 1 / 6, 1 / 6, 1 / 4, 1 / 4, 0], np.float32)
    clean = np.where(np.isnan(x), 0, x)
    r = Rows(clean, ids, counted=weights != 0)
    w = policy(r, np.nan_to_num(adv), weights=weights)
    t = ox.from_numpy(x, True)
    loss = F.policy_loss(t, ids, adv, weights=weights)
    near([loss.item()], w["out"][:1], w["bout"][:1], "loss")
    loss.backward()
    near(t.grad.numpy(), *r.gradient(w["cl"], None, w["bcl"]), "gradient")


@pytest.mark.parametrize("one_pass", [True, False])
def test_preference_loss(ox, F, one_pass):
    from oxitorch_amd import _native

    lengths = np.array([[5, 3], [2, 6]])
    x = logits_of(18, 300, 13)  # two rows behind the last sequence
    ids = chosen(x, 14)
    ids[[0, 1, 5, 8, 10]] = -1
    starts = np.concatenate([[0], np.cumsum(lengths.ravel())])
    on = (ids >= 0) & (np.arange(18) < 16)
    r = Rows(x, ids, counted=on)
    ref = (r.logp + 0.3 * rng(15).standard_normal(18)).astype(np.float32)
    w = preference(r, starts, ref, beta=0.4, smoothing=0.1, margin=0.2)
    kw = dict(beta=0.4, smoothing=0.1, margin=0.2)
    was = _native.set_ce_one_pass(one_pass)
    try:
        t = ox.from_numpy(x, True)
        loss, pair, seq = F.preference_loss(t, ids, lengths, ref, details=True, **kw)
        near([loss.item()], [w["loss"]], w["bloss"], "loss")
        near(pair.numpy(), w["pair"], w["bpair"], "pairs")
        near(seq.numpy().ravel(), w["S"], w["bS"], "sequences")
        loss.backward()
        near(t.grad.numpy(), *r.gradient(w["coef"], None, w["bcoef"]), "gradient")
        t.zero_grad()
        (F.preference_loss(t, ids, lengths, ox.from_numpy(ref), **kw) * 0.5).backward()
        near(t.grad.numpy(), *r.gradient(0.5 * w["coef"], None, 0.5 * w["bcoef"]), "another upstream")
    finally:
        _native.set_ce_one_pass(was)
    for kind in ("hinge", "ipo"):
        w = preference(r, starts, None, kind=kind, average=True)
        near([F.preference_loss(t, ids, lengths.tolist(), kind=kind, average=True).item()], [w["loss"]], w["bloss"], kind)


def test_refusals(ox, F):
    t = ox.from_numpy(np.zeros((3, 5), np.float32), True)
    for call in (lambda i: F.token_log_probs(t, i), lambda i: F.policy_loss(t, i, np.ones(3, np.float32)),
                 lambda i: F.preference_loss(t, i, [[1, 2]])):
        with pytest.raises(ValueError, match="tokens for batch of 3"):
            call([0, 1])
        with pytest.raises(IndexError, match="out of bounds"):
            call([0, 5, 1])
        with pytest.raises(TypeError, match="integers"):
            call([0.0, 1.0, 2.0])
    with pytest.raises(ValueError, match="temperature"):
        F.token_log_probs(t, [0, 1, 2], temperature=0.0)
    with pytest.raises(ValueError, match="shape mismatch"):
        F.policy_loss(t, [0, 1, 2], np.ones(2, np.float32))
    with pytest.raises(ValueError, match="shape mismatch"):
        F.policy_loss(t, [0, 1, 2], np.ones(3, np.float32), weights=np.ones((3, 1), np.float32))
    with pytest.raises(ValueError, match="needs the reference"):
        F.policy_loss(t, [0, 1, 2], np.ones(3, np.float32), kl=0.1)
    with pytest.raises(ValueError, match="clip"):
        F.policy_loss(t, [0, 1, 2], np.ones(3, np.float32), clip=-0.1)
    for lengths in ([1, 2], [[1, 2, 3]]):
        with pytest.raises(ValueError, match=r"\(pairs, 2\)"):
            F.preference_loss(t, [0, 1, 2], lengths)
    for lengths in ([[2, 2]], [[-1, 2]], [[1 << 62, 1 << 62]]):
        with pytest.raises(ValueError, match="a sequence of"):
            F.preference_loss(t, [0, 1, 2], lengths)
    with pytest.raises(ValueError, match="kind must be"):
        F.preference_loss(t, [0, 1, 2], [[1, 2]], kind="other")
    with pytest.raises(ValueError, match="smoothing"):
        F.preference_loss(t, [0, 1, 2], [[1, 2]], smoothing=1.0)


def test_no_rows_and_no_pairs(ox, F):
    t = ox.from_numpy(np.zeros((0, 5), np.float32), True)
    assert F.token_log_probs(t, []).numpy().size == 0
    assert F.policy_loss(t, [], np.zeros(0, np.float32)).item() == 0.0
    assert F.preference_loss(t, [], []).item() == 0.0
    t = ox.from_numpy(np.zeros((2, 5), np.float32), True)
    F.preference_loss(t, [0, 1], []).backward()
    assert (t.grad.numpy() == 0).all()


# ---- gradient clipping -----------------------------------------------------------------

def test_clip_grad_norm_over_many_tensors(ox):
    import oxitorch_amd.optim as op

    r = rng(21)
    shapes = [(3, 5), (1,), (64, 33), (7,), (200, 100), (2, 3, 4)] * 30
    params, grads = [], []
    for s in shapes:
        p = ox.nn.Parameter(ox.from_numpy(np.zeros(s, np.float32), True))
        g = r.standard_normal(s).astype(np.float32)
        p.tensor.grad = ox.from_numpy(g)
        params.append(p)
        grads.append(g)
    flat = np.concatenate([g.ravel() for g in grads]).astype(np.float64)
    for p_norm, want in ((2.0, np.sqrt((flat * flat).sum())), (2, np.sqrt((flat * flat).sum())), (1.0, np.abs(flat).sum()),
                         (float("inf"), np.abs(flat).max())):
        held = [p.grad for p in params]
        total = op.clip_grad_norm_(params, 0.75, norm_type=p_norm)
        assert isinstance(total, float) and abs(total - want) <= flat.size * 2.0 ** -52 * want
        f = 0.75 / (want + 1e-6)
        for p, g, h in zip(params, grads, held):
            w = g.astype(np.float64) * f
            assert (np.abs(p.grad.numpy() - w) <= 2.01 * U * np.abs(w) + 2.0 ** -149).all()
            assert np.array_equal(h.numpy(), g)  # what was held of the gradients stays
            p.tensor.grad = ox.from_numpy(g)
    before = [p.grad for p in params]
    assert op.clip_grad_norm_(params, 1e9) > 1
    for p, b, g in zip(params, before, grads):
        assert np.array_equal(p.grad.numpy(), g)


def test_clip_grad_norm_of_views_and_none(ox):
    """Permuted and broadcast gradients; parameters without one; no gradients at all."""
    import oxitorch_amd.optim as op

    x = rng(23).standard_normal((6, 10)).astype(np.float32)
    a, b, c = (ox.from_numpy(np.ones((10, 6), np.float32), True) for _ in range(3))
    a.grad = ox.from_numpy(x).transpose()
    b.grad = ox.from_numpy(x[:1, :6].copy()).broadcast_to([10, 6])
    want = np.sqrt((x.astype(np.float64) ** 2).sum() + 10 * (x[0, :6].astype(np.float64) ** 2).sum())
    assert op.clip_grad_norm_([a, b, c], 0.5) == pytest.approx(want, rel=1e-12)
    f = 0.5 / (want + 1e-6)
    assert np.allclose(a.grad.numpy(), x.T * f, rtol=3e-7) and np.allclose(b.grad.numpy(), x[:1, :6] * f, rtol=3e-7)
    assert b.grad.shape == [10, 6] and c.grad is None
    for p in (1.0, 2.0, 3.0, float("inf")):
        assert op.clip_grad_norm_([c], 1.0, norm_type=p) == 0.0


# ---- together ----------------------------------------------------------------------------

def test_a_preference_and_a_policy_step(ox, F):
    """A tiny model (embedding, residual norm, tied to nothing) as policy and as frozen reference: scores under no_grad,
    the two losses, their gradients through the model against differences, clipping, the optimizer's step."""
    import oxitorch_amd.optim as op

    r = rng(25)
    V, T = 40, 12
    table = (0.5 * r.standard_normal((V, V))).astype(np.float32)
    prompt = r.integers(0, V, T).astype(np.int64)
    tokens = r.integers(0, V, T).astype(np.int64)
    tokens[[0, 6]] = -1
    lengths = [[4, 2], [3, 3]]
    adv = r.standard_normal(T).astype(np.float32)

    def logits(w):
        h = F.embedding(prompt, w)
        y, _ = F.add_rms_norm(h, h, ox.from_numpy(np.ones(V, np.float32)), vjp="exact")
        return y

    def losses(w, old, ref):
        z = logits(w)
        return (F.policy_loss(z, tokens, adv, old, ref, kl=0.1, entropy=0.02, clip=10.0)
                + F.preference_loss(z, tokens, lengths, ref, beta=0.3))

    with ox.no_grad():
        ref = F.token_log_probs(logits(ox.from_numpy(table + 0.1 * r.standard_normal((V, V)).astype(np.float32))), tokens)
        old = F.token_log_probs(logits(ox.from_numpy(table)), tokens)
    w = ox.nn.Parameter(ox.from_numpy(table, True))
    losses(w.tensor, old, ref).backward()
    g = w.grad.numpy()

    def value(tab):
        h = 2 * tab[prompt].astype(np.float64)
        z = h / np.sqrt((h * h).mean(1, keepdims=True) + 1e-6)
        lq = z - z.max(1, keepdims=True)
        lq -= np.log(np.exp(lq).sum(1, keepdims=True))
        on = tokens >= 0
        lp = np.where(on, lq[np.arange(T), np.maximum(tokens, 0)], 0.0)
        H = -(np.exp(lq) * lq).sum(1)
        d = ref.numpy().astype(np.float64) - lp
        row = -np.exp(lp - old.numpy()) * adv + 0.1 * (np.expm1(d) - d) - 0.02 * H
        rel = np.where(on, lp - ref.numpy(), 0.0)
        s = [rel[0:4].sum(), rel[4:6].sum(), rel[6:9].sum(), rel[9:12].sum()]
        pref = np.mean([np.logaddexp(0, -0.3 * (s[0] - s[1])), np.logaddexp(0, -0.3 * (s[2] - s[3]))])
        return (row * on).sum() / on.sum() + pref

    for i in range(6):
        d = r.standard_normal((V, V))
        e = 1e-5
        num = (value(table + e * d) - value(table - e * d)) / (2 * e)
        assert abs(num - (g * d).sum()) <= 2e-5 * (1 + abs(num))
    norm = np.sqrt((g.astype(np.float64) ** 2).sum())
    opt = op.Sgd([w], lr=0.5)
    assert op.clip_grad_norm_([w], 0.1) == pytest.approx(norm, rel=1e-9)
    opt.step()
    step = -0.5 * g.astype(np.float64) * min(1.0, 0.1 / (norm + 1e-6))
    assert np.abs(w.tensor.numpy() - (table + step)).max() <= 4 * U * np.abs(table).max()


# ---- capture -----------------------------------------------------------------------------

@pytest.mark.parametrize("n,c", [(24, 1000), (10, 70001)])
def test_capture_and_replay(hip, n, c):
    """A step of the C-ABI calls in one graph: scores, policy loss, preference loss, another upstream's gradient, the
    joint norm and the clipping; replayed on new inputs between eager calls."""
    from test_gpu_graph import CAPTURE_MODE_RELAXED, _runtime

    rt = _runtime()
    D = hip.DeviceArray.from_numpy

    def inputs(seed):
        x = logits_of(n, c, seed)
        ids = chosen(x, seed + 1, 0.2)
        q = rng(seed + 2)
        return [x, ids, q.standard_normal(n).astype(np.float32), (Rows(x, ids).logp - 0.1).astype(np.float32)]

    buf = [D(a) for a in inputs(31)]
    starts = D(np.array([0, n // 4, n // 2, n // 2 + 1, n - 2], np.int64))
    up = D(np.array([0.5], np.float32))
    new = lambda *s, dtype=np.float32: hip.DeviceArray(s, dtype)  # noqa: E731
    o = {"logp": new(n), "H": new(n), "saved": new(n, 4), "dx": new(n, c), "out": new(4), "rows": new(4, n), "coef": new(2, n),
         "psaved": new(n, 4), "pdx": new(n, c), "loss": new(1), "pair": new(2), "seq": new(4), "qcoef": new(n),
         "qsaved": new(n, 4), "qdx": new(n, c), "total": new(1, dtype=np.float64), "clip": new(n, c)}
    ws = [new(max(16, b), dtype=np.uint8) for b in (hip.token_logp_workspace(n, c), hip.policy_loss_workspace(n, c),
                                                    hip.preference_loss_workspace(n, c), hip.grad_norm_workspace([o["dx"], o["pdx"]]))]
    s = hip.slice_array(hip.GradSlice, [(o["dx"].ptr, o["clip"].ptr, n * c), (o["pdx"].ptr, o["pdx"].ptr, n * c)])

    def step():
        x, ids, adv, old = (b.ptr for b in buf)
        p = {k: v.ptr for k, v in o.items()}
        hip.call("oxi_token_logp_fwd", x, ids, p["logp"], p["H"], p["saved"], ws[0].ptr, n, c, 1.0)
        hip.call("oxi_token_logp_bwd", x, ids, p["saved"], adv, old, up.ptr, p["dx"], n, c, 1.0)
        hip.call("oxi_policy_loss_fwd", x, ids, adv, old, old, None, p["out"], p["rows"], None, p["coef"], p["psaved"],
                 p["pdx"], ws[1].ptr, n, c, 1.0, 0.05, 0.05, 0.0, 0.1, 0.01, float(n))
        hip.call("oxi_preference_loss_fwd", x, ids, starts.ptr, old, p["loss"], p["pair"], p["seq"], p["qcoef"], p["qsaved"],
                 p["qdx"], ws[2].ptr, n, c, 2, 0, 0, 0.1, 0.0, 0.0)
        hip.call("oxi_grad_norm", s, 2, 2.0, p["total"], ws[3].ptr)
        hip.call("oxi_grad_clip", s, 2, p["total"], 0.01)

    def results():
        return {k: v.numpy() for k, v in o.items()}

    stream = ctypes.c_void_p()
    hip.call("oxi_hip_stream", ctypes.byref(stream))
    step()
    hip.sync()
    graph = ctypes.c_void_p()
    assert rt.hipStreamBeginCapture(stream, CAPTURE_MODE_RELAXED) == 0
    try:
        step()
    finally:
        rc = rt.hipStreamEndCapture(stream, ctypes.byref(graph))  # the stream never stays capturing
    assert rc == 0
    ex = ctypes.c_void_p()
    assert rt.hipGraphInstantiate(ctypes.byref(ex), graph, None, None, 0) == 0
    for seed in (31, 41, 51, 31):
        for b, a in zip(buf, inputs(seed)):
            hip.call("oxi_hip_memcpy_h2d", b.ptr, a.ctypes.data, a.nbytes)
        step()
        want = results()
        for k in ("logp", "dx", "pdx", "qdx", "out", "loss", "total", "clip"):
            hip.call("oxi_fill", o[k].ptr, o[k].nbytes // 4, 9.0)
        assert rt.hipGraphLaunch(ex, stream) == 0
        hip.sync()
        got = results()
        for k in want:
            assert np.array_equal(got[k], want[k], equal_nan=True), (seed, k)
    rt.hipGraphExecDestroy(ex)
    rt.hipGraphDestroy(graph)
