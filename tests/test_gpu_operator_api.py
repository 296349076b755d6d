"""The residual RMS norm, rotary positions, distillation and draft verification
through the Python surface: values and gradients of the graph nodes, views, the
modules, a run of them together, and graph capture of their C-ABI calls.

Gradients of small cases are compared with complex-step derivatives of the same
formula in numpy (exact to float64). Tolerances, u = 2^-24: the kernels' own are
derived in the tests of each; here sums of a few dozen terms of size up to about
8 pass through at most some 40 roundings, 8 * 40 u = 2e-5 absolute.
"""

import ctypes

import numpy as np
import pytest

from conftest import rng

pytestmark = pytest.mark.gpu

TOL = 8 * 40 * 2.0 ** -24


@pytest.fixture(scope="module")
def ox(hip):
    import oxitorch_amd

    return oxitorch_amd


@pytest.fixture(scope="module")
def F(ox):
    return ox.nn.functional


def near(got, want, tol=TOL, what=""):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert (np.abs(got - want) <= tol * (1 + np.abs(want))).all(), f"{what}: {np.abs(got - want).max():.3g}"


def steps(f, args, i, picks):
    """d f / d args[i] at the flat places `picks`, by a complex step."""
    out = []
    for p in picks:
        a = [np.asarray(v, np.complex128) for v in args]
        a[i] = a[i].copy()
        a[i].reshape(-1)[p] += 1e-30j
        out.append(f(*a).imag / 1e-30)
    return np.array(out)


def norm(h, w, eps=1e-6):
    return h / np.sqrt((h * h).mean(-1, keepdims=True) + eps) * w


# ---- residual norm -----------------------------------------------------------------

@pytest.mark.parametrize("use_h", [True, False])
@pytest.mark.parametrize("shape", [(3, 5), (2, 3, 64), (7, 1003)])
def test_add_rms_norm(ox, F, shape, use_h):
    r = rng(len(shape))
    x, res, gy, gh = (r.standard_normal(shape).astype(np.float32) for _ in range(4))
    w = (1 + 0.1 * r.standard_normal(shape[-1])).astype(np.float32)
    tx, tr, tw = (ox.from_numpy(a, True) for a in (x, res, w))
    y, h = F.add_rms_norm(tx, tr, tw, vjp="exact")
    assert np.array_equal(h.numpy(), x + res)
    near(y.numpy(), norm((x + res).astype(np.float64), w.astype(np.float64)))
    loss = (y * ox.from_numpy(gy)).sum()
    if use_h:
        loss = loss + (h * ox.from_numpy(gh)).sum()
    loss.backward()

    def f(x, res, w):
        v = x + res
        return (norm(v, w) * gy).sum() + ((v * gh).sum() if use_h else 0)

    picks = r.integers(0, x.size, 12)
    want = steps(f, (x, res, w), 0, picks)
    near(tx.grad.numpy().reshape(-1)[picks], want, what="dx")
    assert np.array_equal(tx.grad.numpy(), tr.grad.numpy())
    wp = r.integers(0, w.size, 8)
    near(tw.grad.numpy()[wp], steps(f, (x, res, w), 2, wp), what="dw")


@pytest.mark.parametrize("mode", ["ref", "exact"])
def test_residual_stream_with_and_without_the_joined_pass(ox, F, mode):
    """Three layers along one stream: the pass that adds the stream's gradient gives the node-by-node gradients."""
    r = rng(3)
    x0, ws = r.standard_normal((6, 260)).astype(np.float32), (1 + 0.1 * r.standard_normal((3, 260))).astype(np.float32)
    got = []
    from oxitorch_amd import _native
    for fuse in (True, False):
        old = _native.set_fuse_norm_act(fuse)
        try:
            x = ox.from_numpy(x0, True)
            w = [ox.from_numpy(a, True) for a in ws]
            h, out = x, x
            for i in range(3):
                out, h = F.add_rms_norm(F.silu(out), h, w[i], vjp=mode)
            ((out * out).sum() + (h * 0.5).sum()).backward()
            got.append([x.grad.numpy()] + [v.grad.numpy() for v in w])
        finally:
            _native.set_fuse_norm_act(old)
    for a, b in zip(*got):
        near(a, b, 4 * TOL)


def test_a_graph_kept_and_run_again(ox, F):
    x = rng(1).standard_normal((4, 64)).astype(np.float32)
    t, w = ox.from_numpy(x, True), ox.from_numpy(np.ones(64, np.float32), True)
    y, h = F.add_rms_norm(t, t, w)
    loss = (y * y).sum() + (h * h).sum()
    loss.backward(retain_graph=True)
    first = t.grad.numpy()
    t.zero_grad()
    loss.backward()
    assert np.array_equal(t.grad.numpy(), first)
    with pytest.raises(ValueError):
        loss.backward()


def test_add_rms_norm_of_other_shapes(ox, F):
    """A residual that broadcasts goes through the separate nodes; views are taken as they are."""
    r = rng(5)
    x, res = r.standard_normal((3, 4, 32)).astype(np.float32), r.standard_normal((1, 4, 32)).astype(np.float32)
    w = ox.from_numpy(np.ones(32, np.float32), True)
    y, h = F.add_rms_norm(ox.from_numpy(x), ox.from_numpy(res), w)
    near(y.numpy(), norm((x + res).astype(np.float64), 1.0))
    assert h.shape == [3, 4, 32]
    xt = ox.from_numpy(x, True)
    v = xt.permute([1, 0, 2])
    y, h = F.add_rms_norm(v, v, w, vjp="exact")
    near(y.numpy(), norm(2 * x.transpose(1, 0, 2).astype(np.float64), 1.0))
    (y.sum() + h.sum()).backward()
    assert xt.grad.shape == [3, 4, 32]


@pytest.mark.parametrize("host", range(3))
def test_a_host_operand_among_the_norms_is_refused(ox, F, host):
    a = [ox.from_numpy(np.ones(s, np.float32), device="cpu" if i == host else "hip")
         for i, s in enumerate([(3, 8), (3, 8), (8,)])]
    with pytest.raises(NotImplementedError, match="add_rms_norm"):
        F.add_rms_norm(*a)
    with pytest.raises(NotImplementedError, match="add_rms_norm_e4m3"):
        F.add_rms_norm_e4m3(*a)


def test_e4m3(ox, F):
    r = rng(7)
    x, res = (r.standard_normal((2, 5, 300)).astype(np.float32) for _ in range(2))
    w = ox.from_numpy((1 + 0.1 * r.standard_normal(300)).astype(np.float32))
    y, h = F.add_rms_norm(ox.from_numpy(x), ox.from_numpy(res), w)
    q, h8 = F.add_rms_norm_e4m3(ox.from_numpy(x), ox.from_numpy(res), w, group=128)
    assert np.array_equal(h8.numpy(), h.numpy()) and q.shape == [2, 5, 300] and q.scale.shape == [2, 5, 3]
    back, yv = q.dequantize().numpy(), y.numpy()
    s = np.repeat(q.scale.numpy(), 128, axis=-1)[..., :300]
    # half a step of e4m3, and float32's of the norm
    assert (np.abs(back - yv) <= np.maximum(2.0 ** -4 * np.abs(yv), 2.0 ** -10 * s) * (1 + 1e-5) + 1e-6 * np.abs(yv)).all()
    assert q.codes().dtype == np.uint8 and q.codes().shape == (2, 5, 300) and q.group == 128
    q1, none = F.add_rms_norm_e4m3(ox.from_numpy(x), None, w, group=300)
    assert none is None and q1.scale.shape == [2, 5, 1]


# ---- rotary ---------------------------------------------------------------------------

def turn(x, pos, inv, layout, scale):
    """x (B, T, H, D), pos (B, T)."""
    a = (pos[..., None] * inv)[:, :, None, :]
    c, s, n = np.cos(a) * scale, np.sin(a) * scale, len(inv)
    y = x.copy()
    i0, i1 = (slice(0, n), slice(n, 2 * n)) if layout == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    y[..., i0], y[..., i1] = x[..., i0] * c - x[..., i1] * s, x[..., i1] * c + x[..., i0] * s
    return y


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_values_views_and_gradients(ox, F, layout):
    r = rng(11)
    B, T, H, D = 2, 5, 3, 24
    freq = F.rotary_frequencies(16, scaling={"type": "yarn", "factor": 4.0, "original_length": 64})
    x = r.standard_normal((B, T, H, D)).astype(np.float32)
    g = r.standard_normal((B, T, H, D)).astype(np.float32)
    pos = r.integers(0, 5000, (B, T))
    want = turn(x.astype(np.float64), pos, freq[0], layout, freq[1])
    back = turn(g.astype(np.float64), pos, -freq[0], layout, freq[1])
    tx = ox.from_numpy(x, True)
    y = F.rotary_embedding(tx, freq, pos, layout=layout)
    near(y.numpy(), want)
    y.backward(ox.from_numpy(g))
    near(tx.grad.numpy(), back)
    # heads before tokens in memory
    tv = ox.from_numpy(np.ascontiguousarray(x.transpose(0, 2, 1, 3)), True)
    yv = F.rotary_embedding(tv.permute([0, 2, 1, 3]), freq, pos, layout=layout)
    near(yv.numpy(), want)
    yv.backward(ox.from_numpy(g))
    near(tv.grad.numpy(), back.transpose(0, 2, 1, 3))
    # three dims, positions shared or counted from an offset
    one = F.rotary_embedding(ox.from_numpy(x[0]), freq, pos[0], layout=layout)
    near(one.numpy(), want[0])
    off = F.rotary_embedding(ox.from_numpy(x), freq, offset=70, layout=layout)
    near(off.numpy(), turn(x.astype(np.float64), np.broadcast_to(70 + np.arange(T), (B, T)), freq[0], layout, freq[1]))
    shared = F.rotary_embedding(ox.from_numpy(x), freq, pos[1], layout=layout)
    near(shared.numpy(), turn(x.astype(np.float64), np.broadcast_to(pos[1], (B, T)), freq[0], layout, freq[1]))


def test_rotary_module_and_refusals(ox, F):
    from oxitorch_amd import nn

    m = nn.RotaryEmbedding(8, layout="interleaved")
    assert m.parameters() == [] and m.frequencies.pairs == 4
    x = rng(2).standard_normal((1, 3, 2, 8)).astype(np.float32)
    inv, _ = F.rotary_frequencies(8)
    want = turn(x.astype(np.float64), np.arange(3)[None], inv, "interleaved", 1.0)
    near(m(ox.from_numpy(x)).numpy(), want)
    # one token at a time, as decoding does, gives the rows of the whole
    for t in range(3):
        near(m(ox.from_numpy(x[:, t:t + 1]), offset=t).numpy(), want[:, t:t + 1])
    t = ox.from_numpy(x)
    with pytest.raises(ValueError, match="do not fit"):
        F.rotary_embedding(t, F.rotary_frequencies(10))
    with pytest.raises(ValueError, match="positions for"):
        F.rotary_embedding(t, inv, [1, 2])
    with pytest.raises(TypeError, match="integers"):
        F.rotary_embedding(t, inv, [0.5, 1, 2])
    with pytest.raises(ValueError, match="layout"):
        F.rotary_embedding(t, inv, layout="other")
    with pytest.raises(ValueError, match="expects"):
        F.rotary_embedding(ox.from_numpy(x[0, 0]), inv)


# ---- distillation -----------------------------------------------------------------------

def distill(x, ids, top, T, lse=None):
    z = x / T
    m = z.real.max(1, keepdims=True)
    lq = z - m - np.log(np.exp(z - m).sum(1, keepdims=True))
    total, rows = 0, 0
    for r in range(x.shape[0]):
        keep = [j for j in range(ids.shape[1]) if ids[r, j] >= 0]
        if not keep:
            continue
        rows += 1
        t = top[r, keep].astype(np.float64) / T
        lp = t - np.log(np.exp(t).sum()) if lse is None else t - float(lse[r])
        p = np.exp(lp)
        total = total + (p * (lp - lq[r, ids[r, keep]])).sum()
        if lse is not None:
            left = 1 - p.sum()
            out = np.delete(np.exp(lq[r]), ids[r, keep]).sum()
            total = total + left * (np.log(left) - np.log(out))
    return T * T * total / max(rows, 1)


@pytest.mark.parametrize("with_lse", [False, True])
def test_distillation_loss(ox, F, with_lse):
    r = rng(13)
    n, c, k, T = 5, 40, 6, 2.0
    teacher = (2 * r.standard_normal((n, c))).astype(np.float32)
    x = (teacher + r.standard_normal((n, c))).astype(np.float32)
    ids = np.argsort(-teacher, 1)[:, :k]
    ids[1, 4:] = -1
    ids[3] = -1
    top = np.take_along_axis(teacher, np.maximum(ids, 0), 1)
    lse = np.log(np.exp(teacher.astype(np.float64) / T).sum(1)).astype(np.float32) if with_lse else None
    want = distill(x.astype(np.float64), ids, top, T, lse)
    picks = np.concatenate([r.integers(0, n * c, 24), [c * 3, ids[0, 0], c + ids[1, 0]]])
    grad = steps(lambda v: distill(v, ids, top, T, lse), (x,), 0, picks)
    t = ox.from_numpy(x, True)
    loss = F.distillation_loss(t, ids, top, T, lse)
    near(loss.item(), want)
    loss.backward()
    near(t.grad.numpy().reshape(-1)[picks], grad)
    assert (t.grad.numpy()[3] == 0).all()
    # another upstream gradient, a tensor for the teacher's logits, and a second backward
    t2 = ox.from_numpy(x, True)
    l2 = F.distillation_loss(t2, ids.tolist(), ox.from_numpy(top), T, lse) * -3.0
    l2.backward(retain_graph=True)
    near(t2.grad.numpy().reshape(-1)[picks], -3 * grad)
    t2.zero_grad()
    l2.backward()
    near(t2.grad.numpy().reshape(-1)[picks], -3 * grad)
    # next to the targets' loss, as it is trained
    t3 = ox.from_numpy(x, True)
    hard = np.argmax(teacher, 1)
    (F.distillation_loss(t3, ids, top, T, lse) * 0.5 + F.cross_entropy(t3, hard) * 0.5).backward()
    t4 = ox.from_numpy(x, True)
    F.cross_entropy(t4, hard).backward()
    near(t3.grad.numpy(), 0.5 * (t2.grad.numpy() / -3 + t4.grad.numpy()))
    with ox.no_grad():
        near(F.distillation_loss(ox.from_numpy(x), ids, top, T, lse).item(), want)


def test_distillation_refusals(ox, F):
    x = ox.from_numpy(np.zeros((3, 8), np.float32), True)
    ids, top = np.zeros((3, 2), np.int64), np.zeros((3, 2), np.float32)
    with pytest.raises(ValueError, match="teacher_ids"):
        F.distillation_loss(x, ids[:2], top)
    with pytest.raises(ValueError, match="teacher_logits"):
        F.distillation_loss(x, ids, top[:, :1])
    with pytest.raises(IndexError, match="out of bounds"):
        F.distillation_loss(x, ids + 8, top)
    with pytest.raises(TypeError, match="integers"):
        F.distillation_loss(x, ids + 0.5, top)
    with pytest.raises(ValueError, match="temperature"):
        F.distillation_loss(x, ids, top, 0.0)
    with pytest.raises(ValueError):
        F.distillation_loss(x, ids, top, 1.0, np.zeros(2, np.float32))
    # a batch of padding alone
    loss = F.distillation_loss(x, ids - 1, top)
    loss.backward()
    assert loss.item() == 0 and (x.grad.numpy() == 0).all()


# ---- verification ------------------------------------------------------------------------

def test_verify_drafts(ox, F):
    from test_gpu_verify import make, oracle

    target, draft, tokens, u = make(6, 3, 50, 17)
    T = ox.from_numpy
    a, o = F.verify_drafts(tokens, T(draft), T(target), u)
    wa, wo, _ = oracle(target, draft, tokens, u)
    assert a.dtype == o.dtype == np.int64 and np.array_equal(a, wa) and np.array_equal(o, wo)
    lengths = [0, 1, 2, 3, 3, 0]
    a, o = F.verify_drafts(tokens.tolist(), T(draft), T(target), T(u), lengths)
    wa, wo, _ = oracle(target, draft, tokens, u, lengths)
    assert np.array_equal(a, wa) and np.array_equal(o, wo)
    # through the softmax and a view, drafts without probabilities
    logits = np.log(np.maximum(target, 1e-30)).astype(np.float32)
    p = F.softmax(T(np.ascontiguousarray(logits.transpose(1, 0, 2))).permute([1, 0, 2]), -1)
    a, o = F.verify_drafts(tokens, None, p, u)
    wa, wo, margin = oracle(p.numpy(), None, tokens, u)
    assert (margin > 1e-12).all() and np.array_equal(a, wa) and np.array_equal(o, wo)
    with pytest.raises(ValueError, match="draft_tokens"):
        F.verify_drafts(tokens[:, :2], T(draft), T(target), u)
    with pytest.raises(RuntimeError, match="out of bounds"):
        F.verify_drafts(tokens + 50, T(draft), T(target), u)
    with pytest.raises(ValueError, match="length"):
        F.verify_drafts(tokens, T(draft), T(target), u, [4, 0, 0, 0, 0, 0])
    with pytest.raises(ValueError, match="shape mismatch"):
        F.verify_drafts(tokens, T(draft[:, :2].copy()), T(target), u)
    with pytest.raises(ValueError, match="shape mismatch"):
        F.verify_drafts(tokens, T(draft), T(target), u[:, :3].copy())


# ---- together ------------------------------------------------------------------------------

def test_a_drafting_model_trained_and_verified(ox, F):
    """Two layers of (residual norm, rotary, silu gate) over an embedding, distilled from a teacher's top logits: the
    gradients of every parameter against complex steps; then its probabilities draft, and are verified."""
    from oxitorch_amd import nn, optim

    r = rng(21)
    V, D, H, L, k, T = 24, 24, 2, 6, 5, 1.5
    ids = r.integers(0, V, L)
    W = (0.5 * r.standard_normal((V, D))).astype(np.float32)
    ws = (1 + 0.1 * r.standard_normal((3, D))).astype(np.float32)
    gates = (1 + 0.3 * r.standard_normal((2, D))).astype(np.float32)
    inv, _ = F.rotary_frequencies(8)
    teacher = (2 * r.standard_normal((L, V))).astype(np.float32)
    tids = np.argsort(-teacher, 1)[:, :k]
    top = np.take_along_axis(teacher, tids, 1)
    lse = np.log(np.exp(teacher.astype(np.float64) / T).sum(1)).astype(np.float32)
    pos = np.arange(L)

    def logits64(W, ws, gates):
        h = W[ids]
        out = np.zeros_like(h)
        for i in range(2):
            h = h + out
            y = norm(h, ws[i])
            q = turn(y.reshape(1, L, H, D // H), pos[None], inv, "half", 1.0).reshape(L, D)
            out = q / (1 + np.exp(-q)) * gates[i]
        return norm(h + out, ws[2])

    def loss64(W, ws, gates):
        return distill(logits64(W, ws, gates), tids, top, T, lse)

    tW = ox.from_numpy(W, True)
    tws, tgs = [ox.from_numpy(a, True) for a in ws], [ox.from_numpy(a, True) for a in gates]
    rot = nn.RotaryEmbedding(8)

    def forward():
        h = F.embedding(ids, tW)
        out = h * 0.0
        for i in range(2):
            y, h = F.add_rms_norm(out, h, tws[i], vjp="exact")
            q = rot(y.reshape([L, H, D // H])).reshape([L, D])
            out = F.silu(q) * tgs[i]
        return F.add_rms_norm(out, h, tws[2], vjp="exact")[0]

    params = [tW, *tws, *tgs]
    logits = forward()
    near(logits.numpy(), logits64(*(a.astype(np.float64) for a in (W, ws, gates))))
    loss = F.distillation_loss(logits, tids, top, T, lse)
    near(loss.item(), loss64(*(a.astype(np.float64) for a in (W, ws, gates))))
    loss.backward()
    got = [tW.grad.numpy(), np.stack([t.grad.numpy() for t in tws]), np.stack([t.grad.numpy() for t in tgs])]
    for i, name in enumerate(("W", "ws", "gates")):
        picks = r.integers(0, got[i].size, 20)
        near(got[i].reshape(-1)[picks], steps(loss64, (W, ws, gates), i, picks), what=name)
    opt = optim.Sgd(params, lr=0.1)
    opt.step()

    with ox.no_grad():
        p = F.softmax(forward(), -1)  # (L, V): drafts of the last three positions
        q = p.numpy()[None, L - 3:].copy()
        tokens = q.argmax(2).astype(np.int64)
        target = F.softmax(ox.from_numpy(np.concatenate([teacher[None, L - 3:], teacher[None, :1]], 1)), -1)
        u = r.random((1, 4), dtype=np.float32)
        from test_gpu_verify import oracle

        a, o = F.verify_drafts(tokens, ox.from_numpy(q), target, u)
        wa, wo, margin = oracle(target.numpy(), q, tokens, u)
        assert (margin > 1e-12).all() and np.array_equal(a, wa) and np.array_equal(o, wo)


# ---- capture ----------------------------------------------------------------------------------

def test_captured_and_replayed(hip):
    """The calls in two graphs on the library stream, each with its own workspaces, replayed in turn on new inputs
    with eager calls between: every replay has the eager bits."""
    from test_gpu_graph import CAPTURE_MODE_RELAXED, _runtime

    rt = _runtime()
    A, D = hip.DeviceArray, hip.DeviceArray.from_numpy
    stream = ctypes.c_void_p()
    hip.check(hip.lib.oxi_hip_stream(ctypes.byref(stream)))
    R, H, n, c, k = 700, 260, 9, 5000, 7
    freq = D(10000.0 ** (-np.arange(16, dtype=np.float64) / 16))
    pos = D(np.arange(R, dtype=np.int64))
    w = D((1 + 0.1 * rng(0).standard_normal(H)).astype(np.float32))

    def buffers():
        b = {m: A((R, H)) for m in ("x", "r", "gy", "gh", "h", "y", "dx", "turned", "hq")}
        b.update(rstd=A((R,)), dw=A((H,)), q=A((R, H), np.uint8), scale=A((R, 3)), logits=A((n, c)), d=A((n, c)),
                 d2=A((n, c)), ids=A((n, k), np.int64), top=A((n, k)), loss=A((1,)), row=A((n,)), lse=A((n,)), rest=A((n,)),
                 g=A((1,)), target=A((n, 2, c)), draft=A((n, 1, c)), tok=A((n, 1), np.int64), u=A((n, 2)),
                 acc=A((n,), np.int64), out=A((n, 2), np.int64))
        b["ws"] = A((hip.add_rms_norm_bwd_workspace(R, H) // 4 + 1,))
        b["vs"] = A((hip.verify_drafts_workspace(n, c) // 8 + 1,), np.int64)
        return b

    st = hip._i64arr(hip.row_major_strides((1, R, 5, 52)))
    shape, ps = hip._i64arr((1, R, 5, 52)), hip._i64arr((0, 1))

    def step(b, eager):
        p = {m: v.ptr for m, v in b.items()}
        hip.call("oxi_add_rms_norm_fwd", p["x"], p["r"], w.ptr, p["h"], p["y"], p["rstd"], R, H, 1e-6)
        hip.call("oxi_rotary", p["y"], st, p["turned"], st, shape, pos.ptr, ps, 3, freq.ptr, 32, 0, 0, 1.0)
        hip.call("oxi_add_rms_norm_bwd", p["h"], w.ptr, p["rstd"], p["gy"], p["gh"], p["dx"], p["dw"],
                 None if eager else p["ws"], R, H, 1)
        hip.call("oxi_add_rms_norm_e4m3_fwd", p["x"], p["r"], w.ptr, p["hq"], p["q"], p["scale"], R, H, 128, 1e-6)
        hip.call("oxi_distill_fwd", p["logits"], p["ids"], p["top"], None, p["loss"], p["row"], p["lse"], p["rest"],
                 p["d"], n, c, k, 2.0, float(n))
        hip.call("oxi_distill_bwd", p["logits"], p["ids"], p["top"], None, p["lse"], p["rest"], p["g"], p["d2"], n, c, k,
                 2.0, float(n))
        hip.call("oxi_verify_drafts", p["target"], p["draft"], p["tok"], None, p["u"], p["acc"], p["out"],
                 None if eager else p["vs"], n, 1, c)

    outs = ("h", "y", "rstd", "turned", "dx", "dw", "q", "scale", "loss", "row", "d", "d2", "acc", "out")

    def fill(b, seed):
        r = rng(seed)
        z = 2 * r.standard_normal((n, 2, c))
        soft = lambda v: (np.exp(v) / np.exp(v).sum(-1, keepdims=True)).astype(np.float32)  # noqa: E731
        logits = (2 * r.standard_normal((n, c))).astype(np.float32)
        ids = np.argsort(-logits, 1)[:, :k].astype(np.int64)
        for m, v in {**{m: r.standard_normal((R, H)).astype(np.float32) for m in ("x", "r", "gy", "gh")},
                     "logits": (logits + r.standard_normal((n, c))).astype(np.float32), "ids": ids,
                     "top": np.take_along_axis(logits, ids, 1), "g": np.array([1.5], np.float32), "target": soft(z),
                     "draft": soft(z[:, :1] + 0.5), "tok": z[:, :1].argmax(2).astype(np.int64),
                     "u": r.random((n, 2), dtype=np.float32)}.items():
            v = np.ascontiguousarray(v)
            hip.check(hip.lib.oxi_hip_memcpy_h2d(b[m].ptr, v.ctypes.data, v.nbytes))

    sets, exes, graphs = [buffers(), buffers()], [], []
    for b in sets:
        fill(b, 1)
        step(b, False)
    hip.sync()
    try:
        for b in sets:
            graph, exe = ctypes.c_void_p(), ctypes.c_void_p()
            assert rt.hipStreamBeginCapture(stream, CAPTURE_MODE_RELAXED) == 0
            try:
                step(b, False)
            finally:
                rc = rt.hipStreamEndCapture(stream, ctypes.byref(graph))  # the stream never stays capturing
            assert rc == 0 and graph.value
            graphs.append(graph)
            assert rt.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0) == 0
            exes.append(exe)
        eager = buffers()
        for i in range(4):
            print("[case] replay", i, flush=True)
            for j, b in enumerate(sets):
                fill(b, 100 + 10 * i + j)
            for e in exes:  # one after the other, nothing between
                assert rt.hipGraphLaunch(e, stream) == 0
            hip.sync()
            for j, b in enumerate(sets):
                fill(eager, 100 + 10 * i + j)
                step(eager, True)
                hip.sync()
                for m in outs:
                    assert np.array_equal(b[m].numpy(), eager[m].numpy(), equal_nan=m not in ("q", "acc", "out")), (i, j, m)
    finally:
        for e in exes:
            rt.hipGraphExecDestroy(e)
        for g in graphs:
            rt.hipGraphDestroy(g)
