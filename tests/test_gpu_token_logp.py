"""Log-probabilities of chosen tokens, their entropies and the gradient
(oxi_token_logp_*) against float64; the bounds are derived in token_oracle.py."""

import numpy as np
import pytest

from conftest import rng
from token_oracle import Rows, near

pytestmark = pytest.mark.gpu


def logits_of(n, c, seed, spread=3.0):
    """Rows of which some are all but decided."""
    r = rng(seed)
    x = (spread * r.standard_normal((n, c))).astype(np.float32)
    lift = np.where(r.random(n) < 0.5, 30 * r.random(n), 0.0).astype(np.float32)
    x[np.arange(n), r.integers(0, c, n)] += lift
    return x


def chosen(x, seed, pad=0.0):
    """The likeliest class of half of the rows, any of the others, -1 in padded ones."""
    r = rng(seed)
    n, c = x.shape
    ids = np.where(r.random(n) < 0.5, x.argmax(1), r.integers(0, c, n)).astype(np.int64)
    return np.where(r.random(n) < pad, -1 - r.integers(0, 3, n), ids)


def check(hip, x, ids, T=1.0, seed=0, what=""):
    D = hip.DeviceArray.from_numpy
    n, c = x.shape
    r = Rows(x, ids, T)
    dx, di = D(x), D(ids)
    logp, entropy, saved = hip.token_logp_fwd(dx, di, T, need_entropy=True)
    near(logp.numpy(), r.logp, r.b_logp, f"{what} logp")
    near(entropy.numpy(), r.entropy, r.b_entropy, f"{what} entropy")
    alone, none, _ = hip.token_logp_fwd(dx, di, T)
    assert none is None and np.array_equal(alone.numpy(), logp.numpy(), equal_nan=True)
    g = rng(seed + 1).standard_normal((2, n)).astype(np.float32)
    if n > 2:
        g[:, 1] = 0.0
    gl, gh = D(g[0]), D(g[1])
    for a, b, up in ((gl, None, None), (gl, gh, None), (None, gh, None), (gl, gh, -0.375)):
        f = 1.0 if up is None else up
        want, bound = r.gradient(g[0] * f if a else np.zeros(n), g[1] * f if b else None)
        got = hip.token_logp_bwd(dx, di, saved, a, b, None if up is None else D(np.array([up], np.float32)), T).numpy()
        near(got, want, bound, f"{what} gradient of {'logp ' if a else ''}{'entropy' if b else ''}")


@pytest.mark.parametrize("c", [1, 2, 3, 4, 5, 7, 8, 9, 31, 33, 64, 100, 255, 256, 257, 289, 511, 1000, 1003, 1024, 2051,
                               4096, 4099, 8191, 8192, 8225, 12289, 16411, 20000, 32000, 32768, 32801, 50257, 65536, 65571])
def test_widths(hip, c):
    for n, seed in ((1, 1), (9, 2)):
        x = logits_of(n, c, seed)
        check(hip, x, chosen(x, seed + 10, pad=0.2 if n > 1 else 0.0), what=f"{(n, c)}")


@pytest.mark.parametrize("n,c", [(3, 131072), (2, 131075), (5, 200003), (1, 400009)])
def test_long_rows(hip, n, c):
    x = logits_of(n, c, 5)
    check(hip, x, chosen(x, 6), what=f"{(n, c)}")


@pytest.mark.parametrize("n,c", [(700, 1003), (2000, 257), (300, 32000), (1100, 8195), (5000, 40), (600, 16411)])
def test_many_rows(hip, n, c):
    x = logits_of(n, c, 7)
    check(hip, x, chosen(x, 8, pad=0.3), what=f"{(n, c)}")


@pytest.mark.parametrize("T", [0.01, 0.7, 1.3, 50.0])
@pytest.mark.parametrize("c", [33, 5000, 70001])
def test_temperatures(hip, T, c):
    x = logits_of(6, c, 11)
    check(hip, x, chosen(x, 12), T, what=f"T={T} c={c}")


@pytest.mark.parametrize("c", [4, 300, 5003, 32000, 70001])
def test_every_place_of_the_chosen_class(hip, c):
    """The row's ends, the classes around a 128-byte line, and around a block's parts."""
    places = sorted({p for p in (0, 1, 2, 3, 4, 30, 31, 32, 33, 35, 8190, 8191, 8192, 8193, 8223, 8224, c - 5, c - 4,
                                 c - 3, c - 2, c - 1) if 0 <= p < c})
    x = logits_of(len(places), c, 13)
    check(hip, x, np.array(places, np.int64), what=f"c={c}")


def test_certain_tokens_keep_their_digits(hip):
    """A token of probability 1 - 1e-12: logp and the gradient at it are the others' mass, not 0."""
    for c in (5, 1003, 32000, 70001):
        x = np.zeros((4, c), np.float32)
        ids = np.array([0, c - 1, c // 2, 3 % c], np.int64)
        x[np.arange(4), ids] = [30.0, 40.0, 60.0, 85.0]
        r = Rows(x, ids)
        assert (r.logp < 0).all() and (r.rest > 0).all()
        check(hip, x, ids, what=f"c={c}")


@pytest.mark.parametrize("c", [6, 300, 5003, 32000, 70001])
@pytest.mark.parametrize("lowest", [-np.inf, np.finfo(np.float32).min])
def test_masked_classes(hip, c, lowest):
    """Masked classes have probability 0 and no gradient, whatever masks them; one class may be left."""
    x = logits_of(6, c, 17)
    ids = x.argmax(1).astype(np.int64)
    keep = rng(18).random((6, c)) < 0.3
    keep[1] = False  # the chosen class alone
    keep[2, : c // 2] = False
    keep[np.arange(6), ids] = True
    x = np.where(keep, x, np.float32(lowest))
    for T in (1.0, 0.5):
        check(hip, x, ids, T, what=f"masked with {lowest}, c={c}, T={T}")
    got = hip.token_logp_fwd(hip.DeviceArray.from_numpy(x), hip.DeviceArray.from_numpy(ids), 1.0, need_entropy=True)
    assert got[0].numpy()[1] == 0.0 and got[1].numpy()[1] == 0.0


@pytest.mark.parametrize("c", [6, 5003, 70001])
def test_chosen_class_that_is_masked(hip, c):
    x = logits_of(3, c, 19)
    ids = np.array([0, 1, c - 1], np.int64)
    x[np.arange(3), ids] = -np.inf
    logp, entropy, saved = hip.token_logp_fwd(*map(hip.DeviceArray.from_numpy, (x, ids)), 1.0, need_entropy=True)
    assert np.all(logp.numpy() == -np.inf)
    r = Rows(x, ids)
    near(entropy.numpy(), r.entropy, r.b_entropy, "entropy")
    g = np.array([1.0, -2.0, 0.5], np.float32)
    got = hip.token_logp_bwd(*map(hip.DeviceArray.from_numpy, (x, ids)), saved, hip.DeviceArray.from_numpy(g)).numpy()
    near(got, *r.gradient(g), "gradient")


@pytest.mark.parametrize("c", [1, 4, 300, 5003, 32000, 70001])
def test_rows_without_a_finite_logit(hip, c):
    """All masked, or holding NaN or +inf: NaN in that row alone."""
    x = logits_of(5, c, 21)
    x[1] = -np.inf
    x[2, c // 2] = np.nan
    x[3, c - 1] = np.inf
    ids = np.zeros(5, np.int64)
    logp, entropy, saved = hip.token_logp_fwd(*map(hip.DeviceArray.from_numpy, (x, ids)), 1.0, need_entropy=True)
    bad = np.array([False, True, True, True, False])
    assert np.array_equal(np.isnan(logp.numpy()), bad) and np.array_equal(np.isnan(entropy.numpy()), bad)
    g = hip.DeviceArray.from_numpy(np.ones(5, np.float32))
    d = hip.token_logp_bwd(*map(hip.DeviceArray.from_numpy, (x, ids)), saved, g, g).numpy()
    assert np.array_equal(np.isnan(d).any(1), bad)


@pytest.mark.parametrize("c", [5, 300, 5003, 32000, 70001])
def test_padded_rows_are_not_read(hip, c):
    """NaN in padded rows goes nowhere, their results are 0; all rows padded."""
    x = logits_of(6, c, 23)
    ids = np.array([0, -1, 2, -7, 1, -(1 << 62)], np.int64)
    x[ids < 0] = np.nan
    logp, entropy, saved = hip.token_logp_fwd(*map(hip.DeviceArray.from_numpy, (x, ids)), 1.0, need_entropy=True)
    for v in (logp, entropy):
        assert np.isfinite(v.numpy()).all() and (v.numpy()[ids < 0] == 0).all()
    g = hip.DeviceArray.from_numpy(np.ones(6, np.float32))
    d = hip.token_logp_bwd(*map(hip.DeviceArray.from_numpy, (x, ids)), saved, g, g).numpy()
    assert np.isfinite(d).all() and (d[ids < 0] == 0).all() and (d[ids >= 0] != 0).any()
    ids[:] = -1
    logp, _, saved = hip.token_logp_fwd(*map(hip.DeviceArray.from_numpy, (x, ids)))
    d = hip.token_logp_bwd(*map(hip.DeviceArray.from_numpy, (x, ids)), saved, g).numpy()
    assert (logp.numpy() == 0).all() and (d == 0).all()


def test_ids_past_the_classes_raise_the_guard(hip):
    x = hip.DeviceArray.from_numpy(logits_of(3, 50, 25))
    ids = hip.DeviceArray.from_numpy(np.array([1, 50, 1 << 40], np.int64))
    hip.sync()
    logp, _, saved = hip.token_logp_fwd(x, ids)
    with pytest.raises(RuntimeError):
        hip.sync()
    assert (logp.numpy()[1:] == 0).all()
    g = hip.DeviceArray.from_numpy(np.ones(3, np.float32))
    d = hip.token_logp_bwd(x, ids, saved, g)
    with pytest.raises(RuntimeError):
        hip.sync()
    assert (d.numpy()[1:] == 0).all()


def test_no_rows(hip):
    x, ids = hip.DeviceArray((0, 7)), hip.DeviceArray((0,), np.int64)
    logp, entropy, saved = hip.token_logp_fwd(x, ids, 1.0, need_entropy=True)
    assert logp.numpy().size == 0
    hip.call("oxi_token_logp_fwd", None, None, None, None, None, None, 0, 0, 1.0)
    hip.sync()


def test_logits_and_gradient_at_any_float(hip):
    """Views that start at any float: the logits and the gradient lie differently in their lines."""
    n, c = 5, 9001
    x = logits_of(n, c, 27)
    ids = chosen(x, 28)
    r = Rows(x, ids)
    g = rng(29).standard_normal(n).astype(np.float32)
    want, bound = r.gradient(g)
    G, I = hip.DeviceArray.from_numpy(g), hip.DeviceArray.from_numpy(ids)
    for off_x, off_d in ((1, 0), (0, 3), (2, 31), (33, 1)):
        buf = np.zeros(n * c + 40, np.float32)
        buf[off_x:off_x + n * c] = x.ravel()
        bx, bd = hip.DeviceArray.from_numpy(buf), hip.DeviceArray.from_numpy(np.full(n * c + 40, 7.0, np.float32))
        logp, saved = hip.DeviceArray((n,)), hip.DeviceArray((n, 4))
        hip.call("oxi_token_logp_fwd", bx.ptr + 4 * off_x, I.ptr, logp.ptr, None, saved.ptr, None, n, c, 1.0)
        hip.call("oxi_token_logp_bwd", bx.ptr + 4 * off_x, I.ptr, saved.ptr, G.ptr, None, None, bd.ptr + 4 * off_d, n, c, 1.0)
        near(logp.numpy(), r.logp, r.b_logp, "logp")
        d = bd.numpy()
        near(d[off_d:off_d + n * c].reshape(n, c), want, bound, f"gradient at {off_x}, {off_d}")
        assert (d[:off_d] == 7).all() and (d[off_d + n * c:] == 7).all(), "written outside"


def test_gradient_against_differences(hip):
    n, c = 4, 37
    x = logits_of(n, c, 31, spread=1.0)
    ids = np.array([0, 5, -1, 36], np.int64)
    g = rng(32).standard_normal((2, n)).astype(np.float32)
    D = hip.DeviceArray.from_numpy
    T = 0.8
    _, _, saved = hip.token_logp_fwd(D(x), D(ids), T)
    got = hip.token_logp_bwd(D(x), D(ids), saved, D(g[0]), D(g[1]), None, T).numpy()

    def value(x64):
        z = x64 / float(np.float32(T))
        lq = z - z.max(1, keepdims=True)
        lq -= np.log(np.exp(lq).sum(1, keepdims=True))
        lp = np.take_along_axis(lq, np.maximum(ids, 0)[:, None], 1)[:, 0]
        H = -(np.exp(lq) * lq).sum(1)
        return ((g[0] * lp + g[1] * H) * (ids >= 0)).sum()

    h = 1e-5
    for r in range(n):
        for j in (0, 5, 11, 36):
            up, down = x.astype(np.float64), x.astype(np.float64)
            up[r, j] += h
            down[r, j] -= h
            assert abs((value(up) - value(down)) / (2 * h) - got[r, j]) < 1e-6


def test_workspace_of_the_caller_and_determinism(hip):
    n, c = 40, 33333
    x = logits_of(n, c, 33)
    ids = chosen(x, 34)
    dx, di = hip.DeviceArray.from_numpy(x), hip.DeviceArray.from_numpy(ids)
    ws = hip.DeviceArray((max(1, hip.token_logp_workspace(n, c)),), np.uint8)
    a = hip.token_logp_fwd(dx, di, 0.9, True)
    b = hip.token_logp_fwd(dx, di, 0.9, True, workspace=ws)
    for p, q in zip(a, b):
        assert np.array_equal(p.numpy(), q.numpy())
