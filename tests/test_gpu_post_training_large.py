"""The post-training losses and gradient clipping on many rows, long ones, and buffers
past 2^31 elements: a few rows of chosen values among rows of equal logits, checked
against float64 with the bounds of token_oracle.py.

A row of equal logits is exact in float32: its exponentials are 1 and their sum is the
number of classes, so its logp is -log(c), its entropy log(c), up to 2^-52 and the last
rounding.
"""

import types

import numpy as np
import pytest

from conftest import rng
from test_gpu_operator_large import put, take
from token_oracle import Rows, U, near, policy, preference

pytestmark = pytest.mark.gpu

# (rows, classes): the first rows of a second pass from the cache's on (past 208 MB), each way a row is laid over
# threads, and offsets past 2^31
SHAPES = [(2300, 32000), (20001, 4099), (300000, 300), (4000001, 9), (600, 20003), (1500, 50257), (600, 131075),
          (66000, 32768), (33000, 65537), (11000, 200001), (5000, 524289)]


class Many:
    """n rows of equal logits but for a few, whose values are known."""

    def __init__(self, hip, n, c, seed):
        self.n, self.c = n, c
        cold = n - (208 << 20) // (4 * c)  # around there the first pass changes its loads
        at = {0, 1, 2, 7, 8, n // 2, n - 9, n - 2, n - 1, *(cold + i for i in (-1, 0, 1))}
        self.at = np.array(sorted(i for i in at if 0 <= i < n))
        r = rng(seed)
        self.x = (2 * r.standard_normal((len(self.at), c))).astype(np.float32)
        self.x[::2, c // 3] += 20
        picks = np.where(np.arange(len(self.at)) % 4 < 2, self.x.argmax(1), r.integers(0, c, len(self.at)))
        picks[3] = -1
        self.ids = np.full(n, c - 1, np.int64)
        self.ids[5::11] = -1  # padding among the others
        self.ids[self.at] = picks
        self.small = Rows(self.x, picks.astype(np.int64))
        A = hip.DeviceArray
        self.X = A((n * c,))
        hip.call("oxi_fill", self.X.ptr, n * c, 0.25)
        for i, row in zip(self.at, self.x):
            put(hip, self.X.ptr + int(i) * c * 4, row)
        self.I = hip.DeviceArray.from_numpy(self.ids)
        # all rows' values and errors
        on = self.ids >= 0
        full = lambda plain, few: self._with(np.where(on, plain, 0.0), few)  # noqa: E731
        self.rows = types.SimpleNamespace(
            on=on, logp=full(-np.log(c), self.small.logp), d_logp=full(1e-13, self.small.d_logp),
            entropy=full(np.log(c), self.small.entropy), d_entropy=full(1e-13, self.small.d_entropy))

    def _with(self, all_rows, few):
        a = np.array(all_rows, np.float64)
        a[self.at] = few
        return a

    def check_gradient(self, hip, D, gl, gh, dgl, dgh, what):
        """The chosen rows' gradients, and, of one row of equal logits before each, its value."""
        n, c, at = self.n, self.c, self.at
        got = np.stack([take(hip, D.ptr + int(i) * c * 4, (c,)) for i in at])
        near(got, *self.small.gradient(gl[at], None if gh is None else gh[at], dgl[at], dgh[at]), what)
        for i in at:
            j = int(i) + 1
            if j < n and j not in at:
                d = take(hip, D.ptr + j * c * 4, (c,)).astype(np.float64)
                want = np.full(c, -gl[j] / c if self.ids[j] >= 0 else 0.0)
                if self.ids[j] >= 0:
                    want[self.ids[j]] = gl[j] * (1 - 1 / c)
                assert (np.abs(d - want) <= 12 * U * np.abs(want) + dgl[j]).all(), (what, j)


@pytest.mark.parametrize("n,c", SHAPES)
def test_rows(hip, n, c):
    print("[case] many rows", n, c, flush=True)
    m = Many(hip, n, c, c)
    A, r = hip.DeviceArray, m.rows
    near_rows = lambda v, want, d, what: near(v, want, d + 2 * U * np.abs(want), what)  # noqa: E731
    q = rng(1)
    adv = q.standard_normal(n).astype(np.float32)
    lp, H, saved, d = A((n,)), A((n,)), A((n, 4)), A((n * c,))
    for keep in (saved, None):  # with a backward to come and without
        hip.call("oxi_token_logp_fwd", m.X.ptr, m.I.ptr, lp.ptr, H.ptr, keep and keep.ptr, None, n, c, 1.0)
        near_rows(lp.numpy(), r.logp, r.d_logp, "logp")
        near_rows(H.numpy(), r.entropy, r.d_entropy, "entropy")
    G = hip.DeviceArray.from_numpy(adv)
    hip.call("oxi_token_logp_bwd", m.X.ptr, m.I.ptr, saved.ptr, G.ptr, None, None, d.ptr, n, c, 1.0)
    zero = np.zeros(n)
    m.check_gradient(hip, d, adv.astype(np.float64), None, zero, zero, "backward")
    hip.call("oxi_token_logp_bwd", m.X.ptr, m.I.ptr, saved.ptr, G.ptr, G.ptr, None, d.ptr, n, c, 1.0)
    m.small_gradient = m.small.gradient(adv[m.at], adv[m.at])
    near(np.stack([take(hip, d.ptr + int(i) * c * 4, (c,)) for i in m.at]), *m.small_gradient, "backward with entropies")

    old = (r.logp - 0.1).astype(np.float32)
    w = policy(r, adv, old, old, kl=0.1, ent=0.01, divisor=100.0)
    out, rows, coef, ps = A((4,)), A((4, n)), A((2, n)), A((n, 4))
    O = hip.DeviceArray.from_numpy(old)
    hip.call("oxi_policy_loss_fwd", m.X.ptr, m.I.ptr, G.ptr, O.ptr, O.ptr, None, out.ptr, rows.ptr, lp.ptr, coef.ptr,
             ps.ptr, d.ptr, None, n, c, 1.0, 0.2, 0.2, 0.0, 0.1, 0.01, 100.0)
    near(rows.numpy(), w["rows"], w["brows"], "policy rows")
    near(out.numpy(), w["out"], w["bout"], "policy out")
    near(coef.numpy(), np.stack([w["cl"], w["ch"]]), np.stack([w["bcl"], w["bch"]]), "policy coefficients")
    at = m.at
    near(np.stack([take(hip, d.ptr + int(i) * c * 4, (c,)) for i in at]),
         *m.small.gradient(w["cl"][at], w["ch"][at], w["bcl"][at], w["bch"][at]), "policy gradient")

    starts = np.array([1, n // 4, n // 2, n // 2, n - 2], np.int64)
    r.on = (m.ids >= 0) & (np.arange(n) >= 1) & (np.arange(n) < n - 2)
    w = preference(r, starts, kind="ipo", average=True, beta=0.5)
    S = hip.DeviceArray.from_numpy(starts)
    loss, pair, seq = A((1,)), A((2,)), A((4,))
    hip.call("oxi_preference_loss_fwd", m.X.ptr, m.I.ptr, S.ptr, None, loss.ptr, pair.ptr, seq.ptr, lp.ptr, ps.ptr, d.ptr,
             None, n, c, 2, 2, 1, 0.5, 0.0, 0.0)
    near(seq.numpy(), w["S"], w["bS"], "sequences")
    near(pair.numpy(), w["pair"], w["bpair"], "pairs")
    near(lp.numpy(), w["coef"], w["bcoef"], "preference coefficients")
    m.small.on = r.on[at]
    m.ids = np.where(r.on, m.ids, -1)
    m.check_gradient(hip, d, w["coef"], None, w["bcoef"], zero, "preference gradient")


def test_gradients_past_2_31_elements(hip):
    n = (1 << 31) + 12345
    print("[case] large gradients", n, flush=True)
    A = hip.DeviceArray
    g, o = A((n,)), A((n,))
    hip.call("oxi_fill", g.ptr, n, 2.0 ** -10)
    tail = rng(3).standard_normal(1000).astype(np.float32)
    put(hip, g.ptr + (n - 1000) * 4, tail)
    small = [hip.DeviceArray.from_numpy(np.full(3, 1.0, np.float32)) for _ in range(150)]
    rows = [(v.ptr, v.ptr, 3) for v in small[:75]] + [(g.ptr, o.ptr, n)] + [(v.ptr, v.ptr, 3) for v in small[75:]]
    s = hip.slice_array(hip.GradSlice, rows)
    total = A((1,), np.float64)
    hip.call("oxi_grad_norm", s, len(rows), 2.0, total.ptr, None)
    want = np.sqrt((n - 1000) * 2.0 ** -20 + (tail.astype(np.float64) ** 2).sum() + 450)
    assert abs(total.numpy()[0] - want) <= n * 2.0 ** -53 * want
    hip.call("oxi_grad_clip", s, len(rows), total.ptr, 1.0)
    f = 1.0 / (want + 1e-6)
    got = take(hip, o.ptr + (n - 1000) * 4, (1000,))
    assert (np.abs(got - tail * f) <= 2.01 * U * np.abs(tail * f)).all()
    for k in (0, 1 << 30, n - 1001 - 4096):
        assert (np.abs(take(hip, o.ptr + k * 4, (4096,)) - 2.0 ** -10 * f) <= 2.01 * U * f).all()
    for v in small:
        assert (np.abs(v.numpy() - f) <= 2.01 * U * f).all()
