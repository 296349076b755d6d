"""Log-probabilities and the losses on them with the tightest bounds that the kernels' orders of
summation allow, and with the rounding of the exponents' factor.

token_oracle.py counts the additions of a row's sum as if they grew with the row. They do not: a
thread adds at most 16 float4s and a class more (65), a block's threads are joined in a tree of at
most 10 levels, parts and pieces of a row in 64 bits, each by a factor of one more exponential
(its argument's part of the error is in that of the whole argument; 4 u of its own and one
rounding). With u = 2^-24 a sum is off by (min(c, 65) + 10 + 5) u of itself beside what its
exponentials are.
"""

import numpy as np
import pytest

from conftest import rng
from test_gpu_token_logp import chosen, logits_of
from token_oracle import TINY, U, Rows, near, policy, preference

pytestmark = pytest.mark.gpu


def tight(x, ids, T=1.0, counted=None):
    r = Rows(x, ids, T, counted)
    seq = (min(x.shape[1], 65) + 15) * U
    mean = r.off  # -sum q (z - m)
    less = r.seq - seq
    assert less >= 0  # a bound above the oracle's would be no tighter
    r.dsum = r.dsum - r.rest * less
    dmean = (r.q * r.size * (r.eps + 6 * U)).sum(1) + seq * mean + mean * r.dsum
    r.b_off = dmean + 2 * U * mean
    r.rest_rel = r.rest_rel - less
    r.seq = seq
    on = lambda v: np.where(r.on, v, 0.0)  # noqa: E731
    r.d_logp, r.d_entropy = on(r.dsum + 1e-14), on(r.dsum + dmean + 1e-14)
    r.b_logp = on(r.d_logp + 2 * U * np.abs(r.logp) + TINY)
    r.b_entropy = on(r.d_entropy + 2 * U * np.abs(r.entropy) + TINY)
    return r


WIDTHS = [4099, 8195, 12289, 16384, 16411, 20000, 32000, 32768, 32801, 50257, 65571, 131072, 200003, 530001]


@pytest.mark.parametrize("spread", [0.02, 3.0])
@pytest.mark.parametrize("c", WIDTHS)
def test_sums(hip, c, spread):
    """Rows of nearly equal logits, where a class left out or taken twice shows, and decided ones."""
    n = 4
    x = logits_of(n, c, 111, spread) if spread > 1 else (spread * rng(112).standard_normal((n, c))).astype(np.float32)
    ids = chosen(x, 113)
    r = tight(x, ids)
    if spread < 1 and c <= 131072:
        assert (r.dsum < 1 / c).all(), "a class of average mass would go unnoticed"
    D = hip.DeviceArray.from_numpy
    dx, di = D(x), D(ids)
    logp, entropy, saved = hip.token_logp_fwd(dx, di, 1.0, need_entropy=True)
    near(logp.numpy(), r.logp, r.b_logp, "logp")
    near(entropy.numpy(), r.entropy, r.b_entropy, "entropy")
    g = rng(114).standard_normal((2, n)).astype(np.float32)
    near(hip.token_logp_bwd(dx, di, saved, D(g[0])).numpy(), *r.gradient(g[0]), "gradient of logp")
    near(hip.token_logp_bwd(dx, di, saved, D(g[0]), D(g[1])).numpy(), *r.gradient(g[0], g[1]), "gradient of both")
    old = (r.logp - 0.05).astype(np.float32)
    for ent in (0.0, 0.02):
        w = policy(r, g[0], old, ent=ent, divisor=float(n))
        out, rows, lp, coef, saved, d = hip.policy_loss_fwd(dx, di, D(g[0]), D(old), entropy_coef=ent, divisor=float(n),
                                                            need_grad=True)
        near(lp.numpy(), r.logp, r.b_logp, "policy logp")
        near(rows.numpy(), w["rows"], w["brows"], "policy rows")
        near(d.numpy(), *r.gradient(w["cl"], w["ch"] if ent else None, w["bcl"], w["bch"] if ent else 0.0), "policy gradient")
    starts = np.array([0, 2, 4], np.int64)
    w = preference(r, starts, beta=0.5)
    loss, pair, S, coef, saved, d = hip.preference_loss_fwd(dx, di, D(starts), beta=0.5, need_grad=True)
    near(S.numpy(), w["S"], w["bS"], "sequences")
    near(d.numpy(), *r.gradient(w["coef"], None, w["bcoef"]), "preference gradient")


def factor_off(T):
    """By how much of itself the exponents' factor log2(e)/T, in 32 bits, is off."""
    T = np.float64(np.float32(T))
    return np.float64(np.float32(1.4426950408889634 / T)) * np.log(2.0) * T - 1.0


def test_the_factors_of_a_temperature():
    """The two temperatures below are ones whose factor is off by nearly all that a rounding can be."""
    assert factor_off(1.4393) > 5e-8 and factor_off(1.4418) < -5e-8


@pytest.mark.parametrize("T", [1.4393, 1.4418])
@pytest.mark.parametrize("c,depth", [(32000, 8.0), (131072, 9.5)])
def test_sums_over_tokens_do_not_keep_the_factors_rounding(hip, c, depth, T):
    """Log-probabilities are summed over sequences, where an error that every row has grows with their number. The
    factor's rounding is such an error: it moves ln s by factor_off times the mean of (x - m)/T. It is taken back, so the
    mean error over many rows is that of the exponentials alone, 4 u of their share, and what is left of roundings that
    differ from class to class and row to row: of the result (a half step of 2^-23 at most for values between 2 and 4, by
    the square root of 12 and of the rows for its deviation, six of those) and of arguments and sums (a tenth of that)."""
    n = 512
    T32 = np.float32(T)
    r = rng(c)
    x = np.empty((n, c), np.float32)
    x[:] = ((r.random((n, c), dtype=np.float32) - 0.5) - np.float32(depth)) * T32
    x[:, 7] = 0.0
    ids = np.full(n, 7, np.int64)
    z = x.astype(np.float64) / np.float64(T32)
    z[:, 7] = -np.inf
    e = np.exp(z)
    rest = e.sum(1)
    want = -np.log1p(rest)
    share = rest / (1 + rest)
    z[:, 7] = 0.0
    mean = (e * z).sum(1) / (1 + rest)
    assert (want > -4).all() and (want < -2).all()
    kept = factor_off(T) * mean.mean()
    bound = 4 * U * share.mean() + 6.6 * 2.0 ** -22 / np.sqrt(12 * n)
    assert abs(kept) > 1.5 * bound, "an error that was kept would go unnoticed"
    logp = hip.token_logp_fwd(hip.DeviceArray.from_numpy(x), hip.DeviceArray.from_numpy(ids), float(T32))[0].numpy()
    off = (logp.astype(np.float64) - want).mean()
    assert abs(off) <= bound, (off, bound, kept)
