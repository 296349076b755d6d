"""Float64 values of the post-training losses with the errors that their float32
parts may have.

u = 2^-24. An exponential of (x - m)/T is off, relatively, by a u for each of the
difference, the factor log2(e)/T and the product, times the argument's size, and by
at most 2 steps (4 u) of its own; a row's sum adds at most c/64 + 24 terms in
sequence in float32 on any path. What is formed of the sums is in float64. `rows`
propagates these through the formulas, per row.
"""

import numpy as np

U = 2.0 ** -24
TINY = 2.0 ** -126  # results below the smallest normal number may be 0


class Rows:
    """logp, entropy and their bounds for x (n, c), ids (n) at temperature T; 0 in rows that do not count."""

    def __init__(self, x, ids, T=1.0, counted=None):
        self.T = T = float(np.float32(T))
        n, c = x.shape
        self.x, self.ids = x, ids
        self.on = (ids >= 0) & (ids < c) if counted is None else counted
        at = np.where(self.on, ids, 0)
        with np.errstate(all="ignore"):
            z = x.astype(np.float64) / T
            self.m = z.max(1, keepdims=True)
            self.d = d = z - self.m
            e = np.exp(d)
            s = e.sum(1, keepdims=True)
            self.q = e / s
            pick = lambda a: np.take_along_axis(a, at[:, None], 1)[:, 0]  # noqa: E731
            # the sum over the others is formed by itself: 1 - q[a] keeps its digits
            others = e.copy()
            np.put_along_axis(others, at[:, None], 0.0, 1)
            rest = others.sum(1)
            self.rest = rest / s[:, 0]
            top = pick(d) == 0
            logp = np.where(top, -np.log1p(rest), pick(d) - np.log(s[:, 0]))
            self.size = size = np.minimum(np.where(e > 0, -d, 0.0), 200.0)  # |z| where it matters
            mean = (self.q * size).sum(1)  # -sum q (z - m)
            H = np.where(top, np.log1p(rest), np.log(s[:, 0])) + mean
            # ln q + H, in which ln s cancels: formed without it, it keeps its digits where q is near 1
            self.lnq_H = np.where(e > 0, d, -200.0) + mean[:, None]
            eps = U * (3 * size + 6)
            self.seq = (c / 64 + 24) * U
            own = np.where(top, 0.0, pick(self.q) * pick(eps))
            off = (others / s * eps).sum(1)  # of the others' exponentials
            self.dsum = off + own + self.rest * (self.seq + 2 * U)  # of the row's sum, relatively
            dmean = (self.q * size * (eps + 6 * U)).sum(1) + self.seq * mean + mean * self.dsum
            b_logp = self.dsum + 2 * U * np.abs(logp) + 1e-14 + TINY
            b_H = self.dsum + dmean + 2 * U * np.abs(H) + 1e-14 + TINY
        self.eps, self.b_off, self.off = eps, dmean + 2 * U * mean, mean
        self.rest_rel = np.where(self.rest > 0, off / np.maximum(self.rest, 1e-300), 0) + self.seq + 2 * U
        zero = np.zeros(n)
        self.logp, self.entropy = np.where(self.on, logp, zero), np.where(self.on, H, zero)
        # 64 bits inside, rounded at the end: what is formed of logp goes by d_logp
        self.d_logp = np.where(self.on, self.dsum + 1e-14, zero)
        self.b_logp, self.b_entropy = np.where(self.on, b_logp, zero), np.where(self.on, b_H, zero)
        self.d_entropy = np.where(self.on, self.dsum + dmean + 1e-14, zero)

    def gradient(self, gl, gh=None, dgl=0.0, dgh=0.0):
        """dx and its bound for gradients gl of logp and gh of the entropy, themselves off by dgl and dgh."""
        n, c = self.x.shape
        gl = np.where(self.on, gl, 0.0).astype(np.float64)
        dgl = np.where(self.on, dgl, 0.0)
        gh_ = np.zeros(n) if gh is None else np.where(self.on, gh, 0.0).astype(np.float64)
        dgh = np.where(self.on, dgh, 0.0)
        a, b = gl[:, None] / self.T, gh_[:, None] / self.T
        lnq = self.lnq_H
        with np.errstate(all="ignore"):
            dx = -a * self.q - b * self.q * lnq
            rel = self.eps + self.dsum[:, None] + 10 * U
            wide = self.size + self.off[:, None] + np.abs(lnq)
            bound = self.q * (np.abs(a) * rel + dgl[:, None] / self.T
                              + np.abs(b) * (wide * (rel + 6 * U) + self.b_off[:, None] + 4 * U * self.size)
                              + dgh[:, None] / self.T * np.abs(lnq))
            at = np.where(self.on, self.ids, 0)[:, None]
            own = a[:, 0] * self.rest - np.take_along_axis(b * self.q * lnq, at, 1)[:, 0]
            b_own = (np.abs(a[:, 0]) * self.rest * (self.rest_rel + self.dsum + 10 * U) + dgl / self.T * self.rest
                     + np.take_along_axis(bound, at, 1)[:, 0] * (gh is not None))
            np.put_along_axis(dx, at, own[:, None], 1)
            np.put_along_axis(bound, at, b_own[:, None], 1)
            bound += 2 * U * np.abs(dx) + TINY * (1 + np.abs(a) + 220 * np.abs(b))
        dx[~self.on] = 0.0
        bound[~self.on] = 0.0
        # a row whose gradients are 0 gets zeros
        none = (gl == 0) & (gh_ == 0)
        dx[none], bound[none] = 0.0, 0.0
        return dx, bound


def near(got, want, bound, what):
    """got within bound of want, elementwise; infinities and NaN in the same places."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, f"{what}: {got.shape} for {want.shape}"
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        bad = ~same & ~(np.abs(got - want) <= bound)
    if bad.any():
        w = np.broadcast_to(bound, got.shape)
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} outside; first {np.argwhere(bad)[0]}: got {got[bad][0]!r} "
                             f"for {want[bad][0]!r}, bound {w[bad][0]!r}")


def policy(r, adv, old=None, ref=None, weights=None, clip=(0.2, 0.2), clip_max=0.0, kl=0.0, ent=0.0, divisor=1.0):
    """The policy loss over Rows r: out, rows (4, n), their bounds, and the coefficients with theirs."""
    f = lambda v: float(np.float32(v))  # noqa: E731
    lo, hi, cm, kl, ent, div = 1 - f(clip[0]), 1 + f(clip[1]), f(clip_max), f(kl), f(ent), f(divisor)
    A = adv.astype(np.float64)
    with np.errstate(all="ignore"):
        ratio = np.ones_like(A) if old is None else np.exp(r.logp - old.astype(np.float64))
        dr = np.zeros_like(A) if old is None else ratio * 1.01 * r.d_logp + 1e-13 * ratio
        free = np.where(A == 0, 0.0, ratio * A)
        bounded = np.clip(ratio, lo, hi) * A
        clipped = free > bounded
        s = np.minimum(free, np.where(A == 0, 0.0, bounded))
        floor = np.where((A < 0) & (cm > 0), cm * A, -np.inf)
        clipped |= s < floor
        s = np.maximum(s, floor)
        g = np.where(clipped, 0.0, -free)
        dg = np.where(clipped, 0.0, np.abs(A) * dr)
        bs = dg.copy()
        k, bk = np.zeros_like(A), np.zeros_like(A)
        if ref is not None:
            d = ref.astype(np.float64) - r.logp
            k = np.expm1(d) - d
            bk = np.abs(np.expm1(d)) * r.d_logp * 1.01 + np.exp(d) * r.d_logp ** 2 + 1e-15 * np.exp(np.abs(d))
        loss, bl = -s, bs
        if kl:
            loss, bl = loss + kl * k, bl + abs(kl) * bk
            g, dg = g - kl * np.expm1(d), dg + abs(kl) * np.exp(d) * (r.d_logp * 1.01 + 1e-14)
        if ent:
            loss, bl = loss - ent * r.entropy, bl + abs(ent) * r.d_entropy
    w = (np.ones_like(A) if weights is None else weights.astype(np.float64)) / div
    on = r.on
    zero = lambda v: np.where(on, v, 0.0)  # noqa: E731
    rows = np.stack([zero(loss), zero(k), zero(r.entropy), zero(clipped.astype(np.float64))])
    brows = np.stack([zero(bl), zero(bk), zero(r.d_entropy), zero(0.0 * A)]) + 2 * U * np.abs(rows)
    w = zero(w)
    out = (rows * w).sum(1)
    bout = (brows * np.abs(w)).sum(1) + 2 * U * np.abs(out)
    cl, ch = zero(g * w), zero(-ent * w)
    bcl = zero(dg * np.abs(w)) + 2 * U * np.abs(cl)
    return dict(out=out, bout=bout, rows=rows, brows=brows, cl=cl, bcl=bcl, ch=ch, bch=2 * U * np.abs(ch))


def preference(r, starts, ref=None, kind="sigmoid", average=False, beta=0.1, margin=0.0, smoothing=0.0):
    """The preference loss over Rows r (whose `on` holds the counted rows), and its coefficients, with bounds."""
    f = lambda v: float(np.float32(v))  # noqa: E731
    beta, margin, eps = f(beta), f(margin), f(smoothing)
    pairs = (len(starts) - 1) // 2
    n = len(r.logp)
    coef, bcoef = np.zeros(n), np.zeros(n)
    losses, blosses = np.zeros(pairs), np.zeros(pairs)
    S, bS = np.zeros(2 * pairs), np.zeros(2 * pairs)
    for p in range(pairs):
        D, dD, cnt = [], 0.0, []
        for side in range(2):
            q = 2 * p + side
            rows = np.arange(starts[q], starts[q + 1])
            rows = rows[r.on[rows]]
            k = max(1, len(rows)) if average else 1
            S[q] = r.logp[rows].sum() / k
            d = r.d_logp[rows].sum() / k + 1e-13
            bS[q] = d + 2 * U * abs(S[q])
            D.append(S[q] - (ref[rows].astype(np.float64).sum() / k if ref is not None else 0.0))
            dD += d
            cnt.append((rows, k))
        h = D[0] - D[1]
        u, du = beta * h - margin, beta * dD + 1e-14
        with np.errstate(over="ignore"):
            if kind == "sigmoid":
                up, down = 1 / (1 + np.exp(-u)), 1 / (1 + np.exp(u))
                losses[p] = (1 - eps) * np.logaddexp(0, -u) + eps * np.logaddexp(0, u)
                slope, dl, ds = beta * (eps * up - (1 - eps) * down), du, beta * up * down * du * 1.05
            elif kind == "hinge":
                losses[p], slope = max(0.0, 1 - u), -beta if u < 1 else 0.0
                dl, ds = (du if u < 1 else 0.0), 0.0
            else:
                e = (u - 0.5) / beta
                losses[p], slope = e * e, 2 * e
                dl, ds = 2 * abs(e) * du / beta + (du / beta) ** 2, 2 * du / beta
        blosses[p] = dl * 1.01 + 2 * U * losses[p] + 1e-15
        for side, (rows, k) in enumerate(cnt):
            coef[rows] = (-slope if side else slope) / (pairs * k)
            bcoef[rows] = ds / (pairs * k) + 2 * U * abs(coef[rows])
    loss = losses.mean() if pairs else 0.0
    return dict(loss=loss, bloss=(blosses.mean() if pairs else 0.0) + 2 * U * abs(loss), pair=losses, bpair=blosses,
                S=S, bS=bS, coef=coef, bcoef=bcoef)
