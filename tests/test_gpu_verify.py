"""Verification of drafted tokens (oxi_verify_drafts) against the definition in
float64: whole numbers, equal. Random cases where a running sum comes within
1e-12 of the number drawn (another order of the sum may round to the other side)
are left out of the comparison; there are none among these seeds."""

import math

import numpy as np
import pytest

from conftest import rng

pytestmark = pytest.mark.gpu


def oracle(target, draft, tokens, u, lengths=None):
    b, rows, v = target.shape
    k = rows - 1
    accepted, out = np.zeros(b, np.int64), np.full((b, rows), -1, np.int64)
    margin = np.full(b, np.inf)
    for s in range(b):
        n = k if lengths is None else int(lengths[s])
        kept = 0
        while kept < n:
            x = int(tokens[s, kept])
            if not 0 <= x < v:
                break
            q = 1.0 if draft is None else float(draft[s, kept, x])
            if not float(u[s, kept]) * q < float(target[s, kept, x]):
                break
            kept += 1
        own = np.where(target[s, kept] > 0, target[s, kept], 0).astype(np.float64)
        w = own
        if kept < n:
            if draft is None:
                left = own.copy()
                if 0 <= tokens[s, kept] < v:
                    left[tokens[s, kept]] = 0
            else:
                with np.errstate(invalid="ignore"):
                    d = target[s, kept].astype(np.float64) - draft[s, kept].astype(np.float64)
                left = np.where(d > 0, d, 0.0)
            if left.sum() > 0:
                w = left
        run = np.cumsum(w)
        accepted[s] = kept
        out[s, :kept] = tokens[s, :kept]
        if run[-1] > 0:
            limit = float(u[s, k]) * run[-1]
            over = np.flatnonzero(run > limit)
            out[s, kept] = over[0] if len(over) else np.flatnonzero(w > 0)[-1]
            if limit > 0:  # against 0 nothing rounds
                margin[s] = np.abs(run - limit).min() / run[-1]
    return accepted, out, margin


def softmax(z):
    e = np.exp(z - z.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


def make(b, k, v, seed, scale=3.0, noise=0.7):
    r = rng(seed)
    z = scale * r.standard_normal((b, k + 1, v))
    target = softmax(z)
    zd = z[:, :k] + noise * r.standard_normal((b, k, v))
    draft = softmax(zd)
    tokens = np.argmax(zd + r.gumbel(size=zd.shape), -1).astype(np.int64)
    u = r.random((b, k + 1), dtype=np.float32)
    return target, draft, tokens, u


def run(hip, target, draft, tokens, u, lengths=None, **kw):
    D = hip.DeviceArray.from_numpy
    a, o = hip.verify_drafts(D(target), D(draft) if draft is not None else None, D(tokens), D(u),
                             D(lengths) if lengths is not None else None, **kw)
    return a.numpy(), o.numpy()


def check(hip, target, draft, tokens, u, lengths=None):
    a, o = run(hip, target, draft, tokens, u, lengths)
    wa, wo, margin = oracle(target, draft, tokens, u, lengths)
    sure = margin > 1e-12
    assert sure.all()
    assert np.array_equal(a, wa)
    assert np.array_equal(o, wo), (o[(o != wo).any(1)][:4], wo[(o != wo).any(1)][:4])
    return wa, wo


@pytest.mark.parametrize("b,k,v", [(1, 1, 1), (2, 3, 2), (5, 4, 7), (3, 1, 255), (4, 4, 1000), (7, 5, 1003), (64, 3, 4099),
                                   (3, 7, 8192), (2, 4, 16385), (4, 4, 32000), (2, 2, 50257), (1, 3, 131072), (1, 1, 262144),
                                   (200, 2, 515), (2, 70, 64)])
@pytest.mark.parametrize("greedy", [False, True])
def test_against_the_definition(hip, b, k, v, greedy):
    print("[case] verify", b, k, v, greedy, flush=True)
    for seed in range(3):
        target, draft, tokens, u = make(b, k, v, 10 * seed + b + k)
        if greedy:
            draft, tokens = None, target[:, :k].argmax(-1).astype(np.int64)
        check(hip, target, draft, tokens, u)
        lengths = rng(seed).integers(0, k + 1, b).astype(np.int64)
        check(hip, target, draft, tokens, u, lengths)


def test_drafts_kept_and_not(hip):
    """The same distribution on both sides keeps every draft; a token that the target rules out is never kept."""
    target, _, tokens, u = make(6, 4, 1003, 3)
    a, o = check(hip, target, np.ascontiguousarray(target[:, :4]), tokens, u)
    assert (a == 4).all() and np.array_equal(o[:, :4], tokens)
    none = target.copy()
    np.put_along_axis(none[:, :4], tokens[:, :, None], 0, 2)
    a, o = check(hip, none, np.ascontiguousarray(target[:, :4]), tokens, np.zeros_like(u))
    assert (a == 0).all() and (o[:, 1:] == -1).all()


@pytest.mark.parametrize("v", [5, 1000, 32000, 131072])
def test_ends_of_the_drawn_number(hip, v):
    """0 draws the first token with weight, the largest float below 1 the last one; one-hot rows draw theirs."""
    target, draft, tokens, u = make(3, 2, v, v)
    target[:, :, 0] = 0
    target[:, :, v - 1] = 0
    for x in (0.0, 1 - 2.0 ** -24):
        u[:, 2] = x
        check(hip, target, draft, tokens, u)
    hot = np.zeros_like(target)
    where = rng(1).integers(0, v, (3, 3))
    np.put_along_axis(hot, where[:, :, None], 1, 2)
    for x in (0.0, 0.5, 1 - 2.0 ** -24):
        u[:] = x
        a, o = run(hip, hot, None, where[:, :2].astype(np.int64), u)
        assert (a == 2).all() and np.array_equal(o, where)


def test_no_drafts(hip):
    """Lengths of 0 and a draft count of 0 draw from the target's first row."""
    target, draft, tokens, u = make(5, 3, 700, 9)
    a, o = check(hip, target, draft, tokens, u, np.zeros(5, np.int64))
    assert (a == 0).all() and (o[:, 1:] == -1).all()
    one, u1 = np.ascontiguousarray(target[:, :1]), np.ascontiguousarray(u[:, 3:])
    a, o1 = run(hip, one, None, np.zeros((5, 0), np.int64), u1)
    assert (a == 0).all() and np.array_equal(o1[:, 0], o[:, 0])


@pytest.mark.parametrize("v", [40, 5000, 131072])
def test_rows_without_weight(hip, v):
    """Nothing left after the draft falls back to the target's row; a row of zeros gives -1; NaN and negative weights
    count nothing."""
    target, draft, tokens, u = make(6, 2, v, v)
    draft[0] = 2.0  # more than the target everywhere
    u[0, :2] = 0.999
    target[1] = 0
    target[2, :, ::3] = np.nan
    draft[2, :, ::5] = np.nan
    tokens[2] = 1
    target[3] = -target[3]
    target[4, :, 1:] = 0
    target[4, :, 0] = 1
    a, o = run(hip, target, draft, tokens, u)
    wa, wo, margin = oracle(target, draft, tokens, u)
    assert np.array_equal(a, wa) and np.array_equal(o, wo)
    assert a[0] == 0 and o[0, 0] >= 0
    assert (a[[1, 3]] == 0).all() and (o[[1, 3]] == -1).all()


def test_tokens_and_lengths_out_of_range_are_reported(hip):
    target, draft, tokens, u = make(4, 3, 300, 2)
    for bad in (-1, 300, 1 << 40):
        t = tokens.copy()
        t[1, 0] = bad
        for d in (draft, None):
            a, o = run(hip, target, d, t, u)
            with pytest.raises(RuntimeError):
                hip.sync()
            wa, wo, _ = oracle(target, d, t, u)
            assert np.array_equal(a, wa) and np.array_equal(o, wo) and a[1] == 0
    for bad, means in ((-2, 0), (9, 3)):
        lengths = np.array([2, bad, 1, 3], np.int64)
        a, o = run(hip, target, draft, tokens, u, lengths)
        with pytest.raises(RuntimeError):
            hip.sync()
        lengths[1] = means
        wa, wo, _ = oracle(target, draft, tokens, u, lengths)
        assert np.array_equal(a, wa) and np.array_equal(o, wo)
    hip.sync()


def test_a_kept_sample_is_the_targets(hip):
    """Over every drawn number the first token is distributed as the target's row: drafts of each token in the
    proportions of the draft, 4096 numbers each, counted."""
    v, n = 6, 4096
    r = rng(4)
    p, q = softmax(r.standard_normal(v)), softmax(r.standard_normal(v))
    target = np.broadcast_to(p, (n * v, 2, v)).astype(np.float32)
    draft = np.broadcast_to(q, (n * v, 1, v)).astype(np.float32)
    tokens = np.repeat(np.arange(v), n).astype(np.int64)[:, None]
    grid = (np.arange(n) + 0.5) / n
    u = np.stack([np.tile(grid, v), np.tile(r.permutation(grid), v)], 1).astype(np.float32)
    _, o = run(hip, np.ascontiguousarray(target), np.ascontiguousarray(draft), tokens, u)
    share = np.zeros(v)
    for x in range(v):
        share += q[x] * np.bincount(o[x * n:(x + 1) * n, 0], minlength=v) / n
    # a stratified first number and a shuffled second: within 4 standard deviations of a proportion over n
    assert (np.abs(share - p) <= 4 * np.sqrt(p * (1 - p) / n)).all()


def test_unaligned_buffers(hip):
    for shift in (1, 2, 3):
        target, draft, tokens, u = make(3, 2, 4100, shift)
        D = hip.DeviceArray.from_numpy
        t = D(np.concatenate([np.zeros(shift, np.float32), target.ravel()]))
        d = D(np.concatenate([np.zeros(shift, np.float32), draft.ravel()]))
        dt, du = D(tokens), D(u)
        a, o = hip.DeviceArray((3,), np.int64), hip.DeviceArray((3, 3), np.int64)
        hip.call("oxi_verify_drafts", t.ptr + 4 * shift, d.ptr + 4 * shift, dt.ptr, None, du.ptr, a.ptr, o.ptr, None, 3, 2,
                 4100)
        wa, wo, margin = oracle(target, draft, tokens, u)
        assert (margin > 1e-12).all() and np.array_equal(a.numpy(), wa) and np.array_equal(o.numpy(), wo)


def test_caller_workspace(hip):
    for b, v in ((1, 300), (3, 40000), (70, 131072), (300, 1003)):
        target, draft, tokens, u = make(b, 1, v, b, scale=1.0)
        n = hip.verify_drafts_workspace(b, v)
        assert n % 8 == 0
        ws = hip.DeviceArray.from_numpy(np.full(n // 8 + 32, 5, np.int64))
        a, o = run(hip, target, draft, tokens, u, workspace=ws)
        a2, o2 = run(hip, target, draft, tokens, u)
        assert np.array_equal(a, a2) and np.array_equal(o, o2)
        assert (ws.numpy()[n // 8:] == 5).all()


@pytest.mark.parametrize("v", [30, 512, 600, 5000, 32000, 131072, 400000])
def test_a_number_where_two_threads_sums_meet(hip, v):
    """Rows of two halves with the same weights in another order, u = 1/2: the limit is where one half's sum ends and
    the other's begins, which differ by their roundings. A sum of v terms here passes fewer than 256 roundings a
    term, so that the token's own stretch [before, before + w) is within 2^8 * 2^-53 of the total."""
    b = 64 if v < 200000 else 2
    r = rng(v)
    half = np.exp(6 * r.standard_normal((b, v // 2))).astype(np.float32)
    row = np.concatenate([half, r.permuted(half, axis=1)], 1)[:, None]
    u = np.full((b, 1), 0.5, np.float32)
    a, o = run(hip, row, None, np.zeros((b, 0), np.int64), u)
    for s in range(b):
        w = row[s, 0].astype(np.float64).tolist()
        total, x = math.fsum(w), int(o[s, 0])
        assert math.fsum(w[:x]) <= total * (0.5 + 2.0 ** -45), (s, x)
        assert math.fsum(w[:x + 1]) >= total * (0.5 - 2.0 ** -45), (s, x)
