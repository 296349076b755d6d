"""What the token log-probability, policy, preference and gradient norm entry
points refuse, no GPU: arguments are checked before any device use."""

import numpy as np
import pytest

N = 1 << 40
P = 1 << 20  # a non-NULL address that no refused call touches
Q = 1 << 21  # another
BAD = (0.0, -1.0, float("nan"), float("inf"))


@pytest.fixture(scope="module")
def capi():
    from oxitorch_amd import capi

    return capi


def without(n, drop):
    a = [P] * n
    if drop is not None:
        a[drop] = None
    return a


@pytest.mark.parametrize("name", ["token", "policy", "preference"])
def test_sizes_and_temperatures(capi, name):
    def call(n=2, c=50, T=1.0):
        if name == "token":
            capi.call("oxi_token_logp_fwd", *[P] * 6, n, c, T)
        elif name == "policy":
            capi.call("oxi_policy_loss_fwd", *[P] * 13, n, c, T, 0.2, 0.2, 0.0, 0.0, 0.0, 1.0)
        else:
            capi.call("oxi_preference_loss_fwd", *[P] * 11, n, c, 1, 0, 0, 0.1, 0.0, 0.0)

    with pytest.raises(ValueError, match="negative size"):
        call(n=-1)
    with pytest.raises(ValueError, match="negative size"):
        call(c=-1)
    with pytest.raises(ValueError, match="kernel limits"):
        call(c=1 << 31)
    with pytest.raises(ValueError, match="kernel limits"):
        call(n=1 << 24)
    with pytest.raises(ValueError, match="zero classes"):
        call(c=0)
    if name != "preference":
        for T in BAD:
            with pytest.raises(ValueError, match="temperature"):
                call(T=T)
        with pytest.raises(ValueError, match="32-bit reciprocal"):
            call(T=1e-40)


def test_token_logp(capi):
    for i in (0, 1, 2):
        with pytest.raises(ValueError, match="NULL tensor"):
            capi.call("oxi_token_logp_fwd", *without(6, i), 2, 50, 1.0)
    with pytest.raises(ValueError, match="16-byte aligned"):
        capi.call("oxi_token_logp_fwd", *[P] * 5, P + 8, 2, 50, 1.0)
    for i in (0, 1, 2, 6):
        with pytest.raises(ValueError, match="NULL tensor"):
            capi.call("oxi_token_logp_bwd", *without(7, i), 2, 50, 1.0)
    with pytest.raises(ValueError, match="NULL tensor"):
        capi.call("oxi_token_logp_bwd", P, P, P, None, None, P, P, 2, 50, 1.0)
    for name in ("token_logp", "policy_loss", "preference_loss"):
        with pytest.raises(ValueError, match="NULL result"):
            capi.call(f"oxi_{name}_workspace", 2, 50, None)
        with pytest.raises(ValueError, match="negative size"):
            getattr(capi, f"{name}_workspace")(-2, 50)
        assert getattr(capi, f"{name}_workspace")(0, 50) == 0


def test_policy_loss(capi):
    def call(drop=None, ws=P, low=0.2, high=0.2, most=0.0, kl=0.0, ent=0.0, div=1.0):
        capi.call("oxi_policy_loss_fwd", *without(12, drop), ws, 2, 50, 1.0, low, high, most, kl, ent, div)

    for i in (0, 1, 2, 6, 7, 9, 10):
        with pytest.raises(ValueError, match="NULL"):
            call(drop=i)
    for v in (-0.1, float("nan"), float("-inf")):
        with pytest.raises(ValueError, match="clipping"):
            call(low=v)
        with pytest.raises(ValueError, match="clipping"):
            call(high=v)
    for v in (0.5, -1.0, float("nan")):
        with pytest.raises(ValueError, match="clip_max"):
            call(most=v)
    for v in (float("nan"), float("inf")):
        with pytest.raises(ValueError, match="finite"):
            call(kl=v)
        with pytest.raises(ValueError, match="finite"):
            call(ent=v)
    for v in BAD:
        with pytest.raises(ValueError, match="divisor"):
            call(div=v)
    with pytest.raises(ValueError, match="needs the reference"):
        call(drop=4, kl=0.1)
    with pytest.raises(ValueError, match="16-byte aligned"):
        call(ws=P + 4)


def test_preference_loss(capi):
    def call(drop=None, ws=P, pairs=1, kind=0, beta=0.1, margin=0.0, smoothing=0.0):
        capi.call("oxi_preference_loss_fwd", *without(10, drop), ws, 2, 50, pairs, kind, 0, beta, margin, smoothing)

    for i in (0, 1, 2, 4, 5, 6, 7, 8):
        with pytest.raises(ValueError, match="NULL"):
            call(drop=i)
    with pytest.raises(ValueError, match="negative size"):
        call(pairs=-1)
    with pytest.raises(ValueError, match="kernel limits"):
        call(pairs=N)
    for k in (-1, 3):
        with pytest.raises(ValueError, match="unknown kind"):
            call(kind=k)
    for v in BAD:
        with pytest.raises(ValueError, match="beta"):
            call(beta=v)
    for v in (float("nan"), float("inf")):
        with pytest.raises(ValueError, match="margin"):
            call(margin=v)
    for v in (-0.1, 1.0, float("nan")):
        with pytest.raises(ValueError, match="smoothing"):
            call(smoothing=v)
    with pytest.raises(ValueError, match="sigmoid kind"):
        call(kind=1, smoothing=0.1)
    with pytest.raises(ValueError, match="16-byte aligned"):
        call(ws=P + 4)


def test_gradient_in_place_of_the_logits(capi):
    with pytest.raises(ValueError, match="must not be the logits"):
        capi.call("oxi_token_logp_bwd", P, Q, Q, Q, Q, Q, P, 2, 50, 1.0)
    with pytest.raises(ValueError, match="must not be the logits"):
        capi.call("oxi_policy_loss_fwd", P, *[Q] * 10, P, Q, 2, 50, 1.0, 0.2, 0.2, 0.0, 0.0, 0.0, 1.0)
    with pytest.raises(ValueError, match="must not be the logits"):
        capi.call("oxi_preference_loss_fwd", P, *[Q] * 8, P, Q, 2, 50, 1, 0, 0, 0.1, 0.0, 0.0)


def test_grad_norm_and_clip(capi):
    def slices(*rows):
        return capi.slice_array(capi.GradSlice, rows)

    def norm(s, count=1, p=2.0, total=P, ws=None):
        capi.call("oxi_grad_norm", s, count, p, total, ws)

    good = slices((P, P, 8))
    with pytest.raises(ValueError, match="negative slice count"):
        norm(good, -1)
    with pytest.raises(ValueError, match="NULL slice array"):
        norm(None)
    with pytest.raises(ValueError, match="negative size"):
        norm(slices((P, P, -1)))
    with pytest.raises(ValueError, match="NULL pointer"):
        norm(slices((None, P, 8)))
    for n in (1 << 50, np.iinfo(np.int64).max):
        with pytest.raises(ValueError, match="too large"):
            norm(slices((P, P, n)))
    for p in (0.0, 3.0, -1.0, float("nan"), float("-inf")):
        with pytest.raises(ValueError, match="must be 1, 2 or infinite"):
            norm(good, p=p)
    with pytest.raises(ValueError, match="total must not be NULL"):
        norm(good, total=None)
    for kw in ({"total": P + 4}, {"ws": P + 4}):
        with pytest.raises(ValueError, match="8-byte aligned"):
            norm(good, **kw)
    with pytest.raises(ValueError, match="NULL result"):
        capi.call("oxi_grad_norm_workspace", good, 1, None)
    with pytest.raises(ValueError, match="NULL pointer"):
        capi.call("oxi_grad_clip", slices((P, None, 8)), 1, P, 1.0)
    with pytest.raises(ValueError, match="total must not be NULL"):
        capi.call("oxi_grad_clip", good, 1, None, 1.0)
    with pytest.raises(ValueError, match="8-byte aligned"):
        capi.call("oxi_grad_clip", good, 1, P + 4, 1.0)
    with pytest.raises(ValueError, match="max_norm is NaN"):
        capi.call("oxi_grad_clip", good, 1, P, float("nan"))
