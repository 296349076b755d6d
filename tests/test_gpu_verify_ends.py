"""Draft verification where the numbers drawn and the probabilities leave their
range: the definition of test_gpu_verify in float64, whole numbers, equal."""

import numpy as np
import pytest

from test_gpu_verify import make, oracle, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("v", [5, 300, 1000, 8192, 32000, 131072])
@pytest.mark.parametrize("u1", [1.0, 1.5, float("inf")])
def test_a_number_that_reaches_one_draws_the_last_class(hip, v, u1):
    """No running sum passes the limit then: the last class with weight, of what the draft leaves and of a row itself,
    where pieces and threads behind it weigh nothing too."""
    target, draft, tokens, u = make(6, 2, v, v)
    target[:, :, v - 1] = 0
    target[3:, :, v // 2:] = 0
    u[:, 2] = u1
    u[1, 0] = u[2, 1] = 0.99999
    for d in (draft, None):
        a, o = run(hip, target, d, tokens, u)
        wa, wo, _ = oracle(target, d, tokens, u)
        assert np.array_equal(a, wa) and np.array_equal(o, wo), (o, wo)


@pytest.mark.parametrize("v", [7, 1003, 40000])
def test_negative_draft_probabilities_weigh_nothing(hip, v):
    """As the zeros that they stand for: neither does such a token's draft get in by its product, nor the class a
    greater weight."""
    target, draft, tokens, u = make(8, 3, v, v)
    draft[:, :, ::2] -= np.float32(0.3)
    draft[0] = -draft[0]
    target[1] = -target[1]  # weighs nothing either, whatever the draft is
    draft[1] = -1.0
    tokens[2] = 0
    draft[3, :, 1] = np.nan
    assert (draft < 0).any()
    a, o = run(hip, target, draft, tokens, u)
    wa, wo, margin = oracle(target, np.where(draft < 0, np.float32(0), draft), tokens, u)
    assert (margin > 1e-12).all()
    assert np.array_equal(a, wa) and np.array_equal(o, wo)
    assert a[1] == 0 and (o[1] == -1).all()


def test_numbers_in_64_bits(hip):
    """Numbers below 1 that 32 bits would round to it draw as the largest float below 1 does."""
    import oxitorch_amd as ox
    from oxitorch_amd.nn import functional as F

    target, draft, tokens, u = make(5, 2, 1000, 3)
    t, d = ox.from_numpy(target), ox.from_numpy(draft)
    high = u.astype(np.float64)
    high[:, 2] = 1 - 2.0 ** -40
    high[0, 0] = 1 - 2.0 ** -53
    below = high.astype(np.float32)
    below[below >= 1] = np.float32(1 - 2.0 ** -24)
    a, o = F.verify_drafts(tokens, d, t, high)
    wa, wo, _ = oracle(target, draft, tokens, below)
    assert np.array_equal(a, wa) and np.array_equal(o, wo)
    a, o = F.verify_drafts(tokens, d, t, high.tolist())
    assert np.array_equal(a, wa) and np.array_equal(o, wo)
