"""Shapes of rotary positions, no GPU: what is not one per token, or one per
batch and token in that order, is refused before any device use."""

import numpy as np
import pytest


@pytest.mark.parametrize("shape,given", [((2, 3, 1, 4), (3, 2)), ((4, 3, 1, 4), (2, 6)), ((2, 6, 1, 4), (3, 4)), ((6, 1, 4), (2, 3)),
                                         ((2, 3, 1, 4), (3, 1, 2)), ((1, 6, 1, 4), (2, 3))])
def test_refused(shape, given):
    import oxitorch_amd as ox
    from oxitorch_amd.nn import functional as F

    x = ox.from_numpy(np.zeros(shape, np.float32), device="cpu")
    pos = np.arange(np.prod(given)).reshape(given)
    for p in (pos, pos.tolist()):
        with pytest.raises(ValueError, match="positions of shape"):
            F.rotary_embedding(x, [1.0, 0.1], p)


@pytest.mark.gpu
@pytest.mark.parametrize("given", [(3,), (1, 3), (3, 1), (2, 3), (6,), (6, 1), (1, 2, 3)])
def test_taken(hip, given):
    """A row of positions for every batch, or one a batch, in any nesting that keeps their order."""
    import oxitorch_amd as ox
    from oxitorch_amd.nn import functional as F

    x = ox.from_numpy(np.random.default_rng(1).standard_normal((2, 3, 2, 4)).astype(np.float32))
    pos = (np.arange(np.prod(given)) * 7 + 1).reshape(given)
    full = np.broadcast_to(pos.reshape(-1, 3), (2, 3))
    want = F.rotary_embedding(x, [1.0, 0.1], full).numpy()
    assert np.array_equal(F.rotary_embedding(x, [1.0, 0.1], pos).numpy(), want)
    one = ox.from_numpy(x.numpy()[0])
    if pos.size == 3:
        assert np.array_equal(F.rotary_embedding(one, [1.0, 0.1], pos).numpy(), want[0])
