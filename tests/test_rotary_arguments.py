"""Rotary offsets that are not whole numbers."""

import numpy as np
import pytest


@pytest.mark.parametrize("offset", [0.5, np.float64(2.25), float("inf"), float("nan")])
def test_an_offset_that_is_not_whole_is_refused(offset):
    """No GPU: it is checked before any device use."""
    import oxitorch_amd as ox
    from oxitorch_amd.nn import functional as F

    x = ox.from_numpy(np.zeros((2, 3, 1, 4), np.float32), device="cpu")
    with pytest.raises((TypeError, ValueError, OverflowError), match="offset|infinity|NaN"):
        F.rotary_embedding(x, [1.0, 0.1], offset=offset)


@pytest.mark.gpu
def test_whole_offsets(hip):
    import oxitorch_amd as ox
    from oxitorch_amd.nn import functional as F

    x = ox.from_numpy(np.random.default_rng(1).standard_normal((2, 3, 2, 4)).astype(np.float32))
    want = F.rotary_embedding(x, [1.0, 0.1], [7, 8, 9]).numpy()
    for offset in (7, np.int64(7), 7.0):
        assert np.array_equal(F.rotary_embedding(x, [1.0, 0.1], offset=offset).numpy(), want)
