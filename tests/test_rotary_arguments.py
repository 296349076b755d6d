"""Rotary frequencies as a tuple of numbers, and offsets that are not whole."""

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


@pytest.mark.gpu
@pytest.mark.parametrize("inv", [(0.5,), (0.5, 0.25), (1.0, 0.5, 0.25)])
def test_frequencies_as_a_tuple_of_numbers(hip, inv):
    """Two of them are two frequencies, not one with a scale."""
    import oxitorch_amd as ox
    from oxitorch_amd.nn import functional as F

    x = ox.from_numpy(np.random.default_rng(2).standard_normal((1, 3, 2, 8)).astype(np.float32))
    want = F.rotary_embedding(x, np.array(inv)).numpy()
    assert np.array_equal(F.rotary_embedding(x, inv).numpy(), want)
    scaled = F.rotary_embedding(x, (np.array(inv), 2.0)).numpy()
    n = 2 * len(inv)
    assert np.allclose(scaled[..., :n], 2 * want[..., :n], rtol=1e-6) and np.array_equal(scaled[..., n:], want[..., n:])
