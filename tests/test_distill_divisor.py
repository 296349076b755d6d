"""The divisor that the ctypes binding of distillation is given reaches the call, no GPU."""

import pytest


class Buffer:
    ptr, shape = 1 << 20, (3, 2)

    def __init__(self, *_):
        pass


@pytest.mark.parametrize("divisor", [0, 0.0, -1.0, float("nan")])
def test_a_divisor_that_divides_nothing_is_refused(monkeypatch, divisor):
    """Given as 0 it was taken for none given."""
    from oxitorch_amd import capi

    monkeypatch.setattr(capi, "DeviceArray", Buffer)
    b = Buffer()
    with pytest.raises(ValueError, match="divisor"):
        capi.distill_fwd(b, b, b, divisor=divisor)
    with pytest.raises(ValueError, match="divisor"):
        capi.distill_bwd(b, b, b, b, b, b, divisor=divisor)
