"""What the distillation calls that count their rows refuse, no GPU."""

import pytest

P = 1 << 20  # a non-NULL address that no refused call touches


def test_refusals():
    from oxitorch_amd import capi

    def fwd(n=2, c=50, k=4, T=1.0, drop=None):
        a = [P] * 10
        if drop is not None:
            a[drop] = None
        capi.call("oxi_distill_fwd_counted", *a, n, c, k, T)

    for i in (0, 1, 2, 4, 5, 6, 7, 9):
        with pytest.raises(ValueError, match="distill_fwd_counted.*NULL"):
            fwd(drop=i)
    for kw, match in (({"n": -1}, "negative"), ({"c": 0}, "zero classes"), ({"k": 1025}, "teacher entries"), ({"T": 0.0}, "temperature")):
        with pytest.raises(ValueError, match=match):
            fwd(**kw)
    for i in (0, 1, 2, 4, 5, 6, 7, 8):
        a = [P] * 9
        a[i] = None
        with pytest.raises(ValueError, match="distill_bwd_counted.*NULL"):
            capi.call("oxi_distill_bwd_counted", *a, 2, 50, 4, 1.0)
