"""Numbers that draft verification takes, no GPU: arrays are checked before any device use."""

import numpy as np
import pytest


@pytest.mark.parametrize("bad", [1.0, 1.5, -0.25, float("nan"), float("inf")])
def test_numbers_outside_the_unit_interval_are_refused(bad):
    import oxitorch_amd as ox
    from oxitorch_amd.nn import functional as F

    target = ox.from_numpy(np.zeros((3, 3, 8), np.float32), device="cpu")
    u = np.zeros((3, 3))
    u[1, 2] = bad
    for numbers in (u, u.astype(np.float32), u.tolist()):
        with pytest.raises(ValueError, match=r"\[0, 1\)"):
            F.verify_drafts(np.zeros((3, 2), np.int64), None, target, numbers)
