"""The joint norm and clipping of one tensor whose chunks pass a launch (2^35 floats, 137 GB)."""

import numpy as np
import pytest

from conftest import rng
from test_gpu_operator_large import put, take

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def test_a_tensor_past_one_launch(hip):
    n = (1 << 35) + 12345
    print("[case] gradient of", n, "floats", flush=True)
    hip.call("oxi_hip_empty_cache")
    try:
        g = hip.DeviceArray((n,))
    except RuntimeError as e:
        pytest.skip(f"no room for 137 GB: {e}")
    try:
        hip.call("oxi_fill", g.ptr, n, 2.0 ** -10)
        tail = rng(5).standard_normal(1000).astype(np.float32)
        put(hip, g.ptr + (n - 1000) * 4, tail)
        small = hip.DeviceArray.from_numpy(np.full(3, 0.5, np.float32))
        total = hip.DeviceArray((1,), np.float64)
        s = hip.slice_array(hip.GradSlice, [(small.ptr, small.ptr, 3), (g.ptr, g.ptr, n)])
        hip.call("oxi_grad_norm", s, 2, 2.0, total.ptr, None)
        # the filled part and the small tensor are exact in 64 bits; 2^-53 a chunk's sum and more
        want = np.sqrt((n - 1000) * 2.0 ** -20 + (tail.astype(np.float64) ** 2).sum() + 0.75)
        assert abs(total.numpy()[0] - want) <= n * 2.0 ** -53 * want
        hip.call("oxi_grad_clip", s, 2, total.ptr, 1.0)
        f = 1.0 / (want + 1e-6)
        cut = ((2 ** 32 - 1) // 256) * 2048  # where a launch of 2048 floats a block ends
        for at in (0, 1 << 32, cut - 2048, cut, n - 1000 - 4096):
            got = take(hip, g.ptr + at * 4, (4096,))
            assert (np.abs(got - 2.0 ** -10 * f) <= 2.01 * U * 2.0 ** -10 * f).all(), at
        got = take(hip, g.ptr + (n - 1000) * 4, (1000,))
        assert (np.abs(got - tail * f) <= 2.01 * U * np.abs(tail * f)).all()
        assert (np.abs(small.numpy() - 0.5 * f) <= 2.01 * U * f).all()
        # each element was scaled once: the norm is 1 up to two roundings an element
        hip.call("oxi_grad_norm", s, 2, 2.0, total.ptr, None)
        assert abs(total.numpy()[0] - want * f) <= 2.01 * U
    finally:
        g.free()
        hip.call("oxi_hip_empty_cache")
