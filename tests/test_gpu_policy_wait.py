"""The policy loss over rows that lie over several blocks: a wait between a row's blocks that does
not end is given up and reported (forced from the host with OXI_CLUSTER_SPIN_LIMIT=-1, which fails
every wait at once: no kernel spins)."""

import os

import numpy as np
import pytest

from conftest import rng
from test_gpu_token_logp import logits_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("need_grad", [True, False])
@pytest.mark.parametrize("ent", [0.0, 0.01])
@pytest.mark.parametrize("c", [32801, 50257, 131072, 524288])
def test_waits_that_fail(hip, c, ent, need_grad):
    n = 5
    x = logits_of(n, c, 101)
    ids = x.argmax(1).astype(np.int64)
    ids[2] = -1
    on = ids >= 0
    D = hip.DeviceArray.from_numpy
    args = (D(x), D(ids), D(rng(102).standard_normal(n).astype(np.float32)), D(np.full(n, -1.0, np.float32)))

    def run():
        out, rows, logp, coef, saved, d = hip.policy_loss_fwd(*args, entropy_coef=ent, divisor=4.0, need_grad=need_grad)
        return [out.numpy(), rows.numpy()[0], logp.numpy(), coef.numpy()[0], saved.numpy()] + ([d.numpy()] if need_grad else [])

    clean = run()
    hip.sync()
    assert all(np.isfinite(a).all() for a in clean)
    print("[case] every wait between blocks fails", c, ent, need_grad, flush=True)
    os.environ["OXI_CLUSTER_SPIN_LIMIT"] = "-1"
    try:
        out, *rows = run()
        with pytest.raises(RuntimeError, match="wait between the blocks of a row did not finish"):
            hip.sync()
        # shorter rows have no such wait
        small = D(x[:, :32000].copy())
        got = hip.policy_loss_fwd(small, D(np.where(on, 0, -1)), *args[2:], entropy_coef=ent, need_grad=need_grad)
        assert np.isfinite(got[0].numpy()).all()
        hip.sync()
    finally:
        del os.environ["OXI_CLUSTER_SPIN_LIMIT"]
    assert np.isnan(out[0])
    for a, b in zip(rows[:3], clean[1:4]):
        assert np.isnan(a[on]).all() and np.array_equal(a[~on], b[~on])
    if need_grad:
        assert np.isnan(rows[-1][on]).all() and (rows[-1][~on] == 0).all()
    for a, b in zip(run(), clean):
        assert np.array_equal(a, b)
    hip.sync()
