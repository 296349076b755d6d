"""Which rows the mean of the distillation loss is over: those that hold an entry,
an entry being an id of a class with a teacher's logit above -inf. Against float64,
the bounds of test_gpu_distill."""

import ctypes

import numpy as np
import pytest

from test_gpu_distill import U, oracle, student_and_teacher, teacher_lse

pytestmark = pytest.mark.gpu


def batch(n, c, k):
    x, ids, top, teacher = student_and_teacher(n, c, k, n + c + k)
    top[1] = -np.inf  # every id stays: masked logits
    ids[2] = -1
    ids[3, : k // 2] = -1
    top[3, k // 2:] = -np.inf  # neither half is an entry
    ids[4, : k // 2] = -1
    return x, ids, top, teacher


@pytest.mark.parametrize("n,c,k", [(5, 9, 2), (9, 300, 8), (70, 515, 100), (8, 70001, 70), (300, 40, 6)])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("as_tensor", [False, True])
def test_masked_rows_stay_out_of_the_mean(hip, n, c, k, tail, as_tensor):
    import oxitorch_amd as ox
    from oxitorch_amd.nn import functional as F

    T = 1.5
    x, ids, top, teacher = batch(n, c, k)
    lse = teacher_lse(teacher, T) if tail else None
    w = oracle(x, ids, top, T, lse, float(n - 3))
    for scale in (None, 2.0):
        t = ox.from_numpy(x, True)
        loss = F.distillation_loss(t, ids, ox.from_numpy(top) if as_tensor else top, T, lse)
        assert abs(loss.item() - w["loss"]) <= w["bloss"]
        (loss if scale is None else loss * scale).backward()
        up = scale or 1.0
        assert (np.abs(t.grad.numpy() - up * w["grad"]) <= up * (w["bgrad"] + 16 * U * np.abs(w["grad"]))).all()
        assert (t.grad.numpy()[1:4] == 0).all()


def test_counted_on_the_device(hip):
    """The C-ABI calls: the count, and bit by bit the values of the calls that are given it."""
    D = hip.DeviceArray.from_numpy
    for n, c, k in ((5, 9, 2), (9, 300, 8), (1100, 96, 6), (8, 70001, 1000)):
        x, ids, top, teacher = batch(n, c, k)
        lse = D(teacher_lse(teacher, 2.0))
        a = [D(v) for v in (x, ids, top)]
        for e in (None, lse):
            want = hip.distill_fwd(*a, 2.0, e, float(n - 3), need_grad=True)
            got = [hip.DeviceArray(v.shape) for v in want] + [hip.DeviceArray((1,))]
            hip.call("oxi_distill_fwd_counted", *(v.ptr for v in a), e.ptr if e else None, *(v.ptr for v in got), n, c, k, 2.0)
            assert got[5].numpy()[0] == n - 3
            for p, q in zip(got, want):
                assert np.array_equal(p.numpy(), q.numpy())
            up = D(np.array([-0.7], np.float32))
            back = hip.DeviceArray((n, c))
            hip.call("oxi_distill_bwd_counted", *(v.ptr for v in a), e.ptr if e else None, got[2].ptr, got[3].ptr, up.ptr,
                     back.ptr, got[5].ptr, n, c, k, 2.0)
            assert np.array_equal(back.numpy(), hip.distill_bwd(*a, want[2], want[3], up, 2.0, e, float(n - 3)).numpy())
    one = [hip.DeviceArray((1,)) for _ in range(2)]
    hip.call("oxi_distill_fwd_counted", None, None, None, None, one[0].ptr, None, None, None, None, one[1].ptr, 0, 9, 2, 1.0)
    assert one[0].numpy()[0] == 0 and one[1].numpy()[0] == 1


def test_no_row_holds_an_entry(hip):
    import oxitorch_amd as ox
    from oxitorch_amd.nn import functional as F

    x = np.ones((3, 50), np.float32)
    for ids, top in ((np.full((3, 4), -1), np.zeros((3, 4), np.float32)), (np.zeros((3, 4), np.int64), np.full((3, 4), -np.inf, np.float32))):
        t = ox.from_numpy(x, True)
        loss = F.distillation_loss(t, ids, ox.from_numpy(top))
        loss.backward()
        assert loss.item() == 0 and (t.grad.numpy() == 0).all()


def test_captured_and_replayed(hip):
    """Both calls in a graph, replayed on new inputs with eager calls between: the eager bits every time."""
    from test_gpu_graph import CAPTURE_MODE_RELAXED, _runtime

    rt = _runtime()
    stream = ctypes.c_void_p()
    hip.check(hip.lib.oxi_hip_stream(ctypes.byref(stream)))
    n, c, k, T = 30, 3000, 9, 2.0
    A = hip.DeviceArray

    def buffers():
        return dict(x=A((n, c)), ids=A((n, k), np.int64), top=A((n, k)), tlse=A((n,)), loss=A((1,)), row=A((n,)), lse=A((n,)),
                    rest=A((n,)), d=A((n, c)), d2=A((n, c)), count=A((1,)), up=A((1,)))

    def step(b):
        p = {m: v.ptr for m, v in b.items()}
        hip.call("oxi_distill_fwd_counted", p["x"], p["ids"], p["top"], p["tlse"], p["loss"], p["row"], p["lse"], p["rest"],
                 p["d"], p["count"], n, c, k, T)
        hip.call("oxi_distill_bwd_counted", p["x"], p["ids"], p["top"], p["tlse"], p["lse"], p["rest"], p["up"], p["d2"],
                 p["count"], n, c, k, T)

    def fill(b, seed):
        x, ids, top, teacher = student_and_teacher(n, c, k, seed)
        top[: seed % 7] = -np.inf
        for m, v in (("x", x), ("ids", ids), ("top", top), ("tlse", teacher_lse(teacher, T)), ("up", np.array([0.3], np.float32))):
            v = np.ascontiguousarray(v)
            hip.check(hip.lib.oxi_hip_memcpy_h2d(b[m].ptr, v.ctypes.data, v.nbytes))

    b, eager = buffers(), buffers()
    fill(b, 1)
    step(b)
    hip.sync()
    graph, exe = ctypes.c_void_p(), ctypes.c_void_p()
    assert rt.hipStreamBeginCapture(stream, CAPTURE_MODE_RELAXED) == 0
    try:
        step(b)
    finally:
        rc = rt.hipStreamEndCapture(stream, ctypes.byref(graph))  # the stream never stays capturing
    assert rc == 0 and graph.value
    try:
        assert rt.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0) == 0
        for seed in (3, 5, 6, 2):
            print("[case] replay", seed, flush=True)
            fill(b, seed)
            assert rt.hipGraphLaunch(exe, stream) == 0
            hip.sync()
            fill(eager, seed)
            step(eager)
            hip.sync()
            assert b["count"].numpy()[0] == n - seed % 7
            for m in ("loss", "row", "lse", "rest", "d", "d2"):
                assert np.array_equal(b[m].numpy(), eager[m].numpy()), (seed, m)
    finally:
        if exe.value:
            rt.hipGraphExecDestroy(exe)
        rt.hipGraphDestroy(graph)
