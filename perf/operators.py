"""The language-model operators whose performance is measured: the residual
RMS norm (with its VJP and its 8-bit output), rotary positions, distillation
from a teacher's top logits, and the verification of drafted tokens.

Each has a plain form in elementary tensor operations and, with `own`, the
framework's C-ABI calls on the same buffers. Sizes come from the benchmark's
configurations and the tests, or are generic; `draw` gives more cases of the
same ranges.
"""

from __future__ import annotations

import ctypes
import math

import torch

own = False

F32 = 4
EPS = 1e-6
E4M3_MAX = 448.0
VJP_MODE = {"ref": 0, "exact": 1}
LAYOUT = {"half": 0, "interleaved": 1}


def listed():
    return [
        # one decode step's residual add and norm for a batch of 8 sequences: latency
        {"name": "addnorm_decode", "op": "norm", "rows": 8, "cols": 4096, "out": "f32", "grad": False, "mode": "ref"},
        # a training batch of the benchmark's layer size, both directions, full derivative
        {"name": "addnorm_train", "op": "norm", "rows": 16384, "cols": 4096, "out": "f32", "grad": True, "mode": "exact"},
        # an odd model width of the tests' width sweep, the graph's default VJP
        {"name": "addnorm_odd", "op": "norm", "rows": 8192, "cols": 1003, "out": "f32", "grad": True, "mode": "ref"},
        # a prefill whose normed rows go to an 8-bit product: a scale for each 128 columns
        {"name": "addnorm_e4m3", "op": "norm", "rows": 8192, "cols": 4096, "out": "e4m3", "group": 128, "grad": False,
         "mode": "ref"},
        # one decode step of 64 sequences at far positions, query and key heads in one buffer
        {"name": "rotary_decode", "op": "rotary", "batch": 64, "tokens": 1, "heads": 40, "dim": 128, "rot": 128,
         "layout": "half", "heads_first": False, "far": 131072, "factor": 32.0, "grad": False},
        # a training batch, both directions
        {"name": "rotary_train", "op": "rotary", "batch": 4, "tokens": 4096, "heads": 32, "dim": 128, "rot": 128,
         "layout": "half", "heads_first": False, "far": 0, "factor": 1.0, "grad": True},
        # half of each head rotated, interleaved pairs, heads before tokens, a ragged length
        {"name": "rotary_partial", "op": "rotary", "batch": 16, "tokens": 1023, "heads": 12, "dim": 64, "rot": 32,
         "layout": "interleaved", "heads_first": True, "far": 0, "factor": 1.0, "grad": True},
        # a small batch distilled from a teacher's 8 best tokens: latency
        {"name": "distill_small", "op": "distill", "rows": 64, "classes": 32000, "top": 8, "temperature": 1.0,
         "tail": False, "pad": 0.0},
        # the benchmark's logits, 64 teacher entries and the teacher's remaining mass
        {"name": "distill_large", "op": "distill", "rows": 8192, "classes": 32000, "top": 64, "temperature": 2.0,
         "tail": True, "pad": 0.0},
        # the odd vocabulary, ragged teacher lists, padded rows
        {"name": "distill_odd", "op": "distill", "rows": 4096, "classes": 50257, "top": 50, "temperature": 1.0,
         "tail": False, "pad": 0.25},
        # one step of a few sequences with 4 drafted tokens each: latency
        {"name": "verify_small", "op": "verify", "batch": 4, "drafts": 4, "vocab": 32000, "ragged": False, "greedy": False},
        # a serving batch over a large vocabulary, draft lengths that differ
        {"name": "verify_large", "op": "verify", "batch": 128, "drafts": 7, "vocab": 131072, "ragged": True,
         "greedy": False},
    ]


def _log(rng, lo, hi):
    """A size in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A row width: half of them any number, half a multiple of 64 (or 4)."""
    w = _log(rng, lo, hi)
    if rng.random() < 0.5:
        m = 64 if w >= 128 else 4
        w = max(lo, min(hi, (w + m // 2) // m * m))
    return w


def draw(rng):
    op = rng.choice(["norm", "rotary", "distill", "verify"])
    if op == "norm":
        cols = _width(rng, 16, 16384)
        rows = _log(rng, 1, min(32768, (1 << 26) // cols))
        if rng.random() < 0.3:
            return {"op": op, "rows": rows, "cols": cols, "out": "e4m3", "group": rng.choice([32, 64, 128, 256, cols]),
                    "grad": False, "mode": "ref"}
        return {"op": op, "rows": rows, "cols": cols, "out": "f32", "grad": rng.random() < 0.7,
                "mode": rng.choice(["ref", "exact"])}
    if op == "rotary":
        dim = rng.choice([32, 40, 64, 80, 96, 128, 160, 192, 256])
        rot = dim if rng.random() < 0.6 else rng.choice([dim // 2, dim // 4 * 2, max(2, dim // 8 * 2)])
        heads = _log(rng, 1, 64)
        grad = rng.random() < 0.6
        tokens = _log(rng, 1, 16384)
        batch = _log(rng, 1, max(1, min(128, (1 << 26) // (dim * heads * tokens))))
        while batch * tokens * heads * dim > 1 << 26:
            tokens = max(1, tokens // 2)
        return {"op": op, "batch": batch, "tokens": tokens, "heads": heads, "dim": dim, "rot": rot,
                "layout": rng.choice(["half", "interleaved"]), "heads_first": rng.random() < 0.4,
                "far": rng.choice([0, 4096, 131072, 1000000]), "factor": rng.choice([1.0, 4.0, 32.0]), "grad": grad}
    if op == "distill":
        classes = _width(rng, 256, 200000)
        return {"op": op, "rows": _log(rng, 1, min(16384, (1 << 28) // classes)), "classes": classes,
                "top": _log(rng, 1, 200), "temperature": rng.choice([0.7, 1.0, 2.0, 4.0]), "tail": rng.random() < 0.5,
                "pad": rng.choice([0.0, 0.25])}
    vocab = _width(rng, 256, 262144)
    drafts = _log(rng, 1, 16)
    return {"op": op, "batch": _log(rng, 1, max(1, min(256, (1 << 27) // (vocab * (drafts + 1))))), "drafts": drafts,
            "vocab": vocab, "ragged": rng.random() < 0.5, "greedy": rng.random() < 0.25}


# ---- inputs -----------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape, scale=1.0, shift=0.0):
    t = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    return t.mul_(scale).add_(shift)


def _frequencies(case):
    """Angles per position of the rotated pairs (64 bits): base 10000, and for
    factor > 1 the slow pairs of a context of 4096 stretched by the factor,
    the fast ones (over 32 turns in it) as they are, a ramp between."""
    half = case["rot"] // 2
    f = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
    s = case["factor"]
    if s > 1:
        keep = ((4096 * f / (2 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        f = (1 - keep) * f / s + keep * f
    return f.cuda(), (0.1 * math.log(s) + 1.0) if s > 1 else 1.0


def _strides(t):
    return (ctypes.c_int64 * t.dim())(*t.stride())


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    if case["op"] == "norm":
        r, c = case["rows"], case["cols"]
        s.update(x=_randn(g, r, c, scale=0.5), r=_randn(g, r, c, scale=2.0), w=_randn(g, c, scale=0.1, shift=1.0))
        s["h"] = torch.empty_like(s["x"])
        if case["out"] == "e4m3":
            # a trained norm's outputs have columns that stand out
            s["w"] *= torch.where(torch.rand(c, generator=g, device="cuda") < 0.01, 20.0, 1.0)
            s["q"] = torch.empty(r, c, dtype=torch.uint8, device="cuda")
            s["scale"] = torch.empty(r, -(-c // case["group"]), device="cuda")
        else:
            s.update(y=torch.empty_like(s["x"]), rstd=torch.empty(r, device="cuda"))
        if case["grad"]:
            s.update(gy=_randn(g, r, c), gh=_randn(g, r, c), dx=torch.empty_like(s["x"]), dw=torch.empty(c, device="cuda"))
    elif case["op"] == "rotary":
        b, t, h, d = case["batch"], case["tokens"], case["heads"], case["dim"]

        def make():
            v = _randn(g, b, h, t, d) if case["heads_first"] else _randn(g, b, t, h, d)
            return v.permute(0, 2, 1, 3) if case["heads_first"] else v  # (batch, tokens, heads, dim), strided

        s["x"] = make()
        start = torch.randint(0, max(1, case["far"]), (b, 1), generator=g, device="cuda")
        s["pos"] = start + torch.arange(t, device="cuda")
        s["freq"], s["scale"] = _frequencies(case)
        s["y"] = torch.empty_like(s["x"])
        s["shape"] = (ctypes.c_int64 * 4)(b, t, h, d)
        s["xs"], s["ys"], s["ps"] = _strides(s["x"]), _strides(s["y"]), _strides(s["pos"])
        if case["grad"]:
            s["g"] = make()
            s["dx"] = torch.empty_like(s["g"])
            s["gs"], s["ds"] = _strides(s["g"]), _strides(s["dx"])
    elif case["op"] == "distill":
        n, c, k = case["rows"], case["classes"], min(case["top"], case["classes"])
        teacher = _randn(g, n, c, scale=2.0)
        s["x"] = (teacher * 0.8).add_(_randn(g, n, c))  # a student that follows its teacher
        s["top"], s["ids"] = torch.topk(teacher, k, dim=1)
        s["lse"] = torch.logsumexp(teacher / case["temperature"], 1) if case["tail"] else None
        del teacher
        if case["pad"]:
            count = torch.randint(1, k + 1, (n, 1), generator=g, device="cuda")
            count *= (torch.rand(n, 1, generator=g, device="cuda") >= case["pad"])  # padded tokens: no entry
            s["ids"] = torch.where(torch.arange(k, device="cuda") < count, s["ids"], -1)
        s["divisor"] = float(max(1, int((s["ids"][:, 0] >= 0).sum())))
        new = lambda *shape: torch.empty(shape, device="cuda")  # noqa: E731
        s.update(loss=new(1), row_loss=new(n), slse=new(n), rest=new(n), dx=new(n, c))
    else:
        b, k, v = case["batch"], case["drafts"], case["vocab"]
        logits = _randn(g, b, k + 1, v, scale=3.0)
        s["target"] = torch.softmax(logits, 2)
        if case["greedy"]:  # drafts that come with no probabilities of their own (a lookup, a greedy model)
            s["draft"] = None
            s["tokens"] = logits[:, :k].argmax(2)
        else:
            s["draft"] = torch.softmax(logits[:, :k] + _randn(g, b, k, v, scale=0.7), 2)
            noise = torch.empty_like(s["draft"]).exponential_(generator=g)
            s["tokens"] = (s["draft"] / noise).argmax(2)  # a sample of each row
            del noise
        del logits
        s["lengths"] = torch.randint(0, k + 1, (b,), generator=g, device="cuda") if case["ragged"] else None
        s["u"] = torch.rand(b, k + 1, generator=g, device="cuda")
        s["accepted"] = torch.empty(b, dtype=torch.int64, device="cuda")
        s["out"] = torch.empty(b, k + 1, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()  # the library has a stream of its own
    return s


# ---- one pass -----------------------------------------------------------------------

def run(s):
    case = s["case"]
    if own:
        return _OWN[case["op"]](s, case)
    return _PLAIN[case["op"]](s, case)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _own_norm(s, case):
    from oxitorch_amd import capi

    r, c = case["rows"], case["cols"]
    if case["out"] == "e4m3":
        capi.call("oxi_add_rms_norm_e4m3_fwd", _ptr(s["x"]), _ptr(s["r"]), _ptr(s["w"]), _ptr(s["h"]), _ptr(s["q"]),
                  _ptr(s["scale"]), r, c, case["group"], EPS)
        return {"h": s["h"], "q": s["q"].view(torch.float8_e4m3fn), "scale": s["scale"]}
    capi.call("oxi_add_rms_norm_fwd", _ptr(s["x"]), _ptr(s["r"]), _ptr(s["w"]), _ptr(s["h"]), _ptr(s["y"]),
              _ptr(s["rstd"]), r, c, EPS)
    out = {"h": s["h"], "y": s["y"], "rstd": s["rstd"]}
    if case["grad"]:
        capi.call("oxi_add_rms_norm_bwd", _ptr(s["h"]), _ptr(s["w"]), _ptr(s["rstd"]), _ptr(s["gy"]), _ptr(s["gh"]),
                  _ptr(s["dx"]), _ptr(s["dw"]), None, r, c, VJP_MODE[case["mode"]])
        out.update(dx=s["dx"], dw=s["dw"])
    return out


def _own_rotary(s, case):
    from oxitorch_amd import capi

    tail = (s["shape"], _ptr(s["pos"]), s["ps"], 0, _ptr(s["freq"]), case["rot"], LAYOUT[case["layout"]])
    capi.call("oxi_rotary", _ptr(s["x"]), s["xs"], _ptr(s["y"]), s["ys"], *tail, 0, s["scale"])
    out = {"y": s["y"]}
    if case["grad"]:
        capi.call("oxi_rotary", _ptr(s["g"]), s["gs"], _ptr(s["dx"]), s["ds"], *tail, 1, s["scale"])
        out["dx"] = s["dx"]
    return out


def _own_distill(s, case):
    from oxitorch_amd import capi

    (n, c), k = s["x"].shape, s["ids"].shape[1]
    capi.call("oxi_distill_fwd", _ptr(s["x"]), _ptr(s["ids"]), _ptr(s["top"]), _ptr(s["lse"]), _ptr(s["loss"]),
              _ptr(s["row_loss"]), _ptr(s["slse"]), _ptr(s["rest"]), _ptr(s["dx"]), n, c, k, case["temperature"],
              s["divisor"])
    return {"loss": s["loss"], "row_loss": s["row_loss"], "dx": s["dx"]}


def _own_verify(s, case):
    from oxitorch_amd import capi

    capi.call("oxi_verify_drafts", _ptr(s["target"]), _ptr(s["draft"]), _ptr(s["tokens"]), _ptr(s["lengths"]),
              _ptr(s["u"]), _ptr(s["accepted"]), _ptr(s["out"]), None, case["batch"], case["drafts"], case["vocab"])
    return {"accepted": s["accepted"], "tokens": s["out"]}


_OWN = {"norm": _own_norm, "rotary": _own_rotary, "distill": _own_distill, "verify": _own_verify}


def _grouped(y, group):
    """y's columns in groups, the last filled with zeros."""
    r, c = y.shape
    n = -(-c // group)
    if n * group != c:
        y = torch.cat([y, y.new_zeros(r, n * group - c)], 1)
    return y.view(r, n, group)


def _plain_norm(s, case):
    h = s["x"] + s["r"]
    rstd = 1.0 / torch.sqrt((h * h).mean(1, keepdim=True) + EPS)
    xh = h * rstd
    y = xh * s["w"]
    if case["out"] == "e4m3":
        v = _grouped(y, case["group"])
        scale = (v.abs().amax(2) / E4M3_MAX).clamp_(min=2.0 ** -126)
        q = (v / scale[:, :, None]).view(h.shape[0], -1)[:, : h.shape[1]]
        return {"h": h, "q": q.to(torch.float8_e4m3fn), "scale": scale}
    out = {"h": h, "y": y, "rstd": rstd[:, 0]}
    if case["grad"]:
        gw = s["gy"] * s["w"]
        if case["mode"] == "exact":
            gw = gw - xh * (gw * xh).mean(1, keepdim=True)
        out["dx"] = s["gh"] + gw * rstd
        out["dw"] = (s["gy"] * xh).sum(0)
    return out


def _turned(x, cos, sin, rot, layout):
    a = x[..., :rot]
    if layout == "half":
        u, v = a[..., : rot // 2], a[..., rot // 2:]
        t = torch.cat([u * cos - v * sin, v * cos + u * sin], 3)
    else:
        u, v = a[..., 0::2], a[..., 1::2]
        t = torch.stack([u * cos - v * sin, v * cos + u * sin], 4).flatten(3)
    return t if rot == x.shape[3] else torch.cat([t, x[..., rot:]], 3)


def _plain_rotary(s, case):
    angle = (s["pos"].double()[:, :, None] * s["freq"])[:, :, None, :]
    cos, sin = (torch.cos(angle) * s["scale"]).float(), (torch.sin(angle) * s["scale"]).float()
    out = {"y": _turned(s["x"], cos, sin, case["rot"], case["layout"])}
    if case["grad"]:
        out["dx"] = _turned(s["g"], cos, -sin, case["rot"], case["layout"])
    return out


def _plain_distill(s, case):
    T, ids = case["temperature"], s["ids"]
    there = ids >= 0
    t = torch.where(there, s["top"] / T, -math.inf).double()
    if case["tail"]:
        p = torch.exp(t - s["lse"].double()[:, None])
        rest_p = (1.0 - p.sum(1)).clamp_(min=0.0) * there.any(1)
    else:
        p = torch.exp(t - t.amax(1, keepdim=True).clamp_(min=-1e30))
        p = p / p.sum(1, keepdim=True).clamp_(min=1e-300)
    z = s["x"] / T
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(1, keepdim=True)
    at = ids.clamp(min=0)
    d = s["x"].gather(1, at).double() / T - m - torch.log(total.double()) - torch.log(p)  # log(q / p)
    q = e / total
    if case["tail"]:
        # ids that are padding stand for the row's first entry, whose own value comes back below
        at = torch.where(there, ids, ids[:, :1]).clamp(min=0)
        rest_q = q.scatter(1, at, 0.0).sum(1).double()
        # both sides' masses sum to 1, so p log(p/q) may be summed as q - p + p log(p/q), which is never
        # negative: a student near its teacher has a small loss of large terms otherwise
        row = torch.where(p > 0, p * (torch.expm1(d) - d), 0.0).sum(1)
        d = torch.log(rest_q) - torch.log(rest_p)
        row = row + torch.where(rest_p > 0, rest_p * (torch.expm1(d) - d), rest_q * there.any(1))
        g = (q * ((rest_q - rest_p) / rest_q)[:, None].float()).scatter(1, at, q.gather(1, at))
    else:
        row = torch.where(p > 0, -p * d, 0.0).sum(1)
        g = q
    g = g.scatter_add(1, at, -p.float()) * (T / s["divisor"])
    g = torch.where(there.any(1)[:, None], g, 0.0)
    row = row * (T * T)
    return {"loss": (row.sum() / s["divisor"]).float().reshape(1), "row_loss": row.float(), "dx": g}


def _plain_verify(s, case):
    b, k = case["batch"], case["drafts"]
    rows = torch.arange(b, device="cuda")
    tok = s["tokens"]
    p = s["target"][:, :k].gather(2, tok[:, :, None])[:, :, 0].double()
    q = s["draft"].gather(2, tok[:, :, None])[:, :, 0].double() if s["draft"] is not None else torch.ones_like(p)
    ok = s["u"][:, :k].double() * q < p
    length = s["lengths"] if s["lengths"] is not None else torch.full((b,), k, device="cuda")
    ok = ok & (torch.arange(k, device="cuda") < length[:, None])
    count = ok.long().cumprod(1).sum(1)
    w = s["target"][rows, count].double()
    at = count.clamp(max=k - 1)
    if s["draft"] is not None:
        left = (w - s["draft"][rows, at].double()).clamp_(min=0.0)
    else:
        left = w.scatter(1, tok[rows, at][:, None], 0.0)
    rejected = (count < length) & (left.sum(1) > 0)
    w = torch.where(rejected[:, None], left, w)
    run_sum = torch.cumsum(w, 1)
    token = (run_sum <= s["u"][:, k:].double() * run_sum[:, -1:]).sum(1)
    place = torch.arange(k + 1, device="cuda")
    drafts = torch.cat([tok, tok[:, :1]], 1)
    out = torch.where(place < count[:, None], drafts, torch.where(place == count[:, None], token[:, None], -1))
    return {"accepted": count, "tokens": out}


_PLAIN = {"norm": _plain_norm, "rotary": _plain_rotary, "distill": _plain_distill, "verify": _plain_verify}


# ---- what a pass cannot do without -----------------------------------------------

def work(case):
    """Each input that the pass depends on read once, each output written once."""
    if case["op"] == "norm":
        r, c = case["rows"], case["cols"]
        e = r * c * F32
        if case["out"] == "e4m3":
            return {"bytes": 3 * e + r * c + (r * -(-c // case["group"]) + c) * F32, "flops": 0}
        return {"bytes": (8 if case["grad"] else 4) * e + (r + 2 * c) * F32, "flops": 0}
    if case["op"] == "rotary":
        e = case["batch"] * case["tokens"] * case["heads"] * case["dim"] * F32
        return {"bytes": (4 if case["grad"] else 2) * e + case["batch"] * case["tokens"] * 8 + case["rot"] * 4, "flops": 0}
    if case["op"] == "distill":
        n, c, k = case["rows"], case["classes"], min(case["top"], case["classes"])
        return {"bytes": 2 * n * c * F32 + 12 * n * k + 8 * n, "flops": 0}
    b, k, v = case["batch"], case["drafts"], case["vocab"]
    return {"bytes": b * ((1 if case["greedy"] else 2) * v * F32 + 28 * k + 24), "flops": 0}


# ---- the same in 64 bits -----------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    d = lambda n: s[n].double()  # noqa: E731
    if case["op"] == "norm":
        h = d("x") + d("r")
        norm = torch.sqrt(h.pow(2).sum(1) / case["cols"] + EPS)
        y = h / norm[:, None] * d("w")
        if case["out"] == "e4m3":
            parts = [part.abs().max(1).values for part in y.split(case["group"], 1)]
            scale = torch.stack(parts, 1) / E4M3_MAX
            wide = scale.repeat_interleave(case["group"], 1)[:, : case["cols"]]
            return {"h": h, "q": y / wide, "scale": scale}
        out = {"h": h, "y": y, "rstd": 1 / norm}
        if case["grad"]:
            unit = h / norm[:, None]
            up = d("gy") * d("w")
            along = (up * unit).sum(1, keepdim=True) / case["cols"] if case["mode"] == "exact" else 0.0
            out["dx"] = d("gh") + (up - along * unit) / norm[:, None]
            out["dw"] = torch.einsum("rc,rc->c", d("gy"), unit)
        return out
    if case["op"] == "rotary":
        phase = s["scale"] * torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                                         torch.einsum("bt,f->btf", d("pos"), s["freq"]))[:, :, None]

        def turn(x, by):
            r = case["rot"]
            pairs = x[..., :r].unflatten(3, (2, r // 2)).transpose(3, 4) if case["layout"] == "half" \
                else x[..., :r].unflatten(3, (r // 2, 2))
            z = torch.view_as_real(torch.complex(pairs[..., 0], pairs[..., 1]) * by)
            z = z.transpose(3, 4).flatten(3) if case["layout"] == "half" else z.flatten(3)
            return torch.cat([z, x[..., r:]], 3)

        out = {"y": turn(d("x"), phase)}
        if case["grad"]:
            out["dx"] = turn(d("g"), phase.conj())
        return out
    if case["op"] == "distill":
        T, ids = case["temperature"], s["ids"]
        n, c = s["x"].shape
        log_q = torch.log_softmax(d("x") / T, 1)
        kept = (ids >= 0).double()
        full = ids.clamp(min=0)
        weight = kept * torch.exp(d("top") / T - (s["lse"].double()[:, None] if case["tail"] else 0.0))
        some = kept.sum(1) > 0
        if not case["tail"]:
            weight = weight / weight.sum(1, keepdim=True).clamp(min=1e-300)
        entropy = -torch.special.entr(weight).sum(1)
        row = entropy - (weight * log_q.gather(1, full)).sum(1)
        given = torch.zeros(n, c, dtype=torch.float64, device="cuda").scatter_add_(1, full, weight)
        grad = log_q.exp()
        if case["tail"]:
            seen = torch.zeros(n, c, dtype=torch.float64, device="cuda").scatter_add_(1, full, kept) > 0
            left = torch.where(some, (1 - weight.sum(1)).clamp(min=0), 0.0)
            mass = grad.masked_fill(seen, 0.0).sum(1)
            row = row + torch.xlogy(left, left / mass)
            grad = torch.where(seen, grad, grad * (1 - left / mass)[:, None])
        grad = torch.where(some[:, None], (grad - given) * (T / s["divisor"]), 0.0)
        row = torch.where(some, row, 0.0) * T ** 2
        return {"loss": row.sum().reshape(1) / s["divisor"], "row_loss": row, "dx": grad}
    return None  # whole numbers: the plain form's have to be met
