"""The operators of post-training a language model whose performance is
measured: the log-probabilities of chosen tokens (with the entropy of their
distributions, and the gradient), the clipped policy loss with a KL term, the
preference loss of paired sequences, and the clipping of all gradients by their
joint norm.

Each has a plain form in elementary tensor operations and, with `own`, the
framework's C-ABI calls on the same buffers. Sizes come from the benchmark's
configurations and the tests, or are generic; `draw` gives more cases of the
same ranges.
"""

from __future__ import annotations

import ctypes
import math
import random

import torch

own = False

F32 = 4
KIND = {"sigmoid": 0, "hinge": 1, "ipo": 2}
# the policy loss's setting: clipping below and above, the bound of a loss that grows with the ratio
CLIP_LOW, CLIP_HIGH, CLIP_MAX = 0.2, 0.28, 3.0


class GradSlice(ctypes.Structure):
    """oxi_grad_slice."""

    _fields_ = [("g", ctypes.c_void_p), ("out", ctypes.c_void_p), ("n", ctypes.c_int64)]


def listed():
    return [
        # the sampled tokens' log-probabilities of one decode step of 16 sequences: latency
        {"name": "logp_decode", "op": "logp", "rows": 16, "classes": 32000, "temperature": 1.0, "entropy": False,
         "grad": False, "pad": 0.0},
        # a reference model's scores of a batch of sequences (the benchmark's logits), with their entropies
        {"name": "logp_score", "op": "logp", "rows": 8192, "classes": 32000, "temperature": 1.0, "entropy": True,
         "grad": False, "pad": 0.0},
        # a loss of the user's own on log-probabilities and entropies: both directions, the odd vocabulary, padded rows
        {"name": "logp_train_odd", "op": "logp", "rows": 4096, "classes": 50257, "temperature": 0.7, "entropy": True,
         "grad": True, "pad": 0.25},
        # a small policy step without a reference model: latency
        {"name": "policy_small", "op": "policy", "rows": 64, "classes": 32000, "temperature": 1.0, "kl": 0.0,
         "entropy": 0.0, "pad": 0.0, "weights": False},
        # a policy step over the benchmark's logits with a KL term, completions padded to the longest
        {"name": "policy_large", "op": "policy", "rows": 8192, "classes": 32000, "temperature": 1.0, "kl": 0.04,
         "entropy": 0.0, "pad": 0.25, "weights": False},
        # a large vocabulary, an entropy bonus, each sequence's mean weighted alike
        {"name": "policy_vocab", "op": "policy", "rows": 1024, "classes": 131072, "temperature": 0.8, "kl": 0.01,
         "entropy": 0.003, "pad": 0.1, "weights": True},
        # two short pairs: latency
        {"name": "preference_small", "op": "preference", "pairs": 2, "longest": 32, "classes": 32000, "kind": "sigmoid",
         "average": False, "beta": 0.1, "reference": True, "prompt": 0.25},
        # a batch of pairs over the benchmark's vocabulary, up to 512 tokens a sequence
        {"name": "preference_large", "op": "preference", "pairs": 8, "longest": 512, "classes": 32000,
         "kind": "sigmoid", "average": False, "beta": 0.1, "reference": True, "prompt": 0.25},
        # the odd vocabulary, mean log-probabilities without a reference model
        {"name": "preference_odd", "op": "preference", "pairs": 6, "longest": 300, "classes": 50257, "kind": "ipo",
         "average": True, "beta": 2.0, "reference": False, "prompt": 0.25},
        # a drafting model's gradients, 2 layers: many small tensors
        {"name": "clip_small", "op": "clip", "vocab": 1003, "dim": 256, "layers": 2, "packed": False, "most": 1.0},
        # a 24-layer model's gradients, tensors of their own
        {"name": "clip_large", "op": "clip", "vocab": 50257, "dim": 1024, "layers": 24, "packed": False, "most": 1.0},
        # an odd width, views that lie back to back in one bucket
        {"name": "clip_packed_odd", "op": "clip", "vocab": 32000, "dim": 509, "layers": 8, "packed": True, "most": 1.0},
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
    op = rng.choice(["logp", "policy", "preference", "clip"])
    if op == "clip":
        return {"op": op, "vocab": _log(rng, 256, 50257), "dim": _width(rng, 16, 1024), "layers": _log(rng, 1, 16),
                "packed": rng.random() < 0.5, "most": rng.choice([0.1, 1.0, 1e6])}
    classes = _width(rng, 256, 200000)
    if op == "preference":
        longest = _log(rng, 2, 512)
        return {"op": op, "pairs": _log(rng, 1, max(1, min(64, 4096 * 32000 // (classes * longest)))), "longest": longest,
                "classes": classes, "kind": rng.choice(sorted(KIND)), "average": rng.random() < 0.5,
                "beta": rng.choice([0.1, 0.5, 2.0]), "reference": rng.random() < 0.6,
                "prompt": rng.choice([0.0, 0.25, 0.5])}
    case = {"op": op, "rows": _log(rng, 1, min(16384, 8192 * 32000 // classes)), "classes": classes,
            "temperature": rng.choice([0.7, 1.0, 1.3]), "pad": rng.choice([0.0, 0.1, 0.5])}
    if op == "logp":
        case.update(entropy=rng.random() < 0.5, grad=rng.random() < 0.6)
    else:
        case.update(kl=rng.choice([0.0, 0.04]), entropy=rng.choice([0.0, 0.003]), weights=rng.random() < 0.4)
    return case


# ---- inputs -----------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape, scale=1.0, shift=0.0):
    t = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    return t.mul_(scale).add_(shift)


def _logits(g, n, c):
    """Rows of a language model: some with many likely classes, some all but decided."""
    x = _randn(g, n, c, scale=2.0)
    best = torch.randint(0, c, (n, 1), generator=g, device="cuda")
    lift = 25.0 * torch.rand(n, 1, generator=g, device="cuda") * (torch.rand(n, 1, generator=g, device="cuda") < 0.6)
    return x.scatter_add_(1, best, lift)


def _sample(g, x, temperature):
    """A class of each row, drawn from its softmax."""
    noise = torch.empty_like(x).exponential_(generator=g).log_()
    return torch.sub(x / temperature, noise, out=noise).argmax(1)


def _padded(g, n, share):
    """True in floor(share n) rows, but never in all."""
    order = torch.randperm(n, generator=g, device="cuda")
    return order < min(n - 1, int(share * n))


def _lengths(case):
    """Tokens of each of the 2 * pairs sequences, and how many of them are the prompt's."""
    r = random.Random(case["pairs"] * 1000003 + case["longest"])
    total = [max(1, case["longest"] - r.randrange(case["longest"] // 2 + 1)) for _ in range(2 * case["pairs"])]
    total[0] = case["longest"]
    return total, [min(t - 1, int(t * case["prompt"])) for t in total]


def _shapes(case):
    d = case["dim"]
    layer = [(d,), (d, d), (d, d), (d, d), (d, d), (d,), (4 * d, d), (4 * d,), (d, 4 * d), (d,)]
    return [(case["vocab"], d)] + layer * case["layers"] + [(d,)]


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    new = lambda *shape: torch.zeros(shape, device="cuda")  # noqa: E731
    if case["op"] == "clip":
        shapes = _shapes(case)
        sizes = [math.prod(v) for v in shapes]
        room = sizes if case["packed"] else [-(-v // 128) * 128 for v in sizes]
        at = [sum(room[:i]) for i in range(len(room))]
        s["flat"], s["out"] = new(sum(room)), new(sum(room))
        s["g"] = [s["flat"][a:a + n] for a, n in zip(at, sizes)]
        s["o"] = [s["out"][a:a + n] for a, n in zip(at, sizes)]
        for i, v in enumerate(s["g"]):  # gradients of different layers differ in size
            v.normal_(generator=g).mul_(1e-3 * (1 + i % 7))
        s["slices"] = (GradSlice * len(sizes))(*[GradSlice(v.data_ptr(), o.data_ptr(), v.numel())
                                                 for v, o in zip(s["g"], s["o"])])
        s["total"] = torch.zeros(1, dtype=torch.float64, device="cuda")
    elif case["op"] == "preference":
        total, prompt = _lengths(case)
        n, c = sum(total), case["classes"]
        s["x"] = _logits(g, n, c)
        s["ids"] = _sample(g, s["x"], 1.0)
        starts = torch.tensor([sum(total[:i]) for i in range(len(total) + 1)], dtype=torch.int64)
        s["sequence"] = torch.repeat_interleave(torch.arange(len(total)), torch.tensor(total)).cuda()
        s["starts"] = starts.cuda()
        within = torch.arange(n, device="cuda") - s["starts"][s["sequence"]]
        s["ids"] = torch.where(within < torch.tensor(prompt).cuda()[s["sequence"]], -1, s["ids"])
        s["ref"] = None
        if case["reference"]:
            s["ref"] = (_rows(s["x"], s["ids"], 1.0, False)["logp"] + _randn(g, n, scale=0.1)).float().clamp_(max=0.0)
        p = case["pairs"]
        s.update(loss=new(1), pair_loss=new(p), seq_logp=new(2 * p), coef=new(n), saved=new(n, 4), dx=new(n, c))
    else:
        n, c = case["rows"], case["classes"]
        s["x"] = _logits(g, n, c)
        s["ids"] = torch.where(_padded(g, n, case["pad"]), -1, _sample(g, s["x"], case["temperature"]))
        s.update(logp=new(n), saved=new(n, 4))
        if case["op"] == "logp":
            s["entropy"] = new(n) if case["entropy"] else None
            if case["grad"]:
                s.update(gl=_randn(g, n), ge=_randn(g, n, scale=0.1) if case["entropy"] else None, dx=new(n, c))
        else:
            there = s["ids"] >= 0
            moved = _randn(g, n, scale=0.15)  # how far the policy has moved since it sampled
            for edge in (1 - CLIP_LOW, 1 + CLIP_HIGH, CLIP_MAX):
                # a ratio on an edge of the clipping belongs to either side
                moved = torch.where((moved.exp() - edge).abs() < 1e-4, moved + 5e-4, moved)
            logp = _rows(s["x"], s["ids"], case["temperature"], False)["logp"]
            s["old"] = (logp - moved).float()
            s["ref"] = (logp + _randn(g, n, scale=0.2)).float() if case["kl"] else None
            s["adv"] = _randn(g, n) * (torch.rand(n, generator=g, device="cuda") >= 0.05)
            s["weights"], s["divisor"] = None, float(max(1, int(there.sum())))
            if case["weights"]:  # sequences of 16 tokens: each token by its sequence's count
                part = torch.arange(n, device="cuda") // 16
                count = torch.zeros(n, device="cuda").scatter_add_(0, part, there.float())
                s["weights"] = 1.0 / count[part].clamp(min=1.0)
                s["divisor"] = float(-(-n // 16))
            s.update(out=new(4), rows=new(4, n), coef=new(2, n), dx=new(n, c))
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


def _own_logp(s, case):
    from oxitorch_amd import capi

    n, c = s["x"].shape
    # without a backward to come nothing is saved for it, as in F.token_log_probs under no_grad
    capi.call("oxi_token_logp_fwd", _ptr(s["x"]), _ptr(s["ids"]), _ptr(s["logp"]), _ptr(s["entropy"]),
              _ptr(s["saved"]) if case["grad"] else None, None, n, c, case["temperature"])
    out = {"logp": s["logp"], "entropy": s["entropy"]}
    if case["grad"]:
        capi.call("oxi_token_logp_bwd", _ptr(s["x"]), _ptr(s["ids"]), _ptr(s["saved"]), _ptr(s["gl"]), _ptr(s["ge"]),
                  None, _ptr(s["dx"]), n, c, case["temperature"])
        out["dx"] = s["dx"]
    return out


def _own_policy(s, case):
    from oxitorch_amd import capi

    n, c = s["x"].shape
    capi.call("oxi_policy_loss_fwd", _ptr(s["x"]), _ptr(s["ids"]), _ptr(s["adv"]), _ptr(s["old"]), _ptr(s["ref"]),
              _ptr(s["weights"]), _ptr(s["out"]), _ptr(s["rows"]), _ptr(s["logp"]), _ptr(s["coef"]), _ptr(s["saved"]),
              _ptr(s["dx"]), None, n, c, case["temperature"], CLIP_LOW, CLIP_HIGH, CLIP_MAX, case["kl"],
              case["entropy"], s["divisor"])
    return {"out": s["out"], "rows": s["rows"], "logp": s["logp"], "dx": s["dx"]}


def _own_preference(s, case):
    from oxitorch_amd import capi

    n, c = s["x"].shape
    capi.call("oxi_preference_loss_fwd", _ptr(s["x"]), _ptr(s["ids"]), _ptr(s["starts"]), _ptr(s["ref"]),
              _ptr(s["loss"]), _ptr(s["pair_loss"]), _ptr(s["seq_logp"]), _ptr(s["coef"]), _ptr(s["saved"]),
              _ptr(s["dx"]), None, n, c, case["pairs"], KIND[case["kind"]], int(case["average"]), case["beta"], 0.0, 0.0)
    return {"loss": s["loss"], "pair_loss": s["pair_loss"], "seq_logp": s["seq_logp"], "dx": s["dx"]}


def _own_clip(s, case):
    from oxitorch_amd import capi

    count = len(s["slices"])
    capi.call("oxi_grad_norm", s["slices"], count, 2.0, _ptr(s["total"]), None)
    capi.call("oxi_grad_clip", s["slices"], count, _ptr(s["total"]), case["most"])
    return {"total": s["total"], "out": s["out"]}


_OWN = {"logp": _own_logp, "policy": _own_policy, "preference": _own_preference, "clip": _own_clip}


def _rows(x, ids, temperature, entropy):
    """Of each row the exponentials e relative to its maximum and their sum, the chosen token's log-probability
    (64 bits; 0 in padded rows) and the entropy."""
    there = ids >= 0
    m = x.amax(1, keepdim=True)
    z = (x - m) / temperature
    e = torch.exp(z)
    total = e.sum(1, dtype=torch.float64)
    at = ids.clamp(min=0)[:, None]
    logp = (x.gather(1, at).double() - m)[:, 0] / temperature - torch.log(total)
    out = {"e": e, "z": z, "total": total, "logp": torch.where(there, logp, 0.0)}
    if entropy:
        out["entropy"] = torch.where(there, torch.log(total) - (e * z).sum(1, dtype=torch.float64) / total, 0.0)
    return out


def _gradient(r, ids, temperature, gl, ge=None):
    """d logits for the gradients gl of the log-probabilities and ge of the entropies."""
    there = (ids >= 0)[:, None]
    q = r["e"] / r["total"][:, None].float()
    d = q * -gl[:, None]
    if ge is not None:
        off = (r["entropy"] - torch.log(r["total"]))[:, None].float()
        d = d - ge[:, None] * q * (r["z"] + off)
    d = d.scatter_add(1, ids.clamp(min=0)[:, None], gl[:, None])
    return torch.where(there, d / temperature, 0.0)


def _plain_logp(s, case):
    r = _rows(s["x"], s["ids"], case["temperature"], case["entropy"])
    out = {"logp": r["logp"].float(), "entropy": r["entropy"].float() if case["entropy"] else None}
    if case["grad"]:
        out["dx"] = _gradient(r, s["ids"], case["temperature"], s["gl"], s["ge"])
    return out


def _plain_policy(s, case):
    there = s["ids"] >= 0
    r = _rows(s["x"], s["ids"], case["temperature"], True)
    a = s["adv"].double()
    ratio = torch.exp(r["logp"] - s["old"].double())
    free, bounded = ratio * a, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * a
    surrogate = torch.minimum(free, bounded)
    floor = torch.where(a < 0, CLIP_MAX * a, -math.inf)
    clipped = (free > bounded) | (surrogate < floor)
    surrogate = torch.maximum(surrogate, floor)
    gl = torch.where(clipped, 0.0, -free)
    kl = torch.zeros_like(a)
    if case["kl"]:
        d = s["ref"].double() - r["logp"]
        kl = torch.expm1(d) - d
        gl = gl - case["kl"] * torch.expm1(d)
    row = case["kl"] * kl - surrogate - case["entropy"] * r["entropy"]
    w = there.double() / s["divisor"]
    if s["weights"] is not None:
        w = w * s["weights"].double()
    rows = torch.stack([row, kl, r["entropy"], clipped.double()])
    rows = torch.where(there, rows, 0.0)
    ge = (-case["entropy"] * w).float() if case["entropy"] else None
    return {"out": (rows * w).sum(1).float(), "rows": rows.float(), "logp": r["logp"].float(),
            "dx": _gradient(r, s["ids"], case["temperature"], (gl * w).float(), ge)}


def _plain_preference(s, case):
    there = s["ids"] >= 0
    r = _rows(s["x"], s["ids"], 1.0, False)
    p = case["pairs"]
    zero = torch.zeros(2 * p, dtype=torch.float64, device="cuda")
    count = zero.scatter_add(0, s["sequence"], there.double()).clamp_(min=1.0)
    share = 1.0 / count if case["average"] else torch.ones_like(count)
    total = zero.scatter_add(0, s["sequence"], r["logp"]) * share
    u = total.clone()
    if s["ref"] is not None:
        u = u - zero.scatter_add(0, s["sequence"], torch.where(there, s["ref"], 0.0).double()) * share
    h = u[0::2] - u[1::2]
    b = case["beta"]
    if case["kind"] == "sigmoid":
        t = torch.exp(-torch.abs(b * h))
        loss = torch.clamp(-b * h, min=0.0) + torch.log1p(t)
        slope = -b * torch.where(h > 0, t, 1.0) / (1.0 + t)
    elif case["kind"] == "hinge":
        loss = torch.clamp(1.0 - b * h, min=0.0)
        slope = torch.where(b * h < 1.0, -b, 0.0)
    else:
        d = h - 1.0 / (2.0 * b)
        loss, slope = d * d, 2.0 * d
    per = torch.stack([slope, -slope], 1).reshape(-1) * share / p
    return {"loss": loss.mean().float().reshape(1), "pair_loss": loss.float(), "seq_logp": total.float(),
            "dx": _gradient(r, s["ids"], 1.0, per[s["sequence"]].float())}


def _plain_clip(s, case):
    total = torch.sqrt(torch.stack([v.double().square().sum() for v in s["g"]]).sum())
    scale = (case["most"] / (total + 1e-6)).clamp(max=1.0).float()
    [torch.mul(v, scale, out=o) for v, o in zip(s["g"], s["o"])]
    return {"total": total.reshape(1), "out": s["out"]}


_PLAIN = {"logp": _plain_logp, "policy": _plain_policy, "preference": _plain_preference, "clip": _plain_clip}


# ---- what a pass cannot do without -----------------------------------------------

def work(case):
    """Each input that the pass depends on read once, each output written once. Padded rows' logits are not needed."""
    if case["op"] == "clip":
        n = sum(math.prod(v) for v in _shapes(case))
        return {"bytes": 2 * n * F32, "flops": 3 * n}
    c = case["classes"]
    if case["op"] == "preference":
        total, prompt = _lengths(case)
        n, used, grad, more = sum(total), sum(total) - sum(prompt), True, 12
    else:
        n = case["rows"]
        used, grad, more = n - min(n - 1, int(case["pad"] * n)), case.get("grad", True), 24
    # a product and an exponential for each class, again for its gradient
    return {"bytes": (used + (n if grad else 0)) * c * F32 + more * n, "flops": used * c * (8 if grad else 4)}


# ---- the same in 64 bits -----------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(v, dtype=torch.float64) for v in s["g"]]))
        factor = min(1.0, case["most"] / (float(norm) + 1e-6))
        return {"total": norm.reshape(1), "out": s["flat"].double() * factor}
    x = s["x"].double().requires_grad_()
    rows = torch.nonzero(s["ids"] >= 0)[:, 0]
    n = x.shape[0]
    temperature = case.get("temperature", 1.0)
    logs = torch.log_softmax(x[rows] / temperature, 1)
    some = logs.gather(1, s["ids"][rows][:, None])[:, 0]
    full = lambda v: torch.zeros(n, dtype=torch.float64, device="cuda").index_put((rows,), v)  # noqa: E731
    wants_entropy = bool(case.get("entropy"))
    if wants_entropy or case["op"] == "policy":
        entropy = -(logs.exp() * logs).sum(1)
    if case["op"] == "logp":
        out = {"logp": full(some).detach(), "entropy": full(entropy).detach() if wants_entropy else None}
        if case["grad"]:
            up = (some * s["gl"][rows]).sum()
            if wants_entropy:
                up = up + (entropy * s["ge"][rows]).sum()
            out["dx"] = torch.autograd.grad(up, x)[0]
        return out
    if case["op"] == "policy":
        adv = s["adv"][rows].double()
        ratio = (some - s["old"][rows]).exp()
        ppo = torch.where(adv >= 0, torch.clamp(ratio, max=1 + CLIP_HIGH),
                          torch.clamp(torch.clamp(ratio, min=1 - CLIP_LOW), max=CLIP_MAX)) * adv
        hit = torch.where(adv > 0, ratio > 1 + CLIP_HIGH, (adv < 0) & ((ratio < 1 - CLIP_LOW) | (ratio > CLIP_MAX)))
        gap = s["ref"][rows] - some if case["kl"] else torch.zeros_like(some)
        kl = gap.exp() - 1 - gap
        row = -ppo + case["kl"] * kl - case["entropy"] * entropy
        w = torch.full_like(row, 1 / s["divisor"]) if s["weights"] is None else s["weights"][rows].double() / s["divisor"]
        table = [row, kl, entropy, hit.double()]
        dx = torch.autograd.grad((row * w).sum(), x)[0]
        return {"out": torch.stack([(v * w).sum() for v in table]).detach(),
                "rows": torch.stack([full(v) for v in table]).detach(), "logp": full(some).detach(), "dx": dx}
    sides, both = [], []
    for q in range(2 * case["pairs"]):
        mine = s["sequence"][rows] == q
        size = max(1, int(mine.sum())) if case["average"] else 1
        both.append(some[mine].sum() / size)
        sides.append(both[-1] - (s["ref"][rows][mine].double().sum() / size if s["ref"] is not None else 0.0))
    margin = torch.stack(sides[0::2]) - torch.stack(sides[1::2])
    b = case["beta"]
    each = {"sigmoid": lambda: -torch.nn.functional.logsigmoid(b * margin), "hinge": lambda: torch.relu(1 - b * margin),
            "ipo": lambda: (margin - 0.5 / b) ** 2}[case["kind"]]()
    return {"loss": each.mean().detach().reshape(1), "pair_loss": each.detach(), "seq_logp": torch.stack(both).detach(),
            "dx": torch.autograd.grad(each.mean(), x)[0]}
