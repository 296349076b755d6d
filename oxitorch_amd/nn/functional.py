"""Functional API of the hot path, same signatures as the reference
python/oxitorch/nn/functional.py:182-293.

Where the reference composes each F.* from several graph ops, this module
calls one fused device node (one kernel forward, one kernel backward), whose
values and gradients match the composition within the parity tolerances.
Inputs the fused nodes do not take (a weight that is not a (H,) vector,
for instance) fall back to the reference's composition of graph ops, still
on the device.
"""

from __future__ import annotations

import numpy as np

from .. import _native


def _native_from_numpy(arr, requires_grad=False):
    """Build a graph-connected tensor from a numpy array (default device)."""
    return _native.from_numpy(np.ascontiguousarray(arr, dtype=np.float32), requires_grad)


# ---- activations (functional.py:182-208) ---------------------------------------

def relu(x):
    return x.apply("relu")


def sigmoid(x):
    return x.apply("sigmoid")


def tanh(x):
    return x.apply("tanh")


def gelu(x, approximate="tanh"):
    """GELU. `approximate='tanh'` is the reference's F.gelu
    0.5 x (1 + tanh(sqrt(2/pi) (x + 0.044715 x^3))); `'none'` is the exact
    0.5 x (1 + erf(x / sqrt 2)), which the reference does not have."""
    return _native.gelu(x, approximate)


def silu(x):
    """Sigmoid-weighted linear unit, elementwise: each value times its own
    logistic sigmoid. One device node with its VJP."""
    return _native.silu(x)


def leaky_relu(x, negative_slope=0.01):
    return x.apply("relu") + (x * float(negative_slope)).apply("neg").apply("relu").apply("neg")


# ---- softmax family (functional.py:211-222) -------------------------------------

def softmax(x, dim=-1):
    """Probabilities along `dim`: exponentials of x shifted by the largest
    value of its slice (so no exponential overflows), divided by their sum.
    One device node; the reference composes it from max, exp and sum nodes."""
    return _native.softmax(x, dim)


def log_softmax(x, dim=-1):
    """Log-probabilities along `dim`: x shifted by its slice maximum, minus the
    log of the shifted exponentials' sum. One device node."""
    return _native.log_softmax(x, dim)


# ---- normalization (functional.py:227-240) ----------------------------------------

def _flat_ints(values, what):
    """A flat int64 array of `values` (numbers in any nesting), refusing what is not an integer."""
    a = np.asarray(values)
    if a.size and a.dtype.kind not in "iu":
        raise TypeError(f"{what} must be integers, got {a.dtype}")
    if a.dtype == np.uint64 and a.size and a.max() > np.iinfo(np.int64).max:
        raise OverflowError(f"{what}: {a.max()} does not fit in 64 signed bits")
    return a.astype(np.int64).ravel()


def _is_vec(t, H):
    return t is not None and len(t.shape) == 1 and t.shape[0] == H


def layer_norm(x, weight, bias, eps=1e-5, vjp=None):
    """Normalizes each last-dim row to zero mean and unit variance (eps added
    to the variance), then scales by `weight` and shifts by `bias`.

    `vjp` selects the x-gradient: "ref" (default, or OXI_NORM_VJP) reproduces
    the reference graph, where `.apply("rsqrt")` detaches the inverse std;
    "exact" is the full derivative.

    When the output feeds only a gelu, silu, or last-dim softmax/log_softmax,
    backward runs both VJPs as one device pass (the same values, bit for bit;
    OXI_FUSE_NORM_ACT=0 turns it off)."""
    H = x.shape[-1]
    if _is_vec(weight, H) and _is_vec(bias, H):
        return _native.layer_norm(x, weight, bias, eps, vjp)
    mu = x.mean(-1, True)
    centered = x - mu
    var = (centered * centered).mean(-1, True)
    inv = (var + float(eps)).apply("rsqrt")
    return centered * inv * weight + bias


def rms_norm(x, weight, eps=1e-6, vjp=None):
    """Divides each last-dim row by its root mean square (eps added to the mean
    square) and scales by `weight`; `vjp` as in layer_norm."""
    if _is_vec(weight, x.shape[-1]):
        return _native.rms_norm(x, weight, eps, vjp)
    ms = (x * x).mean(-1, True)
    inv = (ms + float(eps)).apply("rsqrt")
    return x * inv * weight


def add_rms_norm(x, residual, weight, eps=1e-6, vjp=None):
    """The residual stream's step of a pre-norm layer: h = x + residual and
    y = rms_norm(h, weight, eps) in one pass. Returns (y, h): y goes into the
    layer, h on along the stream. `vjp` as in layer_norm.

    In backward, the gradient that h has from its later uses joins the norm's
    in one pass (OXI_FUSE_NORM_ACT=0 runs the add by itself)."""
    if list(residual.shape) == list(x.shape) and _is_vec(weight, x.shape[-1]):
        return _native.add_rms_norm(x, residual, weight, eps, vjp)
    h = x + residual
    return rms_norm(h, weight, eps, vjp), h


def add_rms_norm_e4m3(x, residual, weight, eps=1e-6, group=128):
    """add_rms_norm for serving, with y in 8-bit floating point (OCP e4m3) and a
    scale for each `group` columns of a row (32, 64, 128, 256 or the row's
    length): max|y|/448 of the group. Returns (q, h); q holds `codes()` (numpy
    uint8), `scale` and `dequantize()`, and carries no gradient. `residual` None:
    the norm of x alone, and h is None."""
    return _native.add_rms_norm_e4m3(x, residual, weight, eps, group)


# ---- rotary positions -----------------------------------------------------------------

def rotary_frequencies(dim, base=10000.0, scaling=None):
    """(inv_freq, scale): the angle per position of each of the dim/2 pairs,
    base**(-2i/dim), as float64, and the factor on what they turn.

    `scaling` stretches them for contexts longer than the trained one:
    {"type": "linear", "factor": s} divides all of them by s;
    {"type": "ntk", "factor": s} raises the base to base * s**(dim/(dim-2)), so
    that the slowest pair is divided by s and the fastest is kept;
    {"type": "yarn", "factor": s, "original_length": L} divides the pairs that
    turn less than `slow` (1) times within L positions by s, keeps those that
    turn more than `fast` (32) times, and blends in between; its scale is
    0.1 ln(s) + 1 ("scale" overrides)."""
    dim = int(dim)
    if dim < 0 or dim % 2:
        raise ValueError(f"rotary positions turn pairs: {dim} elements is not an even number")
    base = float(base)
    if not base > 0 or np.isinf(base):
        raise ValueError(f"the rotary base must be positive, got {base}")
    half = dim // 2
    exponent = -np.arange(half, dtype=np.float64) / max(half, 1)
    inv = base ** exponent
    if scaling is None:
        return inv, 1.0
    kind, s = scaling.get("type"), float(scaling.get("factor", 1.0))
    if not s > 0 or np.isinf(s):
        raise ValueError(f"the rotary scaling factor must be positive, got {s}")
    if kind == "linear":
        return inv / s, 1.0
    if kind == "ntk":
        if dim <= 2:
            return inv, 1.0
        return (base * s ** (dim / (dim - 2))) ** exponent, 1.0
    if kind == "yarn":
        length = float(scaling["original_length"])
        slow, fast = float(scaling.get("slow", 1.0)), float(scaling.get("fast", 32.0))
        if not fast > slow:
            raise ValueError(f"rotary scaling: fast ({fast}) must be above slow ({slow})")
        keep = np.clip((length * inv / (2 * np.pi) - slow) / (fast - slow), 0.0, 1.0)
        scale = scaling.get("scale", 0.1 * np.log(s) + 1.0 if s > 1 else 1.0)
        return (1 - keep) * inv / s + keep * inv, float(scale)
    raise ValueError(f"unknown rotary scaling {kind!r}: linear, ntk or yarn")


def _frequencies(f):
    if isinstance(f, _native.RotaryFrequencies):
        return f
    pair = isinstance(f, tuple) and len(f) == 2 and np.ndim(f[0]) > 0  # what rotary_frequencies returns
    inv, scale = f if pair else (f, 1.0)
    return _native.RotaryFrequencies([float(v) for v in np.asarray(inv, dtype=np.float64).ravel()], scale)


def rotary_embedding(x, frequencies, positions=None, offset=0, layout="half"):
    """x (batch, tokens, heads, dim) or (tokens, heads, dim) with the pairs of
    each head's first elements turned by position * frequency: (u, v) to
    scale * (u cos a - v sin a, v cos a + u sin a); elements past the pairs are
    copied. Pair i is elements (i, i + pairs) in the "half" layout,
    (2i, 2i + 1) in the "interleaved" one.

    `frequencies`: what rotary_frequencies returns, an array of angles per
    position, or a _native.RotaryFrequencies that holds them on the device (as
    nn.RotaryEmbedding keeps one). `positions`: integers, one per token or (batch,
    tokens), one per batch and token; None counts from 0. `offset` is added to them. Angles
    are formed in 64 bits. x may be any view (heads before tokens, a slice of a
    fused projection); one call serves query and key heads side by side."""
    if positions is not None:
        given, each = list(np.shape(positions)), list(x.shape[:-2])
        long = [d for d in given if d != 1]  # an order other than (batch, tokens) shows in these
        if len(long) > 1 and long != [d for d in each if d != 1]:
            raise ValueError(f"positions of shape {given} for tokens of shape {each}")
        positions = _flat_ints(positions, "positions")
    if int(offset) != offset:
        raise TypeError(f"offset must be an integer, got {offset}")
    return _native.rotary_embedding(x, _frequencies(frequencies), positions, int(offset), layout)


# ---- embedding (functional.py:245-247) -----------------------------------------------

def embedding(indices, weight):
    """Rows of the `(num_embeddings, dim)` table `weight` picked by `indices`:
    a flat sequence of ints as the reference takes them, or a numpy integer
    array of any shape (read in C order)."""
    if isinstance(indices, np.ndarray):
        indices = indices.ravel()
    return _native.embedding(indices, weight)


# ---- losses (functional.py:270-293) -----------------------------------------------------

def mse_loss(pred, target):
    diff = pred - target
    return (diff * diff).mean()


def cross_entropy(logits, targets):
    """Mean cross-entropy; `targets` is a flat list of int class indices.

    Fused: the forward reads each row once (its log-sum-exp and picked
    log-probability, NaN where the reference's sum(onehot * log_softmax)
    is); when the logits require grad it also writes the gradient that
    backward() with its implicit seed of 1 hands them, and any other
    upstream gradient g runs one backward pass writing
    (softmax - onehot) * g / n. The argument checks mirror the reference's: a batch-size mismatch raises
    ValueError mentioning the targets, and class ids follow numpy indexing
    (negatives wrap, out-of-range raises IndexError)."""
    n, classes = logits.shape
    t = np.asarray(targets)
    if t.size and t.dtype.kind not in "iu":
        # the reference indexes its one-hot with them (functional.py:288-289)
        if isinstance(targets, np.ndarray):
            raise IndexError("arrays used as indices must be of integer (or boolean) type")
        raise IndexError("only integers, slices (`:`), ellipsis (`...`), numpy.newaxis (`None`) and integer or "
                         "boolean arrays are valid indices")
    t = t.astype(np.int64).ravel()
    if len(t) != n:
        raise ValueError(f"{len(t)} targets for batch of {n}")
    bad = (t >= classes) | (t < -classes)
    if bad.any():
        raise IndexError(f"index {int(t[bad][0])} is out of bounds for axis 1 with size {classes}")
    t = np.where(t < 0, t + classes, t)
    return _native.cross_entropy(logits, t)


def _device_values(v):
    """A tensor as it is, anything else as a float32 tensor on the default device."""
    return v if isinstance(v, _native.Tensor) else _native_from_numpy(np.asarray(v, dtype=np.float32))


def distillation_loss(logits, teacher_ids, teacher_logits, temperature=1.0, teacher_lse=None):
    """How far a student's distribution q = softmax(logits/T) is from a
    teacher's that is known by its k best entries a row: T^2 times the mean over
    the rows of sum p (log p - log q[id]).

    `teacher_ids` (batch, k): the entries' classes as integers;
    `teacher_logits` (batch, k): the teacher's logits there, a tensor or an array; no
    gradient goes to them. An entry with a negative id or a logit of -inf is padding,
    and rows of padding alone (padded tokens) count neither in the sum nor in the
    mean. p is their softmax at
    temperature T over the row's entries; with `teacher_lse` (batch: the
    log-sum-exp of all of the teacher's logits/T) p are the teacher's own
    probabilities, and what they leave to the other classes is compared with
    what the student leaves there. The gradient takes them to sum to at most 1, as
    they do where teacher_lse is the teacher's at T.

    Fused as cross_entropy is: one pass over the logits writes the loss and the
    gradient for backward()'s implicit seed."""
    n, classes = logits.shape
    ids = np.asarray(teacher_ids)
    if ids.ndim != 2 or ids.shape[0] != n:
        raise ValueError(f"teacher_ids of shape {list(ids.shape)} for a batch of {n}: (batch, k) is expected")
    flat = _flat_ints(ids, "teacher_ids")
    if flat.size and flat.max() >= classes:
        raise IndexError(f"index {int(flat.max())} is out of bounds for axis 1 with size {classes}")
    top = _device_values(teacher_logits)
    if list(top.shape) != list(ids.shape):
        raise ValueError(f"teacher_logits of shape {list(top.shape)} for teacher_ids of shape {list(ids.shape)}")
    lse = None if teacher_lse is None else _device_values(teacher_lse)
    return _native.distillation_loss(logits, flat, top, lse, float(temperature))


# ---- post-training losses ---------------------------------------------------------------

def _tokens(tokens, n, classes):
    """One class a row as a flat int64 array; negative ones are padding."""
    t = _flat_ints(tokens, "tokens")
    if len(t) != n:
        raise ValueError(f"{len(t)} tokens for batch of {n}")
    if t.size and t.max() >= classes:
        raise IndexError(f"index {int(t.max())} is out of bounds for axis 1 with size {classes}")
    return t


def _optional_values(v):
    return None if v is None else _device_values(v)


def token_log_probs(logits, tokens, temperature=1.0, entropy=False):
    """Log-probabilities (batch,) of one token a row under softmax(logits/T); with
    `entropy` (log-probabilities, entropies of the rows' distributions).

    `tokens`: flat integers; a negative one is padding, whose row is not read and
    gives 0. Under no_grad what policy_loss and preference_loss take as the old
    policy's or the reference's; with gradients the base of losses of one's own: both
    results' gradients go back in one pass. The log-probability of a token that is all
    but certain keeps its digits, and so does the gradient at it."""
    n, classes = logits.shape
    both = _native.token_log_probs(logits, _tokens(tokens, n, classes), float(temperature), bool(entropy))
    return (both.select(0, 0), both.select(0, 1)) if entropy else both


def policy_loss(logits, tokens, advantages, old_log_probs=None, reference_log_probs=None, weights=None, clip=0.2,
                clip_max=None, kl=0.0, entropy=0.0, temperature=1.0, stats=False):
    """The clipped policy loss of sampled tokens, with a KL term against a reference
    policy and an entropy bonus: the mean over the rows of

        -min(r A, clip(r, 1 - clip, 1 + clip) A) + kl (exp(d) - 1 - d) - entropy H

    with r = exp(logp - old_log_probs), d = reference_log_probs - logp, H the entropy of
    the row's distribution, logp as in token_log_probs, A = `advantages`.

    `tokens`: flat integers, a negative one is padding. `advantages`,
    `old_log_probs`, `reference_log_probs`, `weights`: tensors or arrays, one number a row,
    that no gradient goes to. Without old_log_probs r is 1 (the first step after
    sampling). `clip`: a number or (below, above); `clip_max` bounds the loss of a negative
    advantage at clip_max |A|. With `weights` the loss is the sum of weight * row
    instead of the mean, and rows of weight 0 are padding (a mean by sequences: 1 / (its
    tokens * sequences)). With `stats`, (loss, (3,) tensor of the same means of the KL
    term's exp(d) - 1 - d, H and whether r was clipped).

    A row with no finite logit, or with NaN, gives NaN in the loss and in its gradient,
    whatever its advantage.

    Fused as cross_entropy is: one pass over the logits writes the loss and the
    gradient for backward()'s implicit seed."""
    n, classes = logits.shape
    t = _tokens(tokens, n, classes)
    low, high = clip if isinstance(clip, (tuple, list)) else (clip, clip)
    divisor = 1.0 if weights is not None else float(max(1, int((t >= 0).sum())))
    loss, more = _native.policy_loss(logits, t, _device_values(advantages), _optional_values(old_log_probs),
                                     _optional_values(reference_log_probs), _optional_values(weights),
                                     float(temperature), float(low), float(high),
                                     0.0 if clip_max is None else float(clip_max), float(kl), float(entropy), divisor)
    return (loss, more) if stats else loss


def preference_loss(logits, tokens, lengths, reference_log_probs=None, beta=0.1, kind="sigmoid", margin=0.0,
                    smoothing=0.0, average=False, details=False):
    """The preference loss of pairs of sequences: the mean over the pairs of

        "sigmoid": (1 - smoothing) softplus(-u) + smoothing softplus(u)
        "hinge":   max(0, 1 - u)
        "ipo":     (u/beta - 1/(2 beta))^2

    with u = beta ((S_c - R_c) - (S_r - R_r)) - margin, S the sum of the sequence's tokens'
    log-probabilities and R that of `reference_log_probs` (one number a row; None: 0), or
    with `average` their means.

    `lengths` (pairs, 2): the rows of each pair's chosen and rejected sequence, which lie
    one after the other in `logits` (rows, classes). `tokens`: flat integers, a negative
    one (the prompt's) does not count; rows behind the last sequence are padding. With
    `details`, (loss, the pairs' losses, (pairs, 2) S).

    The logits are read twice, the second time for the gradient of backward()'s
    implicit seed, which the forward writes as cross_entropy does."""
    n, classes = logits.shape
    t = _tokens(tokens, n, classes)
    given = np.asarray(lengths)
    if given.size and (given.ndim != 2 or given.shape[1] != 2):
        raise ValueError(f"lengths of shape {list(given.shape)}: (pairs, 2) is expected")
    loss, pair, seq = _native.preference_loss(logits, t, _flat_ints(given, "lengths"),
                                              _optional_values(reference_log_probs), kind, bool(average), float(beta),
                                              float(margin), float(smoothing))
    return (loss, pair, seq) if details else loss


# ---- serving: drafted tokens ------------------------------------------------------------

def _uniforms(u):
    """Numbers in [0, 1) as float32: a tensor as it is; those of an array, checked, and kept below 1 where their
    rounding reaches it."""
    if isinstance(u, _native.Tensor):
        return u
    a = np.asarray(u)
    if not ((a >= 0) & (a < 1)).all():
        raise ValueError("uniforms must lie in [0, 1)")
    return _native_from_numpy(np.minimum(a.astype(np.float32), np.float32(1 - 2.0 ** -24)))


def verify_drafts(draft_tokens, draft_probs, target_probs, uniforms, lengths=None):
    """Which of the tokens that a small model drafted are kept, so that what is
    kept is distributed as the large model's own samples.

    `draft_tokens` (batch, k) integers; `draft_probs` (batch, k, classes): what
    each was drawn from, or None for drafts without probabilities (a lookup, a
    greedy model); `target_probs` (batch, k + 1, classes): the large model's,
    after 0, 1, .. k of them; `uniforms` (batch, k + 1) in [0, 1), a tensor or an
    array (in a tensor's, 1 draws the last class with weight); `lengths` (batch): how many tokens were drafted, None for k.

    Draft i is kept while uniforms[i] * draft_probs[i][token] <
    target_probs[i][token]; after the first that is not, one token is drawn from
    max(target - draft, 0) by uniforms[k], after all of them from the target's
    next row. Returns numpy int64 arrays (accepted (batch,), tokens (batch,
    k + 1)): the kept tokens, the drawn one, then -1. Waits for the device."""
    tokens = np.asarray(draft_tokens)
    b, rows, classes = target_probs.shape
    if tokens.shape != (b, rows - 1):
        raise ValueError(f"draft_tokens of shape {list(tokens.shape)} for target_probs of shape "
                         f"{list(target_probs.shape)}: {[b, rows - 1]} is expected")
    flat = _flat_ints(tokens, "draft_tokens")
    if lengths is not None:
        lengths = _flat_ints(lengths, "lengths")
    return _native.verify_drafts(flat, draft_probs, target_probs, _uniforms(uniforms), lengths)


def _outside(what):
    def op(*args, **kwargs):
        raise NotImplementedError(f"{what} is outside this build's device hot path")
    op.__name__ = what.split(" ")[0]
    op.__doc__ = f"The reference's {what}: not part of this build; raises NotImplementedError."
    return op


# The reference's GEMM, convolution, pooling and dropout entry points
# (functional.py:23-47,49-55,104-148,150-181,255-268) are outside the device
# hot path; calling one says so instead of failing on a missing name.
linear = _outside("linear (SGEMM)")
bmm = _outside("bmm (batched GEMM)")
conv2d = _outside("conv2d (im2col + GEMM)")
max_pool2d = _outside("max_pool2d")
dropout = _outside("dropout")
