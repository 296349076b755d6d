"""oxitorch_amd.nn: the hot-path subset of the reference `oxitorch.nn`
(python/oxitorch/nn/__init__.py): functional norms, activations, softmax
family, cross-entropy and embedding, plus their Module wrappers; and the
operators of language models around them that the reference does not have
(residual RMS norm, rotary positions, distillation, draft verification, token
log-probabilities, policy and preference losses)."""

from .module import Module, Parameter, Sequential
from . import functional
from .functional import (
    add_rms_norm,
    add_rms_norm_e4m3,
    cross_entropy,
    distillation_loss,
    embedding,
    gelu,
    layer_norm,
    leaky_relu,
    log_softmax,
    mse_loss,
    policy_loss,
    preference_loss,
    relu,
    rms_norm,
    rotary_embedding,
    rotary_frequencies,
    sigmoid,
    silu,
    softmax,
    tanh,
    token_log_probs,
    verify_drafts,
)
from .layers import (
    GELU,
    AddRMSNorm,
    Embedding,
    LayerNorm,
    LeakyReLU,
    ReLU,
    RMSNorm,
    RotaryEmbedding,
    SiLU,
    Sigmoid,
    Softmax,
    Tanh,
)
# outside the device hot path: each raises NotImplementedError when called
from .functional import bmm, conv2d, dropout, linear, max_pool2d
from .layers import Conv2d, Dropout, Linear, MaxPool2d

__all__ = [
    "Module", "Parameter", "Sequential", "functional", "cross_entropy", "embedding", "gelu", "layer_norm",
    "leaky_relu", "log_softmax", "mse_loss", "relu", "rms_norm", "sigmoid", "silu", "softmax", "tanh",
    "GELU", "Embedding", "LayerNorm", "LeakyReLU", "ReLU", "RMSNorm", "SiLU", "Sigmoid", "Softmax", "Tanh",
    "add_rms_norm", "add_rms_norm_e4m3", "distillation_loss", "rotary_embedding", "rotary_frequencies", "verify_drafts",
    "policy_loss", "preference_loss", "token_log_probs",
    "AddRMSNorm", "RotaryEmbedding",
    "bmm", "conv2d", "dropout", "linear", "max_pool2d", "Conv2d", "Dropout", "Linear", "MaxPool2d",
]
