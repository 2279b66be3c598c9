"""The operators between a CG network's invariant embedding and its answers, and the classifier head built from them:

    layer_norm(x, weight, bias)                 norm over the features of each row
    gated_feed_forward(x, w_gate, w_up)         act(x w_gate^T) * (x w_up^T), one kernel
    log_probs(logits, targets, top)             log probabilities of given classes, entropy, the ranked best classes
    distillation_loss(logits, ids, scores)      loss against a teacher's best scores

The reference leaves this part to torch (BatchNorm1d, Linear + ReLU, Linear, LogSoftmax: ``MNIST/model.py:28-67``).  Rows are
the last axis of a tensor of any leading shape, in float32, bfloat16 or float16; sums, norms and softmax statistics are held
in float32 or more whatever that type, and each result is rounded once.  The gated block's backward rounds one thing more: on the
tensor cores, the gradients of its two projections take the type of x before they are multiplied (a 16-bit gradient's error is
1.4 times one rounding's; in float16 those that would leave that type's range are scaled by powers of two).  All arithmetic happens in libcgnet_b200.so on the
current stream; the checks of the arguments, the allocations and the autograd nodes are C++ too (``_torch_head.so``,
``csrc/torch_head.cpp``).  There is no CPU path and no fallback: a missing library or a bad argument raises RuntimeError before
anything is launched.  Every operator is differentiable once (in reverse mode), can be captured in a CUDA graph, and gives the same bits from run
to run for the same tensors; ``torch.jit.trace`` is refused.  (As with any torch operator, capture a backward pass only while no eager graph of the same leaves
is alive: torch ties a leaf's gradient accumulation to the stream it was first used on.)  The order of a row's sums follows
the 16-byte groups it lies in, so its last bits can depend on its address modulo 16.
"""
import collections
import importlib
import os

import torch
from torch import nn

from . import _lib

__all__ = ["layer_norm", "gated_feed_forward", "log_probs", "distillation_loss", "LogProbs", "LayerNorm", "GatedFeedForward",
           "InvariantHead"]

ACTIVATIONS = ("silu", "gelu", "relu")

LogProbs = collections.namedtuple("LogProbs", ["log_prob", "entropy", "top_log_probs", "top_ids"])

_native = None


def _load():
    """The torch side of the library, loaded on first use."""
    global _native
    if _native is None:
        _lib.load()
        path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_torch_head.so")
        if not os.path.exists(path):
            raise RuntimeError(f"{path} is missing: build it with `python -m cgnet_b200.build`. cgnet_b200 has no PyTorch fallback.")
        _native = importlib.import_module("._torch_head", __package__)
    return _native


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis.  ``weight`` and ``bias`` (``(dim,)``, of x's type or
    float32, each optional) get gradients of their own type, summed over the rows in a fixed order."""
    return (_native or _load()).layer_norm(x, weight, bias, eps)


def gated_feed_forward(x, w_gate, w_up, activation="silu"):
    """``act(x w_gate^T) * (x w_up^T)`` over the last axis: x ``(..., dim)``, weights ``(hidden, dim)``, all of one type;
    ``activation`` is ``"silu"``, ``"gelu"`` (the exact one, with erf) or ``"relu"``.

    A call that will be differentiated keeps both projections in float32 (8 bytes per row and hidden unit) for its backward.  Values
    that are not finite spoil the results of their own row of x, or of their own hidden unit, and no others; float32 operands are
    multiplied in parts on the tensor cores, where a projection with an infinite term may be NaN instead of infinite."""
    return (_native or _load()).gated_feed_forward(x, w_gate, w_up, activation)


def log_probs(logits, targets=None, top=0):
    """``LogProbs(log_prob, entropy, top_log_probs, top_ids)`` of logits ``(..., classes)``, all float32 but the int64 ids.

    ``targets`` (``(...)``, int64 or int32; optional) selects the class of each row; a negative one marks a row without (log
    probability 0, no gradient through it), one beyond the last class gives NaN.  ``top`` (0 to 128) classes are ranked by
    score, equal scores by class; they carry no gradient, log_prob and entropy do.  A row of nothing but -inf has log
    probabilities -inf, entropy 0 and gradients 0."""
    return LogProbs(*(_native or _load()).log_probs(logits, targets, top))


def distillation_loss(logits, teacher_ids, teacher_scores, temperature=1.0):
    """Loss of each row of ``logits`` ``(..., classes)`` against the teacher's scores for the K classes it names:
    ``T^2 sum_k q_k (log q_k - log p(id_k))`` with ``q`` the softmax of ``teacher_scores / T`` over the row's entries and ``p``
    the softmax of ``logits / T`` over all classes; float32, shape ``(...)``.

    ``teacher_ids`` (int64 or int32) and ``teacher_scores`` (float32, bfloat16 or float16) are ``(..., K)``, K from 1 to 1024.  A
    negative id is an entry that is not there, a score of -inf one of weight 0; one beyond the last class makes the row NaN.  A row
    without entries has loss and gradient 0; one whose logits are all -inf has loss +inf and gradient 0.  The teacher's scores
    get no gradient."""
    return (_native or _load()).distillation_loss(logits, teacher_ids, teacher_scores, temperature)


# ---------------------------------------------------------------------------------------------------------------------
# modules
# ---------------------------------------------------------------------------------------------------------------------
class LayerNorm(nn.Module):
    """Layer norm with a learned weight and bias (``weight``, ``bias``: ``(dim,)``, ones and zeros at first)."""

    def __init__(self, dim, eps=1e-5, device="cuda", dtype=torch.float32):
        super().__init__()
        self.eps = float(eps)
        self.weight = nn.Parameter(torch.ones(dim, device=device, dtype=dtype))
        self.bias = nn.Parameter(torch.zeros(dim, device=device, dtype=dtype))

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)


class GatedFeedForward(nn.Module):
    """Gated hidden layer ``(..., dim) -> (..., hidden)`` with weights ``w_gate`` and ``w_up`` ``(hidden, dim)``, uniform in
    +-1/sqrt(dim) at first."""

    def __init__(self, dim, hidden, activation="silu", device="cuda", dtype=torch.float32):
        super().__init__()
        if activation not in ACTIVATIONS:
            raise RuntimeError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
        self.activation = activation
        bound = dim ** -0.5
        self.w_gate = nn.Parameter(torch.empty(hidden, dim, device=device, dtype=dtype).uniform_(-bound, bound))
        self.w_up = nn.Parameter(torch.empty(hidden, dim, device=device, dtype=dtype).uniform_(-bound, bound))

    def forward(self, x):
        return gated_feed_forward(x, self.w_gate, self.w_up, self.activation)


class InvariantHead(nn.Module):
    """Classifier on the invariant embedding: ``norm`` (layer norm) -> ``ff`` (gated hidden layer) -> ``scores`` (linear),
    ``(..., dim) -> (..., classes)`` logits.  ``SphericalCNN(..., head=(hidden, classes))`` builds one, in float32; with another
    ``dtype`` the embedding is converted to it first and the logits are of it.  (``torch.autocast`` does not change what the operators
    compute in: their types are their arguments'.)"""

    def __init__(self, dim, hidden, classes, activation="silu", device="cuda", dtype=torch.float32):
        super().__init__()
        self.norm = LayerNorm(dim, device=device, dtype=dtype)
        self.ff = GatedFeedForward(dim, hidden, activation, device=device, dtype=dtype)
        self.scores = nn.Linear(hidden, classes, device=device, dtype=dtype)

    def forward(self, x):
        return self.scores(self.ff(self.norm(x.to(self.norm.weight.dtype))))
