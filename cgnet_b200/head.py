"""The operators between a CG network's invariant embedding and its answers, and the classifier head built from them:

    layer_norm(x, weight, bias)                 norm over the features of each row
    gated_feed_forward(x, w_gate, w_up)         act(x w_gate^T) * (x w_up^T), one kernel
    log_probs(logits, targets, top)             log probabilities of given classes, entropy, the ranked best classes
    distillation_loss(logits, ids, scores)      loss against a teacher's best scores

The reference leaves this part to torch (BatchNorm1d, Linear + ReLU, Linear, LogSoftmax: ``MNIST/model.py:28-67``).  Rows are
the last axis of a tensor of any leading shape, in float32, bfloat16 or float16; sums, norms and softmax statistics are held
in float32 or more whatever that type, and each result is rounded once.  All arithmetic happens in libcgnet_b200.so on the
current stream; there is no CPU path.  Every operator is differentiable once, can be captured in a CUDA graph, and gives the same
bits from run to run.  (As with any torch operator, capture a backward pass only while no eager graph of the same leaves is
alive: torch ties a leaf's gradient accumulation to the stream it was first used on.)
"""
import collections
import functools
import math

import torch
from torch import nn

from . import _lib
from .cg_layers import _current_stream

__all__ = ["layer_norm", "gated_feed_forward", "log_probs", "distillation_loss", "LogProbs", "LayerNorm", "GatedFeedForward",
           "InvariantHead"]

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_ACTIVATIONS = {"silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU, "relu": _lib.ACT_RELU}

LogProbs = collections.namedtuple("LogProbs", ["log_prob", "entropy", "top_log_probs", "top_ids"])


# ---------------------------------------------------------------------------------------------------------------------
# argument checks (they run before any pointer reaches the library) and the call itself
# ---------------------------------------------------------------------------------------------------------------------
def _check_values(t, name, device=None, dtype=None):
    """A float32, bfloat16 or float16 CUDA tensor, on ``device`` and of ``dtype`` where those are given."""
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{name} must be a tensor, got {type(t).__name__}")
    own = t.dtype
    if own not in _DTYPES:
        raise RuntimeError(f"{name} must be float32, bfloat16 or float16, got {own}")
    if dtype is not None and own is not dtype:
        raise RuntimeError(f"{name} must be {dtype}, got {own}")
    if device is not None and t.device != device:
        raise RuntimeError(f"{name} lives on {t.device}, expected {device}")
    return t


def _check_shape(t, name, shape):
    if t.shape != shape:
        raise RuntimeError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    return t


def _check_cuda(t, name):
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor (cgnet_b200 has no CPU path)")


def _check_classes(t, name, shape, device):
    """int64 (or int32) class indices; their values are the kernels' business."""
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int64, torch.int32):
        raise RuntimeError(f"{name} must be an int64 or int32 tensor")
    if t.device != device:
        raise RuntimeError(f"{name} lives on {t.device}, expected {device}")
    return _check_shape(t, name, shape).to(torch.int64).contiguous()


def _rows(t):
    """``t`` as (rows, columns) whose columns are neighbours in memory; rows may be any distance apart."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _check_rows(t, name):
    if t.dim() == 0 or t.shape[-1] == 0:
        raise RuntimeError(f"{name} must have at least one value in its last dimension, got shape {tuple(t.shape)}")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(name, index, *args):
    """Run an entry point on the current stream of CUDA device ``index``."""
    fn = getattr(_lib.load(), name)
    if torch.cuda.current_device() == index:
        rc = fn(*args, _current_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _current_stream(index))
    if rc != 0:
        _lib.check(rc, name)


def _once():
    """First line of every backward: the gradients are not differentiable themselves, and say so (autograd runs a backward with
    gradients enabled only where its result is to be differentiated again)."""
    if torch.is_grad_enabled():
        raise RuntimeError("the operators of cgnet_b200.head are differentiable once only")


def _workspace(nbytes, device):
    """Scratch of one call, from torch's allocator (which keeps it apart from other streams' and graphs' calls)."""
    if nbytes < 0:
        _lib.check(1, "workspace size")
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _empty(rows, columns, like):
    """(rows, columns) of ``like``'s type and device, contiguous."""
    return torch.empty((rows, columns), dtype=like.dtype, device=like.device)


# ---------------------------------------------------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------------------------------------------------
def _layer_norm_fwd(x2, weight, bias, eps, keep):
    rows, dim = x2.shape
    index = x2.get_device()
    y = _empty(rows, dim, x2)
    stats = torch.empty((rows, 2), dtype=torch.float32, device=x2.device) if keep else None
    param = weight if weight is not None else bias
    dtype = _DTYPES[x2.dtype]
    _call("cgb200_layer_norm_fwd", index, x2.data_ptr(), x2.stride(0), _ptr(weight), _ptr(bias), eps, y.data_ptr(), _ptr(stats), rows, dim, dtype,
          dtype if param is None else _DTYPES[param.dtype])
    return y, stats


@functools.lru_cache(maxsize=1024)
def _layer_norm_bwd_bytes(rows, dim, dtype):
    return _lib.load().cgb200_layer_norm_bwd_workspace_bytes(rows, dim, dtype)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x2, weight, bias, eps):
        y, stats = _layer_norm_fwd(x2, weight, bias, eps, True)
        ctx.save_for_backward(x2, weight, stats)
        ctx.param_dtype = weight.dtype if weight is not None else bias.dtype if bias is not None else x2.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        _once()
        x2, weight, stats = ctx.saved_tensors
        rows, dim = x2.shape
        dy = _rows(dy)
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        dev, dtype, param_dtype = x2.device, _DTYPES[x2.dtype], ctx.param_dtype
        dx = _empty(rows, dim, x2) if need_x else None
        dw = torch.empty(dim, dtype=param_dtype, device=dev) if need_w else None
        db = torch.empty(dim, dtype=param_dtype, device=dev) if need_b else None
        n = _layer_norm_bwd_bytes(rows, dim, dtype) if need_w or need_b else 0
        ws = _workspace(n, dev)
        _call("cgb200_layer_norm_bwd", x2.get_device(), x2.data_ptr(), x2.stride(0), dy.data_ptr(), dy.stride(0), _ptr(weight), stats.data_ptr(),
              _ptr(dx), _ptr(dw), _ptr(db), rows, dim, dtype, _DTYPES[param_dtype], _ptr(ws), n)
        return dx, dw, db, None


def _check_layer_norm(x, weight, bias):
    _check_values(x, "x")
    _check_rows(x, "x")
    dim = x.shape[-1]
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None:
            _check_shape(_check_values(p, name, x.device), name, (dim,))
            if p.dtype != x.dtype and p.dtype != torch.float32:
                raise RuntimeError(f"{name} must be {x.dtype} or float32, got {p.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError(f"weight and bias must have one type, got {weight.dtype} and {bias.dtype}")


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis.  ``weight`` and ``bias`` (``(dim,)``, of x's type or
    float32, each optional) get gradients of their own type, summed over the rows in a fixed order."""
    if not 0.0 <= eps < math.inf:
        raise RuntimeError(f"eps must be finite and not negative, got {eps}")
    _check_layer_norm(x, weight, bias)
    _check_cuda(x, "x")
    x2 = _rows(x)
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad)):
        y = _LayerNorm.apply(x2, weight, bias, float(eps))
    else:
        y = _layer_norm_fwd(x2, weight, bias, float(eps), False)[0]
    return y if x.dim() == 2 else y.view(x.shape)


# ---------------------------------------------------------------------------------------------------------------------
# gated feed-forward block
# ---------------------------------------------------------------------------------------------------------------------
def _gated_ff_fwd(x2, wg, wu, act, keep):
    rows, dim = x2.shape
    hidden = wg.shape[0]
    dev, dtype = x2.device, _DTYPES[x2.dtype]
    h = torch.empty(rows, hidden, dtype=x2.dtype, device=dev)
    gate_up = torch.empty((2, rows, (hidden + 3) & ~3), dtype=torch.float32, device=dev) if keep else None
    operands = (x2.data_ptr(), x2.stride(0), wg.data_ptr(), wg.stride(0), wu.data_ptr(), wu.stride(0))
    n = _lib.load().cgb200_gated_ff_workspace_bytes(*operands, rows, dim, hidden, dtype, 0)
    ws = _workspace(n, dev)
    _call("cgb200_gated_ff_fwd", x2.get_device(), *operands, act, h.data_ptr(),
          _ptr(gate_up), rows, dim, hidden, dtype, _ptr(ws), n)
    return h, gate_up


class _GatedFeedForward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x2, wg, wu, act):
        h, gate_up = _gated_ff_fwd(x2, wg, wu, act, True)
        ctx.save_for_backward(x2, wg, wu, gate_up)
        ctx.act = act
        return h

    @staticmethod
    def backward(ctx, dh):
        _once()
        x2, wg, wu, gate_up = ctx.saved_tensors
        rows, dim = x2.shape
        hidden = wg.shape[0]
        dh = _rows(dh)
        need = ctx.needs_input_grad
        dev, dtype = x2.device, _DTYPES[x2.dtype]
        dx = torch.empty(rows, dim, dtype=x2.dtype, device=dev) if need[0] else None
        dwg = torch.empty(hidden, dim, dtype=x2.dtype, device=dev) if need[1] else None
        dwu = torch.empty(hidden, dim, dtype=x2.dtype, device=dev) if need[2] else None
        operands = (x2.data_ptr(), x2.stride(0), wg.data_ptr(), wg.stride(0), wu.data_ptr(), wu.stride(0))
        n = _lib.load().cgb200_gated_ff_workspace_bytes(*operands, rows, dim, hidden, dtype, bool(need[0]) + 2 * bool(need[1]) + 4 * bool(need[2]))
        ws = _workspace(n, dev)
        _call("cgb200_gated_ff_bwd", x2.get_device(), *operands, ctx.act, gate_up.data_ptr(), dh.data_ptr(), dh.stride(0), _ptr(dx), _ptr(dwg), _ptr(dwu), rows, dim, hidden, dtype, _ptr(ws), n)
        return dx, dwg, dwu, None


def gated_feed_forward(x, w_gate, w_up, activation="silu"):
    """``act(x w_gate^T) * (x w_up^T)`` over the last axis: x ``(..., dim)``, weights ``(hidden, dim)``, all of one type;
    ``activation`` is ``"silu"``, ``"gelu"`` (the exact one, with erf) or ``"relu"``.

    A call that will be differentiated keeps both projections in float32 (8 bytes per row and hidden unit) for its backward."""
    if activation not in _ACTIVATIONS:
        raise RuntimeError(f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
    _check_values(x, "x")
    _check_rows(x, "x")
    dim = x.shape[-1]
    for name, w in (("w_gate", w_gate), ("w_up", w_up)):
        _check_values(w, name, x.device, x.dtype)
        if w.dim() != 2 or w.shape[1] != dim or w.shape[0] == 0:
            raise RuntimeError(f"{name} has shape {tuple(w.shape)}, expected (hidden, {dim})")
    _check_shape(w_up, "w_up", w_gate.shape)
    _check_cuda(x, "x")
    x2, wg, wu, act = _rows(x), _rows(w_gate), _rows(w_up), _ACTIVATIONS[activation]
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad):
        h = _GatedFeedForward.apply(x2, wg, wu, act)
    else:
        h, _ = _gated_ff_fwd(x2, wg, wu, act, False)
    return h if x.dim() == 2 else h.view(*x.shape[:-1], h.shape[1])


# ---------------------------------------------------------------------------------------------------------------------
# log probabilities
# ---------------------------------------------------------------------------------------------------------------------
def _log_probs_fwd(z2, targets, top, keep):
    rows, classes = z2.shape
    dev = z2.device
    out = torch.empty(2, rows, dtype=torch.float32, device=dev)
    log_prob, entropy = out[0], out[1]
    top_lp = torch.empty(rows, top, dtype=torch.float32, device=dev)
    top_ids = torch.empty(rows, top, dtype=torch.int64, device=dev)
    stats = torch.empty(rows, 2, dtype=torch.float32, device=dev) if keep else None
    _call("cgb200_log_probs_fwd", z2.get_device(), z2.data_ptr(), z2.stride(0), _ptr(targets), top, log_prob.data_ptr(), entropy.data_ptr(),
          top_lp.data_ptr(), top_ids.data_ptr(), _ptr(stats), rows, classes, _DTYPES[z2.dtype])
    return log_prob, entropy, top_lp, top_ids, stats


class _LogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z2, targets, top):
        log_prob, entropy, top_lp, top_ids, stats = _log_probs_fwd(z2, targets, top, True)
        ctx.save_for_backward(z2, targets, entropy, stats)
        ctx.mark_non_differentiable(top_lp, top_ids)
        ctx.set_materialize_grads(False)
        return log_prob, entropy, top_lp, top_ids

    @staticmethod
    def backward(ctx, g_lp, g_ent, _top_lp, _top_ids):
        _once()
        z2, targets, entropy, stats = ctx.saved_tensors
        if targets is None:
            g_lp = None
        if not ctx.needs_input_grad[0] or (g_lp is None and g_ent is None):
            return None, None, None
        rows, classes = z2.shape
        g_lp = None if g_lp is None else g_lp.contiguous()
        g_ent = None if g_ent is None else g_ent.contiguous()
        dz = torch.empty(rows, classes, dtype=z2.dtype, device=z2.device)
        _call("cgb200_log_probs_bwd", z2.get_device(), z2.data_ptr(), z2.stride(0), _ptr(targets), entropy.data_ptr(), stats.data_ptr(), _ptr(g_lp),
              _ptr(g_ent), dz.data_ptr(), rows, classes, _DTYPES[z2.dtype])
        return dz, None, None


def log_probs(logits, targets=None, top=0):
    """``LogProbs(log_prob, entropy, top_log_probs, top_ids)`` of logits ``(..., classes)``, all float32 but the int64 ids.

    ``targets`` (``(...)``, int64 or int32; optional) selects the class of each row; a negative one marks a row without (log
    probability 0, no gradient through it), one beyond the last class gives NaN.  ``top`` (0 to 128) classes are ranked by
    score, equal scores by class; they carry no gradient, log_prob and entropy do.  A row of nothing but -inf has log
    probabilities -inf, entropy 0 and gradients 0."""
    _check_values(logits, "logits")
    _check_rows(logits, "logits")
    lead, classes = logits.shape[:-1], logits.shape[-1]
    if isinstance(top, bool) or not isinstance(top, int) or not 0 <= top <= min(_lib.MAX_TOP, classes):
        raise RuntimeError(f"top must be an integer from 0 to {min(_lib.MAX_TOP, classes)}, got {top!r}")
    if targets is not None:
        targets = _check_classes(targets, "targets", lead, logits.device).reshape(-1)
    _check_cuda(logits, "logits")
    z2 = _rows(logits)
    if torch.is_grad_enabled() and logits.requires_grad:
        lp, ent, top_lp, top_ids = _LogProbs.apply(z2, targets, top)
    else:
        lp, ent, top_lp, top_ids, _ = _log_probs_fwd(z2, targets, top, False)
    if len(lead) != 1:
        lp, ent, top_lp, top_ids = lp.view(lead), ent.view(lead), top_lp.view(*lead, top), top_ids.view(*lead, top)
    return LogProbs(lp if targets is not None else None, ent, top_lp, top_ids)


# ---------------------------------------------------------------------------------------------------------------------
# distillation
# ---------------------------------------------------------------------------------------------------------------------
def _distill_fwd(z2, ids, scores, temperature, keep):
    rows, classes = z2.shape
    dev = z2.device
    loss = torch.empty(rows, dtype=torch.float32, device=dev)
    stats = torch.empty(rows, 4, dtype=torch.float32, device=dev) if keep else None
    _call("cgb200_distill_fwd", z2.get_device(), z2.data_ptr(), z2.stride(0), ids.data_ptr(), scores.data_ptr(), ids.shape[1], _DTYPES[scores.dtype],
          temperature, loss.data_ptr(), _ptr(stats), rows, classes, _DTYPES[z2.dtype])
    return loss, stats


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z2, ids, scores, temperature):
        loss, stats = _distill_fwd(z2, ids, scores, temperature, True)
        ctx.save_for_backward(z2, ids, scores, stats)
        ctx.temperature = temperature
        return loss

    @staticmethod
    def backward(ctx, g):
        _once()
        z2, ids, scores, stats = ctx.saved_tensors
        rows, classes = z2.shape
        g = g.contiguous()
        dz = torch.empty(rows, classes, dtype=z2.dtype, device=z2.device)
        _call("cgb200_distill_bwd", z2.get_device(), z2.data_ptr(), z2.stride(0), ids.data_ptr(), scores.data_ptr(), ids.shape[1],
              _DTYPES[scores.dtype], ctx.temperature, stats.data_ptr(), g.data_ptr(), dz.data_ptr(), rows, classes, _DTYPES[z2.dtype])
        return dz, None, None, None


def distillation_loss(logits, teacher_ids, teacher_scores, temperature=1.0):
    """Loss of each row of ``logits`` ``(..., classes)`` against the teacher's scores for the K classes it names:
    ``T^2 sum_k q_k (log q_k - log p(id_k))`` with ``q`` the softmax of ``teacher_scores / T`` over the row's entries and ``p``
    the softmax of ``logits / T`` over all classes; float32, shape ``(...)``.

    ``teacher_ids`` (int64 or int32) and ``teacher_scores`` (float32, bfloat16 or float16) are ``(..., K)``, K from 1 to 1024.  A
    negative id is an entry that is not there, a score of -inf one of weight 0; one beyond the last class makes the row NaN.  A row
    without entries has loss and gradient 0; one whose logits are all -inf has loss +inf and gradient 0.  The teacher's scores
    get no gradient."""
    _check_values(logits, "logits")
    _check_rows(logits, "logits")
    lead = logits.shape[:-1]
    _check_values(teacher_scores, "teacher_scores", logits.device)
    k = teacher_scores.shape[-1] if teacher_scores.dim() else 0
    if not 1 <= k <= _lib.MAX_TEACHER:
        raise RuntimeError(f"teacher_scores must name 1 to {_lib.MAX_TEACHER} classes a row, got shape {tuple(teacher_scores.shape)}")
    _check_shape(teacher_scores, "teacher_scores", (*lead, k))
    ids = _check_classes(teacher_ids, "teacher_ids", (*lead, k), logits.device).reshape(-1, k)
    if not 1e-3 <= temperature <= 1e3:
        raise RuntimeError(f"temperature must be between 0.001 and 1000, got {temperature}")
    _check_cuda(logits, "logits")
    z2, scores = _rows(logits), teacher_scores.detach().reshape(-1, k).contiguous()
    if torch.is_grad_enabled() and logits.requires_grad:
        loss = _Distill.apply(z2, ids, scores, float(temperature))
    else:
        loss, _ = _distill_fwd(z2, ids, scores, float(temperature), False)
    return loss if len(lead) == 1 else loss.view(lead)


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
        if activation not in _ACTIVATIONS:
            raise RuntimeError(f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
        self.activation = activation
        bound = dim ** -0.5
        self.w_gate = nn.Parameter(torch.empty(hidden, dim, device=device, dtype=dtype).uniform_(-bound, bound))
        self.w_up = nn.Parameter(torch.empty(hidden, dim, device=device, dtype=dtype).uniform_(-bound, bound))

    def forward(self, x):
        return gated_feed_forward(x, self.w_gate, self.w_up, self.activation)


class InvariantHead(nn.Module):
    """Classifier on the invariant embedding: ``norm`` (layer norm) -> ``ff`` (gated hidden layer) -> ``scores`` (linear),
    ``(..., dim) -> (..., classes)`` logits.  ``SphericalCNN(..., head=(hidden, classes))`` builds one."""

    def __init__(self, dim, hidden, classes, activation="silu", device="cuda", dtype=torch.float32):
        super().__init__()
        self.norm = LayerNorm(dim, device=device, dtype=dtype)
        self.ff = GatedFeedForward(dim, hidden, activation, device=device, dtype=dtype)
        self.scores = nn.Linear(hidden, classes, device=device, dtype=dtype)

    def forward(self, x):
        return self.scores(self.ff(self.norm(x)))
