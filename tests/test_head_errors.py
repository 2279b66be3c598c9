"""Operators behind the invariant embedding: errors from below keep their type."""
import pytest
import torch

import cgnet_b200 as cg


class Asked(Exception):
    pass


class Refusing(torch.Tensor):
    """Class indices whose conversion raises."""

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise Asked(str(func))


def test_errors_of_python_code_keep_their_type():
    z, ids = torch.zeros(4, 6), torch.zeros(4, dtype=torch.int32).as_subclass(Refusing)
    with pytest.raises(Asked):
        cg.log_probs(z, ids)
    with pytest.raises(Asked):
        cg.distillation_loss(z, torch.zeros(4, 2, dtype=torch.int32).as_subclass(Refusing), torch.zeros(4, 2))


def cuda_calls():
    """name -> (function of x, x)"""
    g = torch.Generator(device="cuda")
    g.manual_seed(1)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")
    w, b, wg, wu = randn(24), randn(24), randn(36, 24).requires_grad_(), randn(36, 24)
    ids, scores = torch.randint(0, 24, (10, 4), generator=g, device="cuda"), randn(10, 4)
    return {"layer_norm": lambda x: cg.layer_norm(2 * x, w, b), "gated_feed_forward": lambda x: cg.gated_feed_forward(2 * x, wg, wu),
            "log_probs": lambda x: cg.log_probs(2 * x, ids[:, 0]).log_prob, "distillation_loss": lambda x: cg.distillation_loss(2 * x, ids, scores),
            }, randn(10, 24)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["layer_norm", "gated_feed_forward", "log_probs", "distillation_loss"])
@pytest.mark.parametrize("reentrant", [False, True])
def test_activation_checkpointing(name, reentrant):
    """The operator is the last of the checkpointed function to keep anything: its recomputation ends inside the call."""
    from torch.utils.checkpoint import checkpoint
    calls, x = cuda_calls()
    x.requires_grad_()
    (want,) = torch.autograd.grad(calls[name](x).sum(), x)
    checkpoint(calls[name], x, use_reentrant=reentrant).sum().backward()
    assert torch.equal(x.grad, want)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["layer_norm", "gated_feed_forward", "log_probs", "distillation_loss"])
def test_errors_of_saved_tensor_hooks_keep_their_type(name):
    calls, x = cuda_calls()
    x.requires_grad_()

    def pack(t):
        if t.data_ptr() != x.data_ptr():
            raise Asked(name)
        return t
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        with pytest.raises(Asked, match=name):
            calls[name](x)

    def unpack(t):
        raise Asked(name)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        y = calls[name](x)
    with pytest.raises(Asked, match=name):
        torch.autograd.grad(y.sum(), x)
    with torch.autograd.graph.save_on_cpu():
        y = calls[name](x)
    assert torch.equal(torch.autograd.grad(y.sum(), x)[0], torch.autograd.grad(calls[name](x).sum(), x)[0])


@pytest.mark.gpu
def test_memory_that_is_not_there():
    """2^22 x 2^16 results of 2 bytes, 549 GB, are asked for."""
    x = torch.zeros(1, 1, device="cuda", dtype=torch.bfloat16).expand(1 << 22, 1)
    w = torch.zeros(1 << 16, 1, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(torch.OutOfMemoryError):
        cg.gated_feed_forward(x, w, w)
    assert cg.gated_feed_forward(x[:3], w, w).shape == (3, 1 << 16)


def test_tracing_is_refused():
    """A trace would return the memory that the kernels never write."""
    x, w = torch.zeros(4, 6), torch.zeros(5, 6)
    ids, scores = torch.zeros(4, 2, dtype=torch.long), torch.zeros(4, 2)
    for call in (lambda t: cg.layer_norm(t), lambda t: cg.gated_feed_forward(t, w, w), lambda t: cg.log_probs(t).entropy,
                 lambda t: cg.distillation_loss(t, ids, scores)):
        with pytest.raises(RuntimeError, match="torch.jit.trace"):
            torch.jit.trace(call, (x,))
