"""Operators behind the invariant embedding: what they refuse, checked without a GPU (no pointer reaches a kernel)."""
import pytest
import torch

import cgnet_b200 as cg
from cgnet_b200 import _lib

X = torch.zeros(4, 6)
W = torch.zeros(5, 6)


@pytest.mark.parametrize("call, message", [
    (lambda: cg.layer_norm([1.0]), "must be a tensor"),
    (lambda: cg.layer_norm(X.double()), "float32, bfloat16 or float16"),
    (lambda: cg.layer_norm(torch.zeros(())), "at least one value"),
    (lambda: cg.layer_norm(torch.zeros(3, 0)), "at least one value"),
    (lambda: cg.layer_norm(X, torch.zeros(5)), "shape"),
    (lambda: cg.layer_norm(X, torch.zeros(6), torch.zeros(6, 1)), "shape"),
    (lambda: cg.layer_norm(X.bfloat16(), torch.zeros(6).half()), "weight must be"),
    (lambda: cg.layer_norm(X.bfloat16(), torch.zeros(6), torch.zeros(6).bfloat16()), "one type"),
    (lambda: cg.layer_norm(X, torch.zeros(6, device="meta")), "lives on"),
    (lambda: cg.layer_norm(X, eps=-1.0), "eps"),
    (lambda: cg.layer_norm(X, eps=float("nan")), "eps"),
    (lambda: cg.layer_norm(X), "CUDA"),
    (lambda: cg.gated_feed_forward(X, W, W, "tanh"), "activation"),
    (lambda: cg.gated_feed_forward(X, W, W[:4]), "shape"),
    (lambda: cg.gated_feed_forward(X, W[:, :5], W), "shape"),
    (lambda: cg.gated_feed_forward(X, W[:0], W[:0]), "shape"),
    (lambda: cg.gated_feed_forward(X, W.half(), W), "w_gate must be torch.float32"),
    (lambda: cg.gated_feed_forward(X, W, W.to("meta")), "lives on"),
    (lambda: cg.gated_feed_forward(X, W, W), "CUDA"),
    (lambda: cg.log_probs(X.long()), "float32, bfloat16 or float16"),
    (lambda: cg.log_probs(X, torch.zeros(4)), "int64"),
    (lambda: cg.log_probs(X, torch.zeros(3, dtype=torch.long)), "shape"),
    (lambda: cg.log_probs(X, top=7), "top must be"),
    (lambda: cg.log_probs(torch.zeros(2, 500), top=129), "top must be"),
    (lambda: cg.log_probs(X, top=-1), "top must be"),
    (lambda: cg.log_probs(X, top=1.0), "top must be"),
    (lambda: cg.log_probs(X, top=True), "top must be"),
    (lambda: cg.log_probs(X), "CUDA"),
    (lambda: cg.distillation_loss(X, torch.zeros(4, 2, dtype=torch.long), torch.zeros(4, 3)), "shape"),
    (lambda: cg.distillation_loss(X, torch.zeros(4, 2), torch.zeros(4, 2)), "int64"),
    (lambda: cg.distillation_loss(X, torch.zeros(4, 0, dtype=torch.long), torch.zeros(4, 0)), "1 to 1024"),
    (lambda: cg.distillation_loss(X, torch.zeros(4, 1025, dtype=torch.long), torch.zeros(4, 1025)), "1 to 1024"),
    (lambda: cg.distillation_loss(X, torch.zeros(3, 2, dtype=torch.long), torch.zeros(3, 2)), "shape"),
    (lambda: cg.distillation_loss(X, torch.zeros(4, 2, dtype=torch.long), torch.zeros(4, 2), temperature=0.0), "temperature"),
    (lambda: cg.distillation_loss(X, torch.zeros(4, 2, dtype=torch.long), torch.zeros(4, 2), temperature=float("nan")), "temperature"),
    (lambda: cg.distillation_loss(X, torch.zeros(4, 2, dtype=torch.long), torch.zeros(4, 2)), "CUDA"),
    (lambda: cg.GatedFeedForward(6, 5, "tanh", device="cpu"), "activation"),
])
def test_refusals(call, message):
    with pytest.raises(RuntimeError, match=message):
        call()


def test_forward_mode_derivatives_are_refused():
    import torch.autograd.forward_ad as fwad
    ids, scores = torch.zeros(4, 2, dtype=torch.long), torch.zeros(4, 2)
    with fwad.dual_level():
        d, dw = fwad.make_dual(X, torch.ones_like(X)), fwad.make_dual(W, torch.ones_like(W))
        for call in (lambda: cg.layer_norm(d), lambda: cg.gated_feed_forward(X, W, dw), lambda: cg.log_probs(d),
                     lambda: cg.distillation_loss(d, ids, scores)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_library_refusals_need_no_gpu():
    """The C entry points return a status for bad arguments before any CUDA call."""
    lib = _lib.load()
    p = 16     # a pointer that is never followed
    bad = 1
    assert lib.cgb200_layer_norm_fwd(p, 4, None, None, 1e-5, p, None, -1, 4, 0, 0, None) == bad
    assert lib.cgb200_layer_norm_fwd(p, 4, None, None, 1e-5, p, None, 2, 0, 0, 0, None) == bad
    assert lib.cgb200_layer_norm_fwd(p, 4, None, None, 1e-5, p, None, 2, 4, 3, 3, None) == bad
    assert lib.cgb200_layer_norm_fwd(p, 4, None, None, 1e-5, p, None, 2, 4, _lib.BF16, _lib.F16, None) == bad
    assert lib.cgb200_layer_norm_fwd(p, -4, None, None, 1e-5, p, None, 2, 4, 0, 0, None) == bad
    assert lib.cgb200_layer_norm_fwd(None, 4, None, None, 1e-5, p, None, 2, 4, 0, 0, None) == bad
    assert lib.cgb200_layer_norm_fwd(None, 4, None, None, 1e-5, None, None, 0, 4, 0, 0, None) == 0
    assert lib.cgb200_layer_norm_fwd(p, 4, None, None, 1e-5, p, p + 4, 2, 4, 0, 0, None) == bad
    assert lib.cgb200_layer_norm_bwd_workspace_bytes(-1, 4, 0) == -1
    assert lib.cgb200_layer_norm_bwd(p, 64, p, 64, None, p, p, p, p, 100000, 64, 0, 0, None, 0, None) == 4
    assert b"need" in lib.cgb200_last_error()
    assert lib.cgb200_gated_ff_fwd(p, 4, p, 4, p, 4, 3, p, None, 2, 4, 4, 0, None, 0, None) == bad
    assert lib.cgb200_gated_ff_fwd(p, 4, p, 4, None, 4, 0, p, None, 2, 4, 4, 0, None, 0, None) == bad
    assert lib.cgb200_gated_ff_fwd(p, 4, p, 4, p, 4, 0, p, None, 2, 4, (1 << 20) + 1, 0, None, 0, None) == bad
    assert lib.cgb200_gated_ff_fwd(p, 4, p, 4, p, 4, 0, p, p + 4, 2, 4, 4, 0, None, 0, None) == bad
    assert lib.cgb200_gated_ff_fwd(p, 1 << 20, p, 1 << 20, p, 1 << 20, 0, p, None, 1 << 24, 1 << 20, 4, 0, None, 0, None) == bad
    assert lib.cgb200_gated_ff_workspace_bytes(p, 4, p, 4, p, 4, 2, 0, 4, 0, 0) == -1
    assert lib.cgb200_gated_ff_fwd(p, 64, p, 64, p, 64, 0, p, None, 4096, 1024, 1024, 0, None, 0, None) == 4
    assert lib.cgb200_gated_ff_bwd(p, 4, p, 4, p, 4, 0, None, p, 4, p, p, p, 2, 4, 4, 0, None, 0, None) == bad
    assert lib.cgb200_log_probs_fwd(p, 4, None, 5, None, p, p, p, None, 2, 4, 0, None) == bad
    assert lib.cgb200_log_probs_fwd(p, 400, None, 129, None, p, p, p, None, 2, 400, 0, None) == bad
    assert lib.cgb200_log_probs_fwd(p, 4, p, 0, None, p, None, None, None, 2, 4, 0, None) == bad
    assert lib.cgb200_log_probs_fwd(p, 4, None, 1, None, p, p, p, p + 4, 2, 4, 0, None) == bad
    assert lib.cgb200_log_probs_bwd(p, 4, None, p, None, None, p, p, 2, 4, 0, None) == bad
    assert lib.cgb200_distill_fwd(p, 4, p, p, 0, 0, 1.0, p, None, 2, 4, 0, None) == bad
    assert lib.cgb200_distill_fwd(p, 4, p, p, 2, 7, 1.0, p, None, 2, 4, 0, None) == bad
    assert lib.cgb200_distill_fwd(p, 4, p, p, 2, 0, 0.0, p, None, 2, 4, 0, None) == bad
    assert lib.cgb200_distill_fwd(p, 4, p, p, 2, 0, 1.0, p, p + 8, 2, 4, 0, None) == bad
    assert lib.cgb200_distill_bwd(p, 4, p, p, 2, 0, 1.0, None, p, p, 2, 4, 0, None) == bad


def test_network_without_a_head_has_no_answers():
    from cgnet_b200 import SphericalCNN
    net = SphericalCNN.__new__(SphericalCNN)
    torch.nn.Module.__init__(net)
    net.head = None
    with pytest.raises(RuntimeError, match="head"):
        net.log_probs(None)
    with pytest.raises(RuntimeError, match="head"):
        net.distillation_loss(None, None, None)
