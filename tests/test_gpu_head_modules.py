"""The classifier head in the types it can be built in, on the embedding of a network, which is float32."""
import pytest
import torch

from test_gpu_head import TYPES, gen, half, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
def test_head_of_any_type_on_a_float32_embedding(dtype):
    import cgnet_b200 as cg
    torch.manual_seed(3)
    x = randn(gen(1), 33, 52).requires_grad_()
    head = cg.InvariantHead(52, 128, 10, dtype=dtype)
    logits = head(x)
    assert logits.dtype == dtype and logits.shape == (33, 10)
    (gx,) = torch.autograd.grad(cg.log_probs(logits).entropy.sum(), x)
    assert gx.dtype == torch.float32 and torch.isfinite(gx).all() and float(gx.abs().sum()) > 0
    y = torch.nn.functional.layer_norm(x.detach().double(), (52,))
    a, b = y @ head.ff.w_gate.double().t(), y @ head.ff.w_up.double().t()
    h = torch.nn.functional.silu(a) * b
    want = h @ head.scores.weight.double().t() + head.scores.bias.double()
    # four roundings to the type on the way (embedding, norm, hidden layer, logits): an error e of y is at most 52 e |w| |y| of a and b
    e = 2 * half(dtype) + 60 * 2.0 ** -24
    ay = y.abs() + 1
    ea, eb = e * ay @ head.ff.w_gate.double().abs().t(), e * ay @ head.ff.w_up.double().abs().t()
    eh = 1.2 * ea * (b.abs() + eb) + a.abs() * eb + e * h.abs()
    tol = eh @ head.scores.weight.double().abs().t() + e * (h.abs() @ head.scores.weight.double().abs().t() + want.abs())
    assert bool(((logits.double() - want).abs() <= tol).all())
