"""Tensor-core products of the gated block: blocks with several tiles, and what one tile leaves behind for the next."""
import pytest
import torch

from test_gpu_head import TYPES, check_ff, gen, randn

pytestmark = pytest.mark.gpu


def operands(rows, dim, hidden, dtype):
    g = gen(rows + dim + hidden)
    return (randn(g, rows, dim).to(dtype), (randn(g, hidden, dim) * dim ** -0.5).to(dtype), (randn(g, hidden, dim) * dim ** -0.5).to(dtype),
            randn(g, rows, hidden).to(dtype))


@pytest.mark.parametrize("rows, dim, hidden", [(1000, 600, 1400), (2000, 516, 1300), (129, 1100, 5000)])
def test_float32_forward_of_several_tiles_a_block(rows, dim, hidden):
    """More than 148 tiles of 128 x 64 and more than four flushes each: every block uses both accumulators, and reads one while the
    other is written."""
    x, wg, wu, dh = operands(rows, dim, hidden, torch.float32)
    check_ff(x, wg, wu, "silu", dh)
    import cgnet_b200 as cg
    with torch.no_grad():
        h = cg.gated_feed_forward(x, wg, wu)
        assert all(torch.equal(cg.gated_feed_forward(x, wg, wu), h) for _ in range(5))


# (rows, dim, hidden): one of dx and [dWg; dWu] leaves by bulk copies, the other in parts written by threads, and some blocks have a
# unit of the former directly before one of the latter.  dx first: the first four; dW first: the others.
MIXED = [(1652, 880, 288), (4096, 512, 512), (1904, 856, 259), (6180, 296, 775), (1052, 144, 3415), (2901, 360, 4644)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows, dim, hidden", MIXED)
def test_backward_units_that_leave_in_different_ways(rows, dim, hidden, dtype):
    import cgnet_b200 as cg
    x, wg, wu, dh = operands(rows, dim, hidden, dtype)
    check_ff(x, wg, wu, "gelu", dh)
    h = cg.gated_feed_forward(x, wg, wu, activation="gelu")
    grads = torch.autograd.grad(h, (x, wg, wu), dh, retain_graph=True)
    for _ in range(10):
        assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(h, (x, wg, wu), dh, retain_graph=True), grads))


def test_weight_gradients_of_different_alignment():
    """The C interface takes outputs of any alignment: one gradient leaves by copies, the other is written by threads, one stage apart."""
    from cgnet_b200 import _lib
    lib, rows, dim, hidden = _lib.load(), 64, 1024, 4096
    x, wg, wu, dh = operands(rows, dim, hidden, torch.bfloat16)
    gate_up = torch.empty(2, rows, hidden, device=x.device)
    h, ws = torch.empty_like(dh), torch.empty(1 << 24, dtype=torch.uint8, device=x.device)
    stream = torch.cuda.current_stream().cuda_stream
    operand_args = (x.data_ptr(), dim, wg.data_ptr(), dim, wu.data_ptr(), dim)
    assert lib.cgb200_gated_ff_fwd(*operand_args, 0, h.data_ptr(), gate_up.data_ptr(), rows, dim, hidden, _lib.BF16, ws.data_ptr(), ws.numel(), stream) == 0

    def gradients(offset):
        gate, upper = (torch.zeros(hidden * dim + 8, dtype=torch.bfloat16, device=x.device) for _ in range(2))
        out = upper[offset:offset + hidden * dim]
        assert lib.cgb200_gated_ff_bwd(*operand_args, 0, gate_up.data_ptr(), dh.data_ptr(), hidden, None, gate.data_ptr(), out.data_ptr(), rows, dim,
                                       hidden, _lib.BF16, ws.data_ptr(), ws.numel(), stream) == 0, lib.cgb200_last_error()
        assert not upper[:offset].any() and not upper[offset + hidden * dim:].any()
        return gate, out
    want = gradients(0)
    for _ in range(10):
        assert all(torch.equal(p, q) for p, q in zip(gradients(1), want))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, dim, hidden", [(3, 100, 50), (40, 60, 70), (300, 520, 400), (20, 1100, 90)])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_values_that_are_not_finite_stay_in_their_row_and_unit(rows, dim, hidden, dtype, bad):
    """In float32 on the tensor cores an infinite term makes NaN of what may be an infinity, everywhere else it is the formula's."""
    import cgnet_b200 as cg
    x, wg, wu, _ = operands(rows, dim, hidden, dtype)
    want = cg.gated_feed_forward(x, wg, wu, activation="relu")
    xb, wb = x.clone(), wu.clone()
    xb[2, 5], wb[7, 3] = bad, bad
    got = cg.gated_feed_forward(xb, wg, wb, activation="relu")
    r, u = [i for i in range(rows) if i != 2], [j for j in range(hidden) if j != 7]
    assert torch.equal(got[r][:, u], want[r][:, u])
    g, up = xb.double() @ wg.double().t(), xb.double() @ wb.double().t()
    formula = (g.clamp(min=0) * up)
    spoilt = ~torch.isfinite(formula)
    assert not torch.isfinite(got[spoilt]).any() and spoilt[r, 7].sum() > 0 and spoilt[2].sum() > 0
    if dtype != torch.float32 or dim < 512:
        assert torch.equal(torch.isnan(got), torch.isnan(formula)) and torch.equal(torch.isinf(got), torch.isinf(formula))
