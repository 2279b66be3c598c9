"""Tensor-core products of the gated block: blocks with several tiles, and what one tile leaves behind for the next."""
import pytest
import torch

from test_gpu_head import check_ff, gen, randn

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
