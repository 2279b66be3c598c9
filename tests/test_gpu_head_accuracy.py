"""Accuracy of the gated block's tensor-core products by themselves, through the C interface: the kept projections g and u, and the
backward's products with g = u = 1 kept and relu, where dg = du = dh exactly."""
import pytest
import torch

from test_gpu_head import U, gen, half, randn

pytestmark = pytest.mark.gpu


def stream():
    return torch.cuda.current_stream().cuda_stream


def operands(x, wg, wu):
    return x.data_ptr(), x.stride(0), wg.data_ptr(), wg.stride(0), wu.data_ptr(), wu.stride(0)


def workspace(lib, x, wg, wu, code, gradients):
    n = lib.cgb200_gated_ff_workspace_bytes(*operands(x, wg, wu), x.shape[0], x.shape[1], wg.shape[0], code, gradients)
    assert n >= 0
    return torch.empty(max(n, 1), dtype=torch.uint8, device=x.device)


def code_of(t):
    from cgnet_b200 import _lib
    return {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}[t]


def projections(x, wg, wu):
    from cgnet_b200 import _lib
    lib, code, (rows, dim), hidden = _lib.load(), code_of(x.dtype), x.shape, wg.shape[0]
    pitch = -(-hidden // 4) * 4
    kept, h, ws = torch.empty(2, rows, pitch, device=x.device), torch.empty(rows, hidden, dtype=x.dtype, device=x.device), workspace(lib, x, wg, wu, code, 0)
    assert lib.cgb200_gated_ff_fwd(*operands(x, wg, wu), 2, h.data_ptr(), kept.data_ptr(), rows, dim, hidden, code, ws.data_ptr(), ws.numel(), stream()) == 0
    return kept[0, :, :hidden], kept[1, :, :hidden]


def gradients(x, wg, wu, dh, kept=None):
    """dx, dWg, dWu for relu; g = u = 1 unless given as [2][rows][pitch]."""
    from cgnet_b200 import _lib
    lib, code, (rows, dim), hidden = _lib.load(), code_of(x.dtype), x.shape, wg.shape[0]
    if kept is None:
        kept = torch.ones(2, rows, -(-hidden // 4) * 4, device=x.device)
    dx, dwg, dwu, ws = torch.empty_like(x), torch.empty_like(wg), torch.empty_like(wu), workspace(lib, x, wg, wu, code, 7)
    assert lib.cgb200_gated_ff_bwd(*operands(x, wg, wu), 2, kept.data_ptr(), dh.data_ptr(), dh.stride(0), dx.data_ptr(), dwg.data_ptr(), dwu.data_ptr(), rows,
                                   dim, hidden, code, ws.data_ptr(), ws.numel(), stream()) == 0, lib.cgb200_last_error()
    return dx, dwg, dwu


def rms(t):
    return float((t.double() ** 2).mean().sqrt())


# the fused forward with one and with both accumulators and several tiles a block; the split one; both layouts of the backward
SIZES = [(700, 520, 700), (1200, 2048, 900), (156, 1330, 342), (300, 4096, 128)]


@pytest.mark.parametrize("rows, dim, hidden", SIZES)
def test_float32_products_are_off_by_roundings_of_float32(rows, dim, hidden):
    """Root mean square of the error over that of sqrt(sum (a b)^2), which a random walk of roundings scales with.

    A flush holds 16 truncating additions of 16 terms each; addition j is off by at most one step, 2 u |acc|, with |acc| about
    sqrt(16 j): together 2 u * 4 * sum sqrt(j) = 358 u against sqrt(256) = 16, that is 22 u, and flushes are independent of one another.
    Their sum in registers, the parts of a split and the products left out (2 u at most, random) add less than 5 u.  Products
    formed from planes on the CPU are off by 0.1 u so, by 41 without the third plane of one operand, 58 without either, 46 without the
    product of the second ones."""
    g = gen(rows + dim + hidden)
    x, wg, wu, dh = randn(g, rows, dim), randn(g, hidden, dim), randn(g, hidden, dim), randn(g, rows, hidden)
    x64, wg64, wu64, dh64 = (t.double() for t in (x, wg, wu, dh))
    p, q = projections(x, wg, wu)
    dx, dwg, dwu = gradients(x, wg, wu, dh)
    for name, got, want, square in (("g", p, x64 @ wg64.t(), x64 ** 2 @ wg64.t() ** 2), ("u", q, x64 @ wu64.t(), x64 ** 2 @ wu64.t() ** 2),
                                    ("dx", dx, dh64 @ (wg64 + wu64), dh64 ** 2 @ (wg64 ** 2 + wu64 ** 2)),
                                    ("dwg", dwg, dh64.t() @ x64, dh64.t() ** 2 @ x64 ** 2), ("dwu", dwu, dh64.t() @ x64, dh64.t() ** 2 @ x64 ** 2)):
        off = rms(got - want) / rms(square.sqrt())
        assert off <= 32 * U, f"{name}: {off / U:.1f} u"


@pytest.mark.parametrize("rows, dim, hidden", SIZES)
def test_float32_products_of_two_terms(rows, dim, hidden):
    """Rows with two values each, the second nearly the first's negative times the weights' ratio where it matters most: the leading planes
    cancel and the result is what the small ones hold.  Adding zeros is exact, so an output of n terms is off by at most 2 n u of
    its absolute sum, 2 u for the products left out, and the roundings of lead + rest and of the sum of flushes or parts.  (Planes on the
    CPU: 0.6 u; 85 to 197 without one of the small products.)"""
    g = gen(rows * 3 + dim + hidden)

    def sparse(r, c):
        t = torch.zeros(r, c, device="cuda")
        at = torch.stack([torch.randperm(c, generator=g, device="cuda")[:2] for _ in range(r)])
        v = 1 + torch.rand(r, 1, generator=g, device="cuda")
        pair = torch.cat([v, -v * (1 + 2.0 ** -9 * torch.rand(r, 1, generator=g, device="cuda"))], 1)
        return t.scatter_(1, at, pair)
    x, dh = sparse(rows, dim), sparse(rows, hidden)
    # all weights of a row nearly the same
    wg = (1 + torch.rand(hidden, 1, generator=g, device="cuda")) * (1 + 2.0 ** -9 * torch.rand(hidden, dim, generator=g, device="cuda"))
    wu = (1 + torch.rand(hidden, 1, generator=g, device="cuda")) * (1 + 2.0 ** -9 * torch.rand(hidden, dim, generator=g, device="cuda"))
    x64, wg64, wu64, dh64 = (t.double() for t in (x, wg, wu, dh))
    p, q = projections(x, wg, wu)
    dx, dwg, dwu = gradients(x, wg, wu, dh)

    def check(name, got, want, size, terms):
        off = (got.double() - want).abs() - (2 * terms + 5) * U * size
        assert float(off.max()) <= 0, f"{name}: {float(((got.double() - want).abs() / size.clamp(min=1e-30)).max()) / U:.1f} u"
    ax, adh, nx, ndh = x64.abs(), dh64.abs(), (x64 != 0).double(), (dh64 != 0).double()
    check("g", p, x64 @ wg64.t(), ax @ wg64.t(), 2)
    check("u", q, x64 @ wu64.t(), ax @ wu64.t(), 2)
    check("dx", dx, dh64 @ (wg64 + wu64), adh @ (wg64 + wu64), 4)
    for name, got in (("dwg", dwg), ("dwu", dwu)):
        check(name, got, dh64.t() @ x64, adh.t() @ ax, ndh.t() @ nx)


# CUDA cores; tensor cores with rows and units that fill no tile; several tiles with split and with whole contractions; one row, one unit
RANGE_SIZES = [(100, 64, 64), (300, 104, 200), (1111, 1000, 1365), (700, 64, 24), (3000, 48, 9), (5, 40, 800), (2000, 520, 1032)]


def range_bounds(x, wg, wu, dh, kept):
    """dx, dWg, dWu of relu with their bounds: dg and du are off by 4 u (float32) and by half a step of fp16.  Half a subnormal step is 2^-25; where
    the row's (dx) or the unit's (dW) largest value is 2^-4 or more that is 2^-21 of it at most, else 2^-25 of the power of two that brings
    it to 2^14: 2^-39."""
    x, wg, wu, dh, g, u = (t.double() for t in (x, wg, wu, dh, kept[0], kept[1]))
    dg, du = dh * u * (g > 0), dh * g.clamp(min=0)
    e = half(torch.float16) + 4 * U
    most = torch.maximum(dg.abs().amax(1), du.abs().amax(1))[:, None]
    edg, edu = e * dg.abs() + 2.0 ** -21 * most, e * du.abs() + 2.0 ** -21 * most
    rows, hidden = dh.shape
    out = [(dg @ wg + du @ wu, edg @ wg.abs() + edu @ wu.abs() + (4 * hidden + 8) * U * (dg.abs() @ wg.abs() + du.abs() @ wu.abs()))]
    for d in (dg, du):
        ed = e * d.abs() + 2.0 ** -21 * d.abs().amax(0)
        out.append((d.t() @ x, ed.t() @ x.abs() + (2 * rows + 8) * U * (d.abs().t() @ x.abs())))
    return out


def check_range(x, wg, wu, dh, kept):
    got = gradients(x, wg, wu, dh, kept)
    for name, q, (want, tol) in zip(("dx", "dwg", "dwu"), got, range_bounds(x, wg, wu, dh, kept[:, :, :dh.shape[1]])):
        assert float(want.abs().max()) < 6e4, "the case itself leaves the range"
        off = (q.double() - want).abs() - tol - half(torch.float16) * (want.abs() + tol) - 2.0 ** -25
        assert float(off.max()) <= 0, (name, float(off.max()), bool(torch.isfinite(q).all()))


@pytest.mark.parametrize("rows, dim, hidden", RANGE_SIZES)
@pytest.mark.parametrize("case", ["large", "small", "rows", "units", "last", "zeros"])
def test_half_precision_gradients_whose_factors_leave_its_range(case, rows, dim, hidden):
    """dg and du beyond 65504 or below 6e-8 behind gradients that are neither, in all rows, in some rows, in some units."""
    g = gen(rows + dim + hidden)
    pitch = -(-hidden // 4) * 4
    x, wg, wu, dh, kept = randn(g, rows, dim), randn(g, hidden, dim), randn(g, hidden, dim), randn(g, rows, hidden), randn(g, 2, rows, pitch)
    few = torch.arange(rows, device="cuda") % 7 == 0
    if case == "last":          # one row, in the last tile of rows, and the units that it makes large
        few = torch.arange(rows, device="cuda") == rows - 1
    if case == "large":
        dh, kept, wg, wu, x = 300 * dh, 300 * kept, 1e-4 * wg, 1e-4 * wu, 1e-4 * x
    elif case == "small":
        dh, kept, x, wg, wu = 3e-7 * dh, 0.1 * kept, 300 * x, 300 * wg, 300 * wu
    elif case in ("rows", "last"):        # large rows with small inputs beside small rows with ordinary ones
        size = torch.where(few, 3e2, 1e-4)[:, None]
        dh, kept, wg, wu, x = size * dh, torch.where(few, 300.0, 1.0)[:, None] * kept, 1e-3 * wg, 1e-3 * wu, torch.where(few, 1e-4, 1.0)[:, None] * x
    elif case == "units":
        some = torch.arange(hidden, device="cuda") % 5 == 1
        wide = torch.arange(pitch, device="cuda") % 5 == 1
        dh, kept = torch.where(some, 300.0, 1e-5) * dh, torch.where(wide, 300.0, 1.0) * kept
        wg, wu, x = torch.where(some, 1e-4, 1.0)[:, None] * wg, torch.where(some, 1e-4, 1.0)[:, None] * wu, 1e-3 * x
    else:
        dh = torch.where(few[:, None], dh, torch.zeros_like(dh))
        dh[:, ::3] = 0
    x, wg, wu, dh = (t.half() for t in (x, wg, wu, dh))
    check_range(x, wg, wu, dh, kept)


@pytest.mark.parametrize("rows, dim, hidden", RANGE_SIZES)
def test_half_precision_infinities_stay_in_their_row_and_unit(rows, dim, hidden):
    g = gen(rows + dim + hidden)
    x, wg, wu, dh = (t.half() for t in (randn(g, rows, dim), randn(g, hidden, dim) / 8, randn(g, hidden, dim) / 8, randn(g, rows, hidden)))
    kept = randn(g, 2, rows, -(-hidden // 4) * 4).abs() + 0.1
    want = gradients(x, wg, wu, dh, kept)
    bad = dh.clone()
    bad[2, 3], bad[4, 5] = float("inf"), float("nan")
    got = gradients(x, wg, wu, bad, kept)
    rows_left = [r for r in range(rows) if r not in (2, 4)]
    units_left = [j for j in range(hidden) if j not in (3, 5)]
    assert torch.equal(got[0][rows_left], want[0][rows_left]) and not torch.isfinite(got[0][[2, 4]]).any()
    for p, q in zip(got[1:], want[1:]):
        assert torch.equal(p[units_left], q[units_left]) and not torch.isfinite(p[[3, 5]]).any()


@pytest.mark.parametrize("gradient", [1, 2, 4, 3, 5, 6])
def test_half_precision_gradients_one_by_one(gradient):
    """Only the copies that a call's gradients need are made: the same bits as all of them together."""
    import cgnet_b200 as cg
    g = gen(gradient)
    x, wg, wu, dh = (t.half() for t in (randn(g, 300, 104), randn(g, 200, 104) / 8, randn(g, 200, 104) / 8, 300 * randn(g, 300, 200)))
    full = [t.clone().requires_grad_() for t in (x, wg, wu)]
    want = torch.autograd.grad(cg.gated_feed_forward(*full, activation="relu"), full, dh)
    part = [t.clone().requires_grad_(bool(gradient >> i & 1)) for i, t in enumerate((x, wg, wu))]
    got = torch.autograd.grad(cg.gated_feed_forward(*part, activation="relu"), [t for t in part if t.requires_grad], dh)
    assert all(torch.equal(p, q) for p, q in zip(got, [w for w, t in zip(want, part) if t.requires_grad]))


@pytest.mark.parametrize("dtype, terms", [(torch.bfloat16, 32768), (torch.float16, 16384)])
def test_long_sums_of_one_sign(dtype, terms):
    """The tensor core truncates as it adds, so a sum of one sign comes out low, the more the longer it is.  In parts of at most `terms` terms
    its relative error is no more than the largest of its parts', and one rounding for each part.  How far a sum of `terms` terms is off
    is measured by a call of that length; a part of the same length may be off twice as far, for a step of float32 is between u and
    2 u of a value, depending on where the sum ends."""
    def positive(g, *shape):
        return (1 + torch.rand(*shape, generator=g, device="cuda")).to(dtype)
    # a forward of more tiles than are split to fill the SMs
    g, rows, dim, hidden = gen(1), 5000, 65560, 130
    x, w = positive(g, rows, dim), positive(g, hidden, dim)
    some = torch.cat([torch.arange(150), torch.arange(rows - 150, rows)])

    def error(n):
        want = sum(x[some, i:min(i + 8192, n)].double() @ w[:, i:min(i + 8192, n)].double().t() for i in range(0, n, 8192))
        return max(float(((got[some].double() - want) / want).abs().max()) for got in projections(x[:, :n], w[:, :n], w[:, :n]))
    one = error(terms)
    assert one <= half(dtype) / 4, one / U
    assert error(dim) <= 2 * one + (dim / terms + 8) * U
    # weights' gradients; rounding them is random over the 64 x 64 values: half a step / sqrt(3) / 64, five times that at most
    rows, dim, hidden = 1 << 19, 64, 64
    size = 1 + torch.arange(64, device="cuda") / 64
    x, dh = (2.0 ** -9 * size * positive(g, rows, dim).float()).to(dtype), (2.0 ** -7 * size * positive(g, rows, hidden).float()).to(dtype)
    w = torch.zeros(hidden, dim, dtype=dtype, device="cuda")
    want = dh.double().t() @ x.double()
    for got in gradients(x, w, w, dh)[1:]:
        off = abs(float(((got.double() - want) / want).mean()))
        assert off <= 2 * one + (rows / terms + 8) * U + 5 * half(dtype) / 3 ** 0.5 / 64, off / U


def test_half_precision_backward_in_a_captured_graph():
    """One graph, replayed with gradients inside, above and below the range: which tiles are scaled is decided on the GPU."""
    import cgnet_b200 as cg
    g = gen(3)
    x, wg, wu, dh = (t.half() for t in (randn(g, 300, 104), randn(g, 264, 104) / 10, randn(g, 264, 104) / 10, randn(g, 300, 264)))
    leaves = [t.requires_grad_() for t in (x, wg, wu)]

    def step():
        return torch.autograd.grad(cg.gated_feed_forward(*leaves, activation="gelu"), leaves, dh)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = step()
    for size in (1.0, 1e-5, 1e4, 1.0):
        new = size * randn(g, 300, 264)
        new[130:] = new[130:].clamp(-1, 1)
        dh.copy_(new)
        graph.replay()
        assert all(torch.equal(p.nan_to_num(7.0), q.nan_to_num(7.0)) for p, q in zip(grads, step())), size
