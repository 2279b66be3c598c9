"""Operators behind the invariant embedding against plain implementations in 64 bits.

Tolerances follow from counting roundings.  u = 2^-24 is half a step of float32 relative to a value, half(t) half a step of the
result's type; a float32 sum of n terms of absolute sum S is off by at most n u S in any order, and a sum on the tensor cores, whose
accumulator truncates, by at most 2 n u S.  Every test evaluates these bounds in 64 bits beside the reference.
"""
import itertools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half(t):
    return torch.finfo(t).eps / 2


def cuda():
    return torch.device("cuda", 0)


def gen(seed):
    g = torch.Generator(device=cuda())
    g.manual_seed(seed)
    return g


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device=cuda())


def assert_within(got, want, tol, what):
    """|got - want| <= tol elementwise; NaN and infinities have to be the same ones.  Subnormal results of 16-bit types are
    rounded in absolute steps: one smallest step is allowed."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), what
    tol = tol.expand_as(want) if isinstance(tol, torch.Tensor) else torch.full_like(want, tol)
    off = ((got - want).abs() - tol)[fine]
    if off.numel():
        i = off.argmax()
        assert off[i] <= 0, f"{what}: off by {float((got - want).abs()[fine][i]):.3e}, tolerance {float(tol[fine][i]):.3e}, value {float(want[fine][i]):.3e}"


# ---------------------------------------------------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------------------------------------------------
def norm_reference(x, w, b, eps, dy=None):
    x = x.double()
    n = x.shape[-1]
    one = torch.ones(n, device=x.device, dtype=torch.float64)
    w64 = one if w is None else w.double()
    b64 = 0 * one if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    # a row's sums have at most 32 values a thread and 10 joining steps (long rows: dim / 1024 + 10), so the mean is off by that many
    # u of mean |x|; rstd by as many relative u and a few more
    steps = max(32, n // 1024 + 1) + 16
    xh_abs = rstd * (x.abs().mean(-1, keepdim=True) + x.abs() + mean.abs()) + xh.abs()
    y = xh * w64 + b64
    out = {"y": (y, 2 * steps * U * (w64.abs() * xh_abs + b64.abs()))}
    if dy is not None:
        g = dy.double()
        wg = g * w64
        m1, m2 = wg.mean(-1, keepdim=True), (wg * xh).mean(-1, keepdim=True)
        out["dx"] = (rstd * (wg - m1 - xh * m2),
                     6 * steps * U * rstd * (wg.abs() + wg.abs().mean(-1, keepdim=True) + xh_abs * (wg.abs() * xh_abs).mean(-1, keepdim=True)))
        rows = x.reshape(-1, n).shape[0]
        out["dw"] = ((g * xh).reshape(-1, n).sum(0), (4 * steps + rows) * U * (g.abs() * xh_abs).reshape(-1, n).sum(0))
        out["db"] = (g.reshape(-1, n).sum(0), (4 + rows) * U * g.abs().reshape(-1, n).sum(0))
    return out


def check_norm(x, w, b, eps, dy):
    import cgnet_b200 as cg
    leaves = [t for t in (x, w, b) if t is not None]
    for t in leaves:
        t.requires_grad_()
    y = cg.layer_norm(x, w, b, eps)
    assert y.dtype == x.dtype and y.shape == x.shape
    with torch.no_grad():
        assert torch.equal(cg.layer_norm(x, w, b, eps), y)
    grads = torch.autograd.grad(y, leaves, dy)
    ref = norm_reference(x.detach(), w, b, eps, dy)
    names = [n for n, t in (("dx", x), ("dw", w), ("db", b)) if t is not None]
    for name, got in [("y", y.detach())] + list(zip(names, grads)):
        want, tol = ref[name]
        assert_within(got, want, tol + half(got.dtype) * (want.abs() + tol) + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps, name)
    again = torch.autograd.grad(cg.layer_norm(x, w, b, eps), leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(grads, again)), "not the same bits"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, dim", [(1, 1), (3, 1), (2, 2), (5, 7), (100, 52), (1, 52), (64, 512), (700, 40), (33, 513), (9, 1023), (40, 1024),
                                       (3, 1025), (2000, 96), (5, 4096), (7, 4097), (3, 8192), (2, 8200), (700, 8201), (3, 16385), (2, 33000)])
def test_layer_norm(rows, dim, dtype):
    g = gen(rows * 7 + dim)
    x = ((randn(g, rows, dim) + randn(g, rows, 1)) * torch.exp(randn(g, rows, 1))).to(dtype)
    check_norm(x, (1 + 0.2 * randn(g, dim)).to(dtype), randn(g, dim).to(dtype), 1e-5, randn(g, rows, dim).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("weight, bias", [(False, False), (True, False), (False, True)])
def test_layer_norm_without_parameters_and_with_float32_ones(dtype, weight, bias):
    g = gen(3)
    for dim in (52, 777, 2048):
        w = 1 + 0.2 * randn(g, dim) if weight else None      # float32 beside 16-bit activations
        b = randn(g, dim) if bias else None
        check_norm(randn(g, 11, dim).to(dtype), w, b, 1e-3, randn(g, 11, dim).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1023, 2049, 4097, 8200, 16381])
def test_layer_norm_long_rows_with_float32_weights(dim, dtype):
    """Rows of a warp and of a block that end inside a group, and weights that start on and off 16-byte boundaries."""
    g = gen(dim)
    for lo in (0, 1, 3):
        w, b = (1 + 0.2 * randn(g, dim + lo))[lo:], randn(g, dim + lo)[lo:]
        check_norm((randn(g, 7, dim) + randn(g, 7, 1)).to(dtype), w, b, 1e-5, randn(g, 7, dim).to(dtype))
        check_norm((randn(g, 7, dim + 2) + randn(g, 7, 1)).to(dtype)[:, 1:dim + 1], w.to(dtype), b.to(dtype), 1e-5, randn(g, 7, dim).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_layouts(dtype):
    """Rows inside wider rows, rows that start anywhere, transposed and broadcast inputs, more than two dimensions."""
    g = gen(5)
    for wide, lo, dim in ((70, 3, 52), (1200, 8, 1000), (4200, 1, 4099)):
        full = randn(g, 6, wide).to(dtype)
        check_norm(full[:, lo:lo + dim], randn(g, dim).to(dtype), randn(g, dim).to(dtype), 1e-5, randn(g, 6, wide).to(dtype)[:, 1:1 + dim])
    check_norm(randn(g, 52, 9).to(dtype).t(), None, None, 1e-5, randn(g, 9, 52).to(dtype))
    check_norm(randn(g, 1, 64).to(dtype).expand(5, 64), randn(g, 64).to(dtype), None, 1e-5, randn(g, 1, 64).to(dtype).expand(5, 64))
    check_norm(randn(g, 2, 3, 40).to(dtype), randn(g, 40).to(dtype), randn(g, 40).to(dtype), 1e-5, randn(g, 2, 3, 40).to(dtype))
    check_norm(randn(g, 40).to(dtype), randn(g, 40).to(dtype), randn(g, 40).to(dtype), 1e-5, randn(g, 40).to(dtype))


def test_layer_norm_offsets_constants_and_nan():
    import cgnet_b200 as cg
    g = gen(7)
    # a common offset a thousand times the spread: a difference of moments would leave no digit
    check_norm(randn(g, 8, 300) + 1000.0, randn(g, 300), randn(g, 300), 1e-5, randn(g, 8, 300))
    check_norm(torch.full((4, 64), 3.0, device=cuda()), randn(g, 64), randn(g, 64), 1e-5, randn(g, 4, 64))
    x = randn(g, 4, 64)
    x[1, 5], x[2, 6] = float("nan"), float("inf")
    y = cg.layer_norm(x, torch.ones(64, device=cuda()))
    assert torch.isnan(y[1]).all() and torch.isnan(y[2]).all() and torch.isfinite(y[0]).all() and torch.isfinite(y[3]).all()


def test_layer_norm_no_rows():
    import cgnet_b200 as cg
    x = torch.empty(0, 33, device=cuda(), requires_grad=True)
    w, b = torch.ones(33, device=cuda(), requires_grad=True), torch.zeros(33, device=cuda(), requires_grad=True)
    y = cg.layer_norm(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert gx.shape == (0, 33) and torch.equal(gw, torch.zeros_like(w)) and torch.equal(gb, torch.zeros_like(b))


# ---------------------------------------------------------------------------------------------------------------------
# gated feed-forward block
# ---------------------------------------------------------------------------------------------------------------------
def act64(name, g):
    if name == "relu":
        return g.clamp(min=0), (g > 0).double()
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    c = torch.special.ndtr(g)
    return g * c, c + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)


def ff_reference(x, wg, wu, act, dh, dtype):
    """Values and bounds.  A product over n terms is off by 2 n u of its absolute sum (float32 on the tensor cores: 24 bits in three
    parts, of whose nine products the three below 2^-24 are left out: 3 u more); the activations are off by (8 + 4 |g|) u of
    their size, their slopes are at most 1.2; dg and du are rounded to the inputs' type before the second products."""
    x, wg, wu, dh = x.double(), wg.double(), wu.double(), dh.double()
    rows, dim = x.shape
    hidden = wg.shape[0]
    g, u = x @ wg.t(), x @ wu.t()
    ga, ua = x.abs() @ wg.abs().t(), x.abs() @ wu.abs().t()
    a, da = act64(act, g)
    eg, eu = (2 * dim + 8) * U * ga, (2 * dim + 8) * U * ua
    ea = 1.2 * eg + (8 + 4 * g.abs()) * U * (a.abs() + g.abs() * U)
    out = {"h": (a * u, ea * (u.abs() + eu) + a.abs() * eu + 4 * U * (a * u).abs())}
    dg, du = dh * u * da, dh * a
    # slopes change by at most 1.2 per unit of g (relu: they jump at 0, where g may land on either side)
    eda = 1.2 * eg + (8 + 4 * g.abs()) * U * 1.2
    if act == "relu":
        eda = torch.where(g.abs() <= eg, torch.ones_like(g), torch.zeros_like(g))
    edg = dh.abs() * (eu * (da.abs() + eda) + u.abs() * eda) + 4 * U * dg.abs()
    edu = dh.abs() * ea + 4 * U * du.abs()
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    edg, edu = edg + half(dtype) * (dg.abs() + edg) + tiny, edu + half(dtype) * (du.abs() + edu) + tiny
    out["dx"] = (dg @ wg + du @ wu, edg @ wg.abs() + edu @ wu.abs() + (4 * hidden + 8) * U * (dg.abs() @ wg.abs() + du.abs() @ wu.abs()))
    for name, d, ed in (("dwg", dg, edg), ("dwu", du, edu)):
        out[name] = (d.t() @ x, ed.t() @ x.abs() + (2 * rows + 8) * U * (d.abs().t() @ x.abs()))
    return out


def check_ff(x, wg, wu, act, dh):
    import cgnet_b200 as cg
    for t in (x, wg, wu):
        t.requires_grad_()
    h = cg.gated_feed_forward(x, wg, wu, activation=act)
    assert h.dtype == x.dtype and h.shape == (x.shape[0], wg.shape[0])
    with torch.no_grad():
        assert torch.equal(cg.gated_feed_forward(x, wg, wu, activation=act), h)
    grads = torch.autograd.grad(h, (x, wg, wu), dh)
    ref = ff_reference(x.detach(), wg.detach(), wu.detach(), act, dh, x.dtype)
    for name, got in zip(("h", "dx", "dwg", "dwu"), (h.detach(), *grads)):
        want, tol = ref[name]
        t = got.dtype
        assert_within(got, want, tol + half(t) * (want.abs() + tol) + torch.finfo(t).smallest_normal * torch.finfo(t).eps, name)
    again = torch.autograd.grad(cg.gated_feed_forward(x, wg, wu, activation=act), (x, wg, wu), dh)
    assert all(torch.equal(p, q) for p, q in zip(grads, again)), "not the same bits"


FF_SIZES = [(1, 1, 1), (1, 52, 256), (2, 100, 33), (3, 65, 130), (4, 1000, 77), (5, 7, 3), (17, 130, 66), (100, 52, 256), (128, 64, 64), (130, 65, 129),
            (300, 256, 192), (257, 1000, 1365), (129, 128, 1032), (1500, 72, 40), (40, 2056, 264), (1025, 264, 520), (8, 4104, 1032)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, dim, hidden", FF_SIZES)
def test_gated_feed_forward(rows, dim, hidden, dtype):
    g = gen(rows + dim + hidden)
    act = ("silu", "gelu", "relu")[(rows + dim) % 3]
    check_ff(randn(g, rows, dim).to(dtype), (randn(g, hidden, dim) * dim ** -0.5).to(dtype), (randn(g, hidden, dim) * dim ** -0.5).to(dtype), act,
             randn(g, rows, hidden).to(dtype))


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("dtype", TYPES)
def test_gated_feed_forward_activations_and_layouts(act, dtype):
    """Large projections (saturated activations), and operands inside wider rows, transposed, or broadcast."""
    g = gen(11)
    check_ff((4 * randn(g, 70, 40)).to(dtype), randn(g, 96, 40).to(dtype), randn(g, 96, 40).to(dtype), act, randn(g, 70, 96).to(dtype))
    for rows in (3, 150):
        check_ff(randn(g, rows, 300).to(dtype)[:, 5:261], (randn(g, 200, 299) / 16).to(dtype)[:, 1:257], (randn(g, 256, 200) / 16).to(dtype).t(), act,
                 randn(g, rows, 260).to(dtype)[:, 3:203])
    check_ff(randn(g, 1, 64).to(dtype).expand(9, 64), (randn(g, 80, 64) / 8).to(dtype), (randn(g, 80, 64) / 8).to(dtype), act,
             randn(g, 1, 80).to(dtype).expand(9, 80))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, dim, hidden", [(5, 1031, 70), (156, 1330, 342), (129, 1024, 257), (16, 520, 1000), (500, 2048, 128)])
def test_gated_feed_forward_of_few_tiles(rows, dim, hidden, dtype):
    """A forward whose contraction is split over blocks, with and without the projections kept for a backward."""
    g = gen(rows + dim + hidden)
    check_ff(randn(g, rows, dim).to(dtype), (randn(g, hidden, dim) * dim ** -0.5).to(dtype), (randn(g, hidden, dim) * dim ** -0.5).to(dtype),
             ("silu", "gelu", "relu")[rows % 3], randn(g, rows, hidden).to(dtype))


def test_gated_feed_forward_parts_and_shapes():
    """Only the gradients asked for; leading dimensions; no rows; a bad row spoils no other."""
    import cgnet_b200 as cg
    g = gen(13)
    for rows, dim, hidden in ((6, 20, 30), (256, 256, 256)):
        x, wg, wu = randn(g, rows, dim), randn(g, hidden, dim) / 8, randn(g, hidden, dim) / 8
        dh = randn(g, rows, hidden)
        full = [t.clone().requires_grad_() for t in (x, wg, wu)]
        want = torch.autograd.grad(cg.gated_feed_forward(*full), full, dh)
        for mask in itertools.product((False, True), repeat=3):
            if any(mask):
                part = [t.clone().requires_grad_(m) for t, m in zip((x, wg, wu), mask)]
                got = torch.autograd.grad(cg.gated_feed_forward(*part), [t for t, m in zip(part, mask) if m], dh)
                assert all(torch.equal(p, q) for p, q in zip(got, [w for w, m in zip(want, mask) if m]))
        x3 = torch.cat([x, x]).view(2, rows, dim)
        assert torch.equal(cg.gated_feed_forward(x3, wg, wu)[1], cg.gated_feed_forward(torch.cat([x, x]), wg, wu)[rows:])
        bad = x.clone()
        bad[3, 2] = float("nan")
        h = cg.gated_feed_forward(bad, wg, wu)
        keep = [i for i in range(rows) if i != 3]
        assert torch.isnan(h[3]).all() and torch.equal(h[keep], cg.gated_feed_forward(x, wg, wu)[keep])
    x0 = torch.empty(0, 20, device=cuda(), requires_grad=True)
    w = (randn(g, 30, 20) / 4).requires_grad_()
    h = cg.gated_feed_forward(x0, w, w)
    gx, gw = torch.autograd.grad(h, (x0, w), torch.empty_like(h))
    assert h.shape == (0, 30) and gx.shape == (0, 20) and torch.equal(gw, torch.zeros_like(w))


# ---------------------------------------------------------------------------------------------------------------------
# log probabilities
# ---------------------------------------------------------------------------------------------------------------------
def softmax_bounds(z, temp=1.0):
    """log p in 64 bits and a bound on the relative error of float32 softmax terms: 2^-22 of ex2, and 2 u of the exponents
    y = z log2(e) / T (one for the factor's rounding, one for the difference's) that matter (p > 2^-60), and the sum's."""
    z = z.double() / temp
    m = z.max(-1, keepdim=True).values
    dead = m == float("-inf")
    logp = torch.where(dead, torch.full_like(z, float("-inf")), torch.log_softmax(torch.where(dead, torch.zeros_like(z), z), -1))
    seen = torch.where(logp > -42.0, z.abs(), torch.zeros_like(z)).nan_to_num(0.0, 0.0, 0.0).max(-1, keepdim=True).values
    steps = z.shape[-1] / 256 + 64
    return logp, 2.0 ** -22 + (2 * 2 * 1.4427 * (seen + 42.0) + steps) * U


def plogp(logp):
    p = logp.exp()
    return torch.where(p > 0, p * logp, torch.zeros_like(p))


def check_log_probs(z, target, top, g_lp=None, g_ent=None):
    import cgnet_b200 as cg
    rows, classes = z.shape
    logp, rel = softmax_bounds(z)
    bad = torch.isnan(logp).any(1)
    with torch.no_grad():
        out = cg.log_probs(z, target, top=top)
    order = torch.sort(z.double(), dim=1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(out.top_ids, order), "ranked classes"
    e1 = rel + 2 * U
    want = logp.gather(1, order)
    assert_within(out.top_log_probs, want, e1 + half(torch.float32) * want.abs().nan_to_num(0.0, 0.0, 0.0), "top_log_probs")
    if target is not None:
        want = torch.where(target >= 0, logp.gather(1, target.clamp(0, classes - 1)[:, None])[:, 0], torch.zeros(rows, device=z.device, dtype=torch.float64))
        want = torch.where(target >= classes, torch.full_like(want, float("nan")), want)
        assert_within(out.log_prob, want, e1[:, 0] + half(torch.float32) * want.abs().nan_to_num(0.0, 0.0, 0.0), "log_prob")
    pl = plogp(logp)
    dead = logp.max(1).values == float("-inf")
    ent = torch.where(dead, torch.zeros(rows, device=z.device, dtype=torch.float64), -pl.sum(1))
    ent = torch.where(bad, torch.full_like(ent, float("nan")), ent)
    # H = log s - e / s: both terms' errors, e of as many roundings and of terms up to the largest |y - r| that counts
    e_ent = 4 * rel[:, 0] * (1 + pl.abs().sum(1).nan_to_num(0.0) + 42.0 * 2.0 ** -20)
    assert_within(out.entropy, ent, e_ent + half(torch.float32) * ent.abs().nan_to_num(0.0), "entropy")
    # the same values with what the backward needs kept
    leaf = z.detach().requires_grad_()
    kept = cg.log_probs(leaf, target, top=top)
    assert all(torch.equal(p.nan_to_num(7.0), q.nan_to_num(7.0)) for p, q in zip(kept, out) if p is not None)
    if g_lp is None and g_ent is None:
        return
    outs = [(o, c) for o, c in ((kept.log_prob, g_lp), (kept.entropy, g_ent)) if o is not None and c is not None]
    (dz,) = torch.autograd.grad([o for o, _ in outs], leaf, [c for _, c in outs])
    assert dz.dtype == z.dtype
    p = logp.exp()
    a = torch.zeros(rows, 1, device=z.device, dtype=torch.float64)
    if g_lp is not None and target is not None:
        a = torch.where((target >= 0) & ~dead, g_lp.double(), torch.zeros_like(ent))[:, None]
    b = torch.zeros_like(a) if g_ent is None else torch.where(dead, torch.zeros_like(ent), g_ent.double())[:, None]
    want = -a * p - b * (pl + p * ent[:, None])
    if target is not None:
        want = want.scatter_add(1, target.clamp(0, classes - 1)[:, None], a)
        want = torch.where((target >= classes)[:, None] & (a != 0), torch.full_like(want, float("nan")), want)
    if bad.any():       # a row with a NaN or +inf has no gradient that means anything
        want, dz = want[~bad], dz[~bad]
        a, b, p, pl, ent, rel, e_ent = (t[~bad] for t in (a, b, p, pl, ent, rel, e_ent))
        target = None if target is None else target[~bad]
    tol = (rel * 4 + 8 * U) * (a.abs() * p + b.abs() * (pl.abs() + p * ent[:, None])) + b.abs() * p * (e_ent[:, None] + 2 * rel + 2.0 ** -21 * (1 + ent[:, None]))
    if target is not None and target.numel():
        tol = tol.scatter_add(1, target.clamp(0, classes - 1)[:, None], 4 * U * a.abs())
    t = z.dtype
    assert_within(dz, want, tol + half(t) * (want.abs() + tol) + torch.finfo(t).smallest_normal * torch.finfo(t).eps + 2.0 ** -126 * (a.abs() + 100 * b.abs()), "dlogits")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, classes, top", [(1, 1, 1), (3, 2, 2), (4, 10, 10), (64, 55, 5), (9, 130, 128), (17, 1000, 20), (3, 1024, 128), (5, 1025, 20), (2, 2047, 3),
                                                (300, 5000, 7), (2, 9001, 128), (1, 40003, 1), (1, 131072, 20), (3, 131075, 128), (160, 16385, 0), (150, 70001, 128), (150, 40000, 50)])
def test_log_probs(rows, classes, top, dtype):
    g = gen(rows + classes + top)
    z = (3 * randn(g, rows, classes)).to(dtype)
    target = torch.randint(0, classes, (rows,), generator=g, device=cuda())
    if rows > 2:
        target[1] = -1
    check_log_probs(z, target, top, randn(g, rows), 0.3 * randn(g, rows))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes, top", [(30, 12), (900, 50), (3000, 50), (20011, 128), (140000, 100)])
def test_log_probs_hard_rows(classes, top, dtype):
    """Equal scores, rising scores, coarse scores, rows masked by -inf or by the type's lowest value, with few classes or none
    left, zeros of both signs, large scores."""
    g = gen(classes)
    lowest, ninf = torch.finfo(dtype).min, float("-inf")
    z = (2 * randn(g, 14, classes)).to(dtype)
    z[0] = 0.75
    z[1] = torch.linspace(-8, 8, classes, device=cuda()).to(dtype)
    z[2] = z[1].flip(0)
    z[3] = (z[3] * 2).round() / 2
    z[4] = ninf
    z[5, 3:] = ninf
    z[6, :-2] = ninf
    z[7] = lowest
    z[8, classes // 2:] = lowest
    z[9, ::2] = ninf
    z[10] = torch.where(randn(g, classes) > 0, 0.0, -0.0).to(dtype)
    z[11] *= 1000
    z[12, : classes - top // 2] = ninf
    z[13] = -torch.arange(classes, device=cuda()).to(dtype) % 64
    target = torch.randint(0, classes, (14,), generator=g, device=cuda())
    target[4], target[5], target[13] = 1, classes - 1, -1
    check_log_probs(z, target, top, randn(g, 14), 0.3 * randn(g, 14))
    for row in range(14):      # few rows: several blocks share one
        check_log_probs(z[row:row + 1], target[row:row + 1], top, randn(g, 1), None)


@pytest.mark.parametrize("classes", [40, 5000, 140000])
def test_log_probs_nan_infinity_and_bad_targets(classes):
    g = gen(classes)
    z = randn(g, 6, classes)
    z[1, 7], z[2, classes - 1], z[3, 11] = float("nan"), float("nan"), float("inf")
    z[4] = float("-inf")
    z[4, 20] = float("nan")
    z[5, 0], z[5, 1] = float("nan"), float("nan")
    target = torch.tensor([classes, 3, 4, 11, 5, -100], device=cuda())
    check_log_probs(z, target, 9, randn(g, 6), None)
    for row in range(6):
        check_log_probs(z[row:row + 1], target[row:row + 1], 9)


def test_log_probs_layouts():
    import cgnet_b200 as cg
    g = gen(17)
    for dtype, classes in itertools.product(TYPES, (37, 3001)):
        wide = randn(g, 9, classes + 20).to(dtype)
        check_log_probs(wide[:, 3:3 + classes], torch.arange(9, device=cuda()), 5, randn(g, 9), randn(g, 9))
        check_log_probs(wide[:, ::2], None, 5, None, randn(g, 9))
        check_log_probs(wide[:1].expand(4, -1), torch.arange(4, device=cuda()), 3, randn(g, 4), None)
    z = randn(g, 2, 3, 50)
    t = torch.randint(0, 50, (2, 3), generator=g, device=cuda(), dtype=torch.int32)
    out, flat = cg.log_probs(z, t, top=4), cg.log_probs(z.view(6, 50), t.view(6), top=4)
    assert out.log_prob.shape == (2, 3) and out.top_ids.shape == (2, 3, 4) and out.entropy.shape == (2, 3)
    assert all(torch.equal(p.reshape(q.shape), q) for p, q in zip(out, flat))
    one = cg.log_probs(z[0, 0], t[0, 0], top=4)
    assert one.log_prob.shape == () and torch.equal(one.top_ids, out.top_ids[0, 0]) and torch.equal(one.log_prob, out.log_prob[0, 0])
    none = cg.log_probs(torch.empty(0, 50, device=cuda(), requires_grad=True), torch.empty(0, dtype=torch.long, device=cuda()), top=4)
    assert none.log_prob.shape == (0,) and none.top_ids.shape == (0, 4)
    assert cg.log_probs(z).log_prob is None


# ---------------------------------------------------------------------------------------------------------------------
# distillation
# ---------------------------------------------------------------------------------------------------------------------
def check_distill(z, ids, scores, temp, g_loss):
    import cgnet_b200 as cg
    rows, classes = z.shape
    logp, rel = softmax_bounds(z, temp)
    there = ids >= 0
    t = torch.where(there, scores.double() / temp, torch.full_like(scores, float("-inf"), dtype=torch.float64))
    some = (t > float("-inf")).any(1)
    logq = torch.where(some[:, None], torch.log_softmax(torch.where(some[:, None], t, torch.zeros_like(t)), 1), torch.full_like(t, float("-inf")))
    q = logq.exp()
    lp = logp.gather(1, ids.clamp(0, classes - 1))
    terms = torch.where(q > 0, q * (logq - lp), torch.zeros_like(q))
    over = (ids >= classes).any(1) & some
    want = temp * temp * torch.where(over, torch.full_like(terms.sum(1), float("nan")), terms.sum(1))
    leaf = z.detach().requires_grad_()
    loss = cg.distillation_loss(leaf, ids, scores, temperature=temp)
    with torch.no_grad():
        assert torch.equal(cg.distillation_loss(z, ids, scores, temperature=temp).nan_to_num(7.0), loss.nan_to_num(7.0))
    # the terms are taken in 64 bits from the row's float32 statistics: log s is off by rel, the scale by one rounding
    assert_within(loss.detach(), want, temp * temp * (rel[:, 0] + 8 * U) + half(torch.float32) * want.abs().nan_to_num(0.0, 0.0, 0.0), "loss")
    (dz,) = torch.autograd.grad(loss, leaf, g_loss)
    dead = (logp.max(1).values == float("-inf")) | ~some
    p = logp.exp()
    gt = (g_loss.double() * temp)[:, None]
    dq = torch.zeros_like(p).scatter_add(1, ids.clamp(0, classes - 1), q * (there & (ids < classes)))
    grad = torch.where(dead[:, None], torch.zeros_like(p), gt * (p - dq))
    tol = gt.abs() * (p * (4 * rel + 8 * U) + dq * 8 * U)
    ok = ~over & ~torch.isnan(logp).any(1)
    t_ = z.dtype
    assert_within(dz[ok], grad[ok], (tol + half(t_) * (grad.abs() + tol) + torch.finfo(t_).smallest_normal * torch.finfo(t_).eps + 2.0 ** -126 * gt.abs())[ok], "dlogits")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, classes, k", [(1, 1, 1), (3, 2, 1), (100, 10, 10), (7, 55, 8), (5, 1000, 100), (3, 1030, 1), (4, 5001, 1024), (300, 3001, 16), (1, 131073, 64),
                                              (2, 20000, 300)])
def test_distillation(rows, classes, k, dtype):
    g = gen(rows + classes + k)
    z = (2 * randn(g, rows, classes)).to(dtype)
    noisy = z.float() + randn(g, rows, classes)
    k_here = min(k, classes)
    scores, ids = torch.topk(noisy, k_here, dim=1)
    if k > 3:
        ids = ids.clone()
        ids[0, 1:] = -1
        ids[rows - 1, 2] = ids[rows - 1, 0]          # a class named twice
        scores[rows - 1, 1] = float("-inf")
    for temp in (1.0, 2.5):
        check_distill(z, ids, scores.to(dtype if k % 2 else torch.float32), temp, randn(g, rows))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [20, 3000, 70000])
def test_distillation_hard_rows(classes, dtype):
    """No entries, all entries of weight 0, all the same class, masked students, a class beyond the last, padded rows."""
    g = gen(classes)
    z = (2 * randn(g, 9, classes)).to(dtype)
    ids = torch.randint(0, classes, (9, 12), generator=g, device=cuda())
    scores = randn(g, 9, 12)
    ids[0] = -1
    scores[1] = float("-inf")
    ids[2] = 7
    z[3] = float("-inf")
    z[4, ids[4, 0]] = float("-inf")
    ids[5, 3] = classes
    z[6, 9:] = torch.finfo(dtype).min
    ids[6] = torch.arange(12, device=cuda()) % 8
    ids[7, 1:] = -100
    scores[8] *= 1000
    check_distill(z, ids, scores, 1.0, randn(g, 9))
    check_distill(z, ids, scores.to(dtype), 3.0, randn(g, 9))
    for row in (0, 3, 5, 6):
        check_distill(z[row:row + 1], ids[row:row + 1], scores[row:row + 1], 2.0, randn(g, 1))


def test_distillation_layouts():
    import cgnet_b200 as cg
    g = gen(23)
    for classes in (30, 4001):
        wide = randn(g, 8, classes + 9).bfloat16()
        ids = torch.randint(0, classes, (6, 8), generator=g, device=cuda()).t()
        check_distill(wide[:, 5:5 + classes], ids, randn(g, 8, 12)[:, ::2], 2.0, randn(g, 1).expand(8))
    z = randn(g, 2, 3, 40)
    ids, scores = torch.randint(0, 40, (2, 3, 5), generator=g, device=cuda()), randn(g, 2, 3, 5)
    loss = cg.distillation_loss(z, ids.int(), scores)
    assert loss.shape == (2, 3) and torch.equal(loss.view(6), cg.distillation_loss(z.view(6, 40), ids.view(6, 5), scores.view(6, 5)))
    assert cg.distillation_loss(z[:0], ids[:0], scores[:0]).shape == (0, 3)


# ---------------------------------------------------------------------------------------------------------------------
# together, and as a program uses them
# ---------------------------------------------------------------------------------------------------------------------
def test_gradients_against_differences():
    """Directional derivatives of the chain norm -> hidden layer -> scores -> losses against central differences of a 64-bit copy."""
    import cgnet_b200 as cg
    g = gen(29)
    x, w, b = randn(g, 20, 24), 1 + 0.1 * randn(g, 24), 0.1 * randn(g, 24)
    wg, wu, ws = randn(g, 36, 24) / 5, randn(g, 36, 24) / 5, randn(g, 11, 36) / 6
    target = torch.randint(0, 11, (20,), generator=g, device=cuda())
    ids, scores = torch.randint(0, 11, (20, 4), generator=g, device=cuda()), randn(g, 20, 4)

    def total64(ts):
        x_, w_, b_, wg_, wu_, ws_ = ts
        y = torch.nn.functional.layer_norm(x_, (24,), w_, b_, 1e-5)
        z = (torch.nn.functional.silu(y @ wg_.t()) * (y @ wu_.t())) @ ws_.t()
        lp = torch.log_softmax(z, 1)
        lq = torch.log_softmax(scores.double() / 2, 1)
        kl = 4 * (lq.exp() * (lq - torch.log_softmax(z / 2, 1).gather(1, ids))).sum(1)
        return (-lp.gather(1, target[:, None])[:, 0] + 0.1 * (lp.exp() * lp).sum(1) + 0.5 * kl).sum()

    leaves = [t.clone().requires_grad_() for t in (x, w, b, wg, wu, ws)]
    z = cg.gated_feed_forward(cg.layer_norm(leaves[0], leaves[1], leaves[2]), leaves[3], leaves[4]) @ leaves[5].t()
    out = cg.log_probs(z, target)
    total = (-out.log_prob - 0.1 * out.entropy + 0.5 * cg.distillation_loss(z, ids, scores, temperature=2.0)).sum()
    grads = torch.autograd.grad(total, leaves)
    base = [t.double() for t in (x, w, b, wg, wu, ws)]
    for i, grad in enumerate(grads):
        d = torch.randn(base[i].shape, generator=gen(31 + i), device=cuda(), dtype=torch.float64)
        h = 1e-5
        up = total64([t + h * d if j == i else t for j, t in enumerate(base)])
        down = total64([t - h * d if j == i else t for j, t in enumerate(base)])
        want = float((up - down) / (2 * h))
        got = float((grad.double() * d).sum())
        # differences: h^2 of third derivatives (below 1e-6 of the size here); float32 chain: 1e-5 of the gradient's norm
        assert abs(got - want) <= 2e-5 * float(grad.double().norm() * d.norm()) + 1e-6, (i, got, want)


def test_network_with_a_head_trains_and_is_taught():
    import cgnet_b200 as cg
    torch.manual_seed(0)
    taus = [[1] * 4, [3] * 4, [3] * 4]
    student = cg.SphericalCNN(3, taus, head=(32, 10))
    teacher = cg.SphericalCNN(3, [[1] * 4, [6] * 4, [6] * 4], head=(48, 10)).eval()
    assert student.output_length == 14 and {"head.norm.weight", "head.ff.w_gate", "head.scores.bias"} <= set(student.state_dict())
    assert not any(k.startswith("head") for k in cg.SphericalCNN(3, taus).state_dict())
    x = torch.randn(20, 16, 2, device=cuda())
    y = torch.randint(0, 10, (20,), device=cuda())
    with torch.no_grad():
        best = teacher.log_probs(x, top=4)
    loss = -student.log_probs(x, y).log_prob.mean() + student.distillation_loss(x, best.top_ids, best.top_log_probs, 2.0).mean()
    loss.backward()
    for name, p in student.named_parameters():
        if p.requires_grad:
            assert p.grad is not None and torch.isfinite(p.grad).all() and float(p.grad.abs().sum()) > 0, name
    student.eval()
    with torch.no_grad():
        logits, e = student(x), student.embed(x)
        head = student.head
        e64 = torch.nn.functional.layer_norm(e.double(), (14,), head.norm.weight.double(), head.norm.bias.double(), 1e-5)
        h64 = torch.nn.functional.silu(e64 @ head.ff.w_gate.double().t()) * (e64 @ head.ff.w_up.double().t())
        want = h64 @ head.scores.weight.double().t() + head.scores.bias.double()
        # three float32 steps of at most 48 terms, values of size one
        assert float((logits.double() - want).abs().max()) <= 1e-5
        ranked = student.log_probs(x, top=10)
        assert torch.equal(ranked.top_ids, torch.sort(logits, dim=1, descending=True, stable=True).indices)
    fast = cg.SphericalCNN_fast(3, [2] * 4, 2, num_channels_input=2, head=(16, 5))
    c = torch.randn(6, 2, 16, 2, device=cuda())
    assert fast(c).shape == (6, 5) and fast.embed(c).shape == (6, fast.output_length) and fast.log_probs(c, top=2).top_ids.shape == (6, 2)


def test_lazily_negated_views():
    """The imaginary part of a conjugate is a view with torch's negative bit: its memory holds the opposite sign."""
    import cgnet_b200 as cg
    g = gen(47)

    def negated(*shape):
        t = torch.complex(randn(g, *shape), randn(g, *shape)).conj().imag
        assert t.is_neg()
        return t, t.resolve_neg().contiguous()

    (x, x_), (w, w_), (b, b_), (v, v_), (s, s_) = negated(6, 40), negated(40), negated(40), negated(24, 40), negated(6, 5)
    ids = torch.randint(0, 40, (6, 5), generator=g, device=cuda())
    assert torch.equal(cg.layer_norm(x, w, b), cg.layer_norm(x_, w_, b_))
    assert torch.equal(cg.gated_feed_forward(x, v, v), cg.gated_feed_forward(x_, v_, v_))
    assert all(torch.equal(p, q) for p, q in zip(cg.log_probs(x, ids[:, 0], top=3), cg.log_probs(x_, ids[:, 0], top=3)))
    assert torch.equal(cg.distillation_loss(x, ids, s), cg.distillation_loss(x_, ids, s_))


def test_second_derivatives_are_refused():
    import cgnet_b200 as cg
    g = gen(41)
    x, w = randn(g, 4, 8).requires_grad_(), randn(g, 6, 8).requires_grad_()
    ids = torch.zeros(4, 2, dtype=torch.long, device=cuda())
    for out in (cg.layer_norm(x), cg.gated_feed_forward(x, w, w), cg.log_probs(x).entropy, cg.distillation_loss(x, ids, randn(g, 4, 2))):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(out.sum(), x, create_graph=True)


def chain(x, w, b, wg, wu, ws, target, ids, scores):
    import cgnet_b200 as cg
    z = cg.gated_feed_forward(cg.layer_norm(x, w, b), wg, wu) @ ws.t()
    out = cg.log_probs(z, target, top=3)
    loss = (-out.log_prob - 0.1 * out.entropy + cg.distillation_loss(z, ids, scores, temperature=2.0)).mean()
    return loss, out


def chain_inputs(seed, rows=96, dim=64, hidden=160, classes=1500):
    g = gen(seed)
    ts = [randn(g, rows, dim), 1 + 0.1 * randn(g, dim), 0.1 * randn(g, dim), randn(g, hidden, dim) / 8, randn(g, hidden, dim) / 8, randn(g, classes, hidden) / 12]
    return ts + [torch.randint(0, classes, (rows,), generator=g, device=cuda()), torch.randint(0, classes, (rows, 9), generator=g, device=cuda()), randn(g, rows, 9)]


def test_captured_steps_replay_and_do_not_disturb_each_other():
    """Two captured training steps (forward and backward) of the chain, replayed in turn with new inputs, give an eager step's bits."""
    graphs = []
    for seed in (1, 2):
        ts = chain_inputs(seed)
        static = [t.clone().requires_grad_(i < 6) for i, t in enumerate(ts)]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            torch.autograd.grad(chain(*static)[0], static[:6])
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            loss, out = chain(*static)
            grads = torch.autograd.grad(loss, static[:6])
        graphs.append((graph, static, loss, out, grads))
    for seed in (11, 12, 13):
        for graph, static, loss, out, grads in graphs:
            ts = chain_inputs(seed)
            with torch.no_grad():
                for s, t in zip(static, ts):
                    s.copy_(t)
            graph.replay()
        for graph, static, loss, out, grads in graphs:
            ts = [t.requires_grad_(i < 6) for i, t in enumerate(chain_inputs(seed))]
            want_loss, want_out = chain(*ts)
            want = torch.autograd.grad(want_loss, ts[:6])
            assert torch.equal(loss, want_loss) and torch.equal(out.top_ids, want_out.top_ids)
            assert all(torch.equal(p, q) for p, q in zip(grads, want))


def test_threads_that_made_no_cuda_call_before():
    """The first CUDA call of a thread is the operator's (memory comes from torch's cache)."""
    import threading

    import cgnet_b200 as cg
    g = gen(43)
    x, wg, wu, dh = (t.bfloat16() for t in (randn(g, 256, 256), randn(g, 512, 256) / 16, randn(g, 512, 256) / 16, randn(g, 256, 512)))
    leaves = [t.requires_grad_() for t in (x, wg, wu)]
    want = torch.autograd.grad(cg.gated_feed_forward(*leaves), leaves, dh)
    with torch.no_grad():
        h = cg.gated_feed_forward(x, wg, wu)
    torch.cuda.synchronize()
    got = []

    def work():
        try:
            with torch.no_grad():
                got.append(cg.gated_feed_forward(x, wg, wu))
        except RuntimeError as e:
            got.append(e)

    for _ in range(2):
        thread = threading.Thread(target=work)
        thread.start()
        thread.join()
    torch.cuda.synchronize()
    assert all(isinstance(p, torch.Tensor) and torch.equal(p, h) for p in got), got
    assert all(torch.isfinite(p).all() for p in want)


def test_side_streams_and_two_calls_at_once():
    ts = [t.requires_grad_(i < 6) for i, t in enumerate(chain_inputs(3, rows=700, dim=256, hidden=512))]
    loss, _ = chain(*ts)
    want = torch.autograd.grad(loss, ts[:6])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got_loss, _ = chain(*ts)
                results.append((got_loss, torch.autograd.grad(got_loss, ts[:6])))
    torch.cuda.synchronize()
    for got_loss, grads in results:
        assert torch.equal(got_loss, loss) and all(torch.equal(p, q) for p, q in zip(grads, want))


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs a second GPU")
def test_another_device_than_the_current_one():
    ts = [t.to("cuda:1").requires_grad_(i < 6) for i, t in enumerate(chain_inputs(4))]
    loss, _ = chain(*ts)
    got = torch.autograd.grad(loss, ts[:6])
    ref = [t.detach().to("cuda:0").requires_grad_(i < 6) for i, t in enumerate(ts)]
    want = torch.autograd.grad(chain(*ref)[0], ref[:6])
    assert all(torch.equal(p.cpu(), q.cpu()) for p, q in zip(got, want))


def test_offsets_beyond_32_bits():
    """Rows whose values lie more than 2^31 values into a buffer."""
    stride, dim = 1_200_000_000, 1500
    big = torch.empty(2 * stride + dim, dtype=torch.bfloat16, device=cuda())
    z = big.as_strided((3, dim), (stride, 1))
    g = gen(37)
    z.copy_(randn(g, 3, dim))
    check_norm(z.detach(), None, None, 1e-5, randn(g, 3, dim).bfloat16())
    check_log_probs(z, torch.arange(3, device=cuda()), 5, randn(g, 3), randn(g, 3))
    ids, scores = torch.arange(12, device=cuda()).view(3, 4), randn(g, 3, 4)
    check_distill(z, ids, scores, 1.0, randn(g, 3))
    w = (randn(g, 64, dim) / 40).bfloat16()
    check_ff(z.detach(), w, w.clone(), "silu", randn(g, 3, 64).bfloat16())
