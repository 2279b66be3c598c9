"""The operators between the invariant embedding of a CG network and its answers, as work to be timed: layer norm,
gated feed-forward block, log probabilities of classes with entropy and ranked alternatives, distillation from a teacher's
top scores.  Each has a plain form in elementary torch operations and a call of this package's kernels (``own``)."""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the embedding of the five-layer network, 2 (1 + 5 * 5) invariants, at its batch of 100: a training step's norm
        dict(name="norm_head_train", op="norm", rows=100, dim=52, dtype="fp32", train=True),
        # a training step over many rows of a wide model
        dict(name="norm_wide_train", op="norm", rows=8192, dim=4096, dtype="bf16", train=True),
        # scoring ragged rows of an odd width (no row after the first is aligned for wide loads)
        dict(name="norm_odd_score", op="norm", rows=3001, dim=1023, dtype="fp16", train=False),
        # the classifier's hidden layer, 52 -> 256 at batch 100, in training
        dict(name="ff_head_train", op="ff", rows=100, dim=52, hidden=256, dtype="fp32", act="relu", train=True),
        # one row at a time: serving, bound by reading the weights
        dict(name="ff_single", op="ff", rows=1, dim=4096, hidden=8192, dtype="bf16", act="silu", train=False),
        # a training step over many rows of a wide model
        dict(name="ff_wide_train", op="ff", rows=8192, dim=2048, hidden=5120, dtype="bf16", act="silu", train=True),
        # a ragged batch in half precision, a hidden width that no tile divides
        dict(name="ff_ragged_train", op="ff", rows=1111, dim=1000, hidden=1365, dtype="fp16", act="gelu", train=True),
        # 55 classes at batch 64: the loss of a training step and the five best classes of each shape
        dict(name="logp_head_train", op="logp", rows=64, classes=55, top=5, dtype="fp32", train=True),
        # scoring many rows over a large set of classes, with the ranked list of each
        dict(name="logp_wide_score", op="logp", rows=2048, classes=65536, top=20, dtype="bf16", train=False),
        # one row over a large set of classes: serving
        dict(name="logp_single", op="logp", rows=1, classes=131072, top=20, dtype="bf16", train=False),
        # a small network taught by a large one on ten classes, all of the teacher's scores given
        dict(name="distill_head_train", op="distill", rows=100, classes=10, top=10, dtype="fp32", temp=2.0, train=True),
        # a training step over a large set of classes with the teacher's 64 best
        dict(name="distill_wide_train", op="distill", rows=4096, classes=50000, top=64, dtype="bf16", temp=2.0, train=True),
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "ff", "logp", "distill"])
    case = dict(op=op, dtype=rng.choice(["fp32", "bf16", "fp16"]), train=rng.random() < 0.6)
    if op == "norm":
        most = 8192 * 4096 // (2 if case["dtype"] == "fp32" else 1)
        case["dim"] = _spread(rng, 16, 16384)
        case["rows"] = _spread(rng, 1, min(16384, most // case["dim"]))
    elif op == "ff":
        # fp32 has three times the multiply-adds' cost or more: smaller products
        most = 8192 * 2048 * 5120 // (8 if case["dtype"] == "fp32" else 1)
        case["dim"] = _spread(rng, 16, 4096)
        case["hidden"] = _spread(rng, 16, 8192)
        case["rows"] = _spread(rng, 1, min(8192, max(1, most // (case["dim"] * case["hidden"]))))
        case["act"] = rng.choice(["silu", "gelu", "relu"])
    else:
        most = (2048 * 65536 if op == "logp" else 4096 * 50000) // (2 if case["dtype"] == "fp32" else 1)
        case["classes"] = _spread(rng, 10, 131072)
        case["rows"] = _spread(rng, 1, min(8192, most // case["classes"]))
        case["top"] = min(case["classes"], rng.choice([1, 5, 20, 50] if op == "logp" else [1, 8, 64, 100]))
        if op == "distill":
            case["temp"] = rng.choice([1.0, 2.0, 4.0])
    return case


def work(case):
    s, r = _SIZE[case["dtype"]], case["rows"]
    if case["op"] == "norm":
        d = case["dim"]
        if case["train"]:        # x, dy -> y, dx; weight and bias and their gradients
            return {"bytes": 4 * r * d * s + 4 * d * s, "flops": 20 * r * d}
        return {"bytes": 2 * r * d * s + 2 * d * s, "flops": 8 * r * d}
    if case["op"] == "ff":
        d, h = case["dim"], case["hidden"]
        if case["train"]:        # x, W, dh -> h, dx, dW
            return {"bytes": s * (2 * r * d + 4 * h * d + 2 * r * h), "flops": 12 * r * d * h}
        return {"bytes": s * (r * d + 2 * h * d + r * h), "flops": 4 * r * d * h}
    v, k = case["classes"], case["top"]
    if case["op"] == "logp":
        small = r * (8 + 4 + 4) + r * k * 12
        if case["train"]:        # logits -> results, gradient
            return {"bytes": 2 * r * v * s + small + 8 * r, "flops": 12 * r * v}
        return {"bytes": r * v * s + small, "flops": 6 * r * v}
    small = r * k * (8 + s) + 4 * r
    if case["train"]:
        return {"bytes": 2 * r * v * s + small + 4 * r, "flops": 9 * r * v}
    return {"bytes": r * v * s + small, "flops": 4 * r * v}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    t, train, r = _TYPES[case["dtype"]], case["train"], case["rows"]

    def normal(*shape, scale=1.0, shift=0.0, dtype=t):
        return (torch.randn(*shape, generator=gen, device=dev) * scale + shift).to(dtype)

    st = dict(case)
    if case["op"] == "norm":
        d = case["dim"]
        # rows of different size and offset, as activations have them
        size = torch.exp(0.5 * torch.randn(r, 1, generator=gen, device=dev))
        st["x"] = ((torch.randn(r, d, generator=gen, device=dev) + torch.randn(r, 1, generator=gen, device=dev)) * size).to(t)
        st["w"] = normal(d, scale=0.1, shift=1.0)
        st["b"] = normal(d, scale=0.1)
        st["eps"] = 1e-5
        st["leaves"] = ["x", "w", "b"]
        if train:
            st["dy"] = normal(r, d)
    elif case["op"] == "ff":
        d, h = case["dim"], case["hidden"]
        st["x"] = normal(r, d)
        st["wg"] = normal(h, d, scale=d ** -0.5)
        st["wu"] = normal(h, d, scale=d ** -0.5)
        st["leaves"] = ["x", "wg", "wu"]
        if train:
            st["dh"] = normal(r, h)
    else:
        v, k = case["classes"], case["top"]
        # scores with a few classes well above the rest; the last of a large padded set are masked out
        z = torch.randn(r, v, generator=gen, device=dev) * 2.0
        z[torch.rand(r, v, generator=gen, device=dev) < 4.0 / v] += 8.0
        st["leaves"] = ["z"]
        if case["op"] == "logp":
            if v >= 1024:
                z[:, v - v // 1000:] = float("-inf")
            st["z"] = z.to(t)
            st["target"] = torch.randint(0, v - v // 1000 if v >= 1024 else v, (r,), generator=gen, device=dev)
            if r >= 16:
                st["target"][r - r // 16:] = -1        # rows of padding carry no target
            if train:
                # advantages and an entropy bonus, with the loss scaled as half precision needs it
                st["g_lp"] = normal(r, dtype=torch.float32)
                st["g_ent"] = torch.full((r,), 0.01, device=dev)
        else:
            st["z"] = z.to(t)
            # the teacher agrees with the student roughly: its best classes among noisy scores, highest first
            noisy = z + torch.randn(r, v, generator=gen, device=dev)
            top, ids = torch.topk(noisy, k, dim=1)
            st["ids"] = ids
            st["scores"] = top.to(t)
            if r >= 16 and k > 1:
                st["ids"][::16, k // 2:] = -1           # rows with a shorter list
            if train:
                st["g"] = torch.rand(r, generator=gen, device=dev)
    if train:
        for name in st["leaves"]:
            st[name].requires_grad_()
    return st


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    import cgnet_b200 as cg
    op, train = st["op"], st["train"]
    if op == "norm":
        y = cg.layer_norm(st["x"], st["w"], st["b"], st["eps"])
        if not train:
            return y
        return (y.detach(), *torch.autograd.grad(y, (st["x"], st["w"], st["b"]), st["dy"]))
    if op == "ff":
        h = cg.gated_feed_forward(st["x"], st["wg"], st["wu"], activation=st["act"])
        if not train:
            return h
        return (h.detach(), *torch.autograd.grad(h, (st["x"], st["wg"], st["wu"]), st["dh"]))
    if op == "logp":
        out = cg.log_probs(st["z"], st["target"], top=st["top"])
        if not train:
            return tuple(out)
        grads = torch.autograd.grad((out.log_prob, out.entropy), (st["z"],), (st["g_lp"], st["g_ent"]))
        return (*(o.detach() for o in out), *grads)
    loss = cg.distillation_loss(st["z"], st["ids"], st["scores"], temperature=st["temp"])
    if not train:
        return loss
    return (loss.detach(), *torch.autograd.grad(loss, (st["z"],), (st["g"],)))


@torch.no_grad()
def _run_plain(st):
    return {"norm": _plain_norm, "ff": _plain_ff, "logp": _plain_logp, "distill": _plain_distill}[st["op"]](st)


def _plain_norm(st):
    t = st["x"].dtype
    x, w, b = st["x"].float(), st["w"].float(), st["b"].float()
    centred = x - x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + st["eps"])
    xh = centred * rstd
    y = (xh * w + b).to(t)
    if not st["train"]:
        return y
    dy = st["dy"].float()
    wdy = dy * w
    dx = rstd * (wdy - wdy.mean(1, keepdim=True) - xh * (wdy * xh).mean(1, keepdim=True))
    return y, dx.to(t), (dy * xh).sum(0).to(t), dy.sum(0).to(t)


def _act(name, g):
    """The activation and its derivative."""
    if name == "relu":
        on = (g > 0).to(g.dtype)
        return g * on, on
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    c = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return g * c, c + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_ff(st):
    t = st["x"].dtype
    x, wg, wu = st["x"].float(), st["wg"].float(), st["wu"].float()
    g, u = x @ wg.t(), x @ wu.t()
    a, da = _act(st["act"], g)
    h = (a * u).to(t)
    if not st["train"]:
        return h
    dh = st["dh"].float()
    dg, du = dh * u * da, dh * a
    return h, (dg @ wg + du @ wu).to(t), (dg.t() @ x).to(t), (du.t() @ x).to(t)


def _softmax_parts(z):
    """exp(z - max), its sum, and the log of the normaliser, along the rows."""
    m = z.max(1, keepdim=True).values
    e = torch.exp(z - m)
    s = e.sum(1, keepdim=True)
    return e, s, m + torch.log(s)


def _plain_logp(st):
    z, target, k = st["z"].float(), st["target"], st["top"]
    e, s, lse = _softmax_parts(z)
    p = e / s
    logp = z - lse
    ent_terms = torch.where(p > 0, p * logp, torch.zeros_like(p))
    ent = -ent_terms.sum(1)
    has = target >= 0
    at = target.clamp(min=0)[:, None]
    lp = torch.where(has, logp.gather(1, at)[:, 0], torch.zeros_like(ent))
    # the k highest, ties to the lowest index: one integer key that orders by value, then by index downwards
    bits = (z + 0.0).view(torch.int32)
    order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long()
    v = z.shape[1]
    key = order * (1 << 32) + (v - 1 - torch.arange(v, device=z.device))
    ids = torch.topk(key, k, dim=1).indices
    out = (lp, ent, logp.gather(1, ids), ids)
    if not st["train"]:
        return out
    g_lp = torch.where(has, st["g_lp"], torch.zeros_like(ent))[:, None]
    g_ent = st["g_ent"][:, None]
    dz = -g_lp * p - g_ent * (ent_terms + p * ent[:, None])
    dz.scatter_add_(1, at, g_lp)
    return (*out, dz.to(st["z"].dtype))


def _plain_distill(st):
    temp, ids = st["temp"], st["ids"]
    z = st["z"].float() / temp
    e, s, lse = _softmax_parts(z)
    given = ids >= 0
    at = ids.clamp(min=0)
    scores = st["scores"].float() / temp
    scores = torch.where(given, scores, torch.full_like(scores, float("-inf")))
    qe, qs, qlse = _softmax_parts(scores)
    q = qe / qs
    terms = torch.where(q > 0, q * ((scores - qlse) - (z.gather(1, at) - lse)), torch.zeros_like(q))
    loss = temp * temp * terms.sum(1)
    if not st["train"]:
        return loss
    g = (temp * st["g"])[:, None]
    dz = g * (e / s)
    dz.scatter_add_(1, at, -g * torch.where(given, q, torch.zeros_like(q)))
    return loss, dz.to(st["z"].dtype)


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits, gradients by differentiating them
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    with torch.enable_grad():
        leaves = [st[n].detach().double().requires_grad_(case["train"]) for n in st["leaves"]]
        if case["op"] == "norm":
            x, w, b = leaves
            var = x.var(1, unbiased=False, keepdim=True)
            outs, cot = ((x - x.mean(1, keepdim=True)) * torch.rsqrt(var + st["eps"]) * w + b,), ("dy",)
            rest = ()
        elif case["op"] == "ff":
            x, wg, wu = leaves
            g = torch.einsum("md,hd->mh", x, wg)
            a = {"relu": lambda v: v.clamp(min=0), "silu": lambda v: v * torch.sigmoid(v),
                 "gelu": lambda v: v * torch.special.ndtr(v)}[case["act"]](g)
            outs, cot, rest = (a * torch.einsum("md,hd->mh", x, wu),), ("dh",), ()
        elif case["op"] == "logp":
            z = leaves[0]
            logp = torch.log_softmax(z, dim=1)
            ent = -torch.special.xlogy(logp.exp(), logp.exp()).sum(1) if not case["train"] else \
                -(logp.exp() * logp.masked_fill(z == float("-inf"), 0.0)).sum(1)
            target = st["target"]
            lp = -torch.nn.functional.nll_loss(logp, target, ignore_index=-1, reduction="none")
            ids = torch.sort(z.detach(), dim=1, descending=True, stable=True).indices[:, :case["top"]]
            outs, cot = (lp, ent), ("g_lp", "g_ent")
            rest = (logp.detach().gather(1, ids), ids)
        else:
            z = leaves[0]
            ids, temp = st["ids"], case["temp"]
            logq = torch.log_softmax((st["scores"].double() / temp).masked_fill(ids < 0, float("-inf")), dim=1)
            picked = torch.log_softmax(z / temp, dim=1).gather(1, ids.clamp(min=0)).masked_fill(ids < 0, 0.0)
            kl = (logq.exp() * (logq.masked_fill(ids < 0, 0.0) - picked)).sum(1)
            outs, cot, rest = (temp * temp * kl,), ("g",), ()
        grads = ()
        if case["train"]:
            grads = torch.autograd.grad(outs, leaves, [st[c].double() for c in cot])
    result = (*(o.detach() for o in outs), *rest, *(g.detach() for g in grads))
    return result[0] if len(result) == 1 else result
