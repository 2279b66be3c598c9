"""Classes beyond the last and NaN scores: which gradients they spoil, and which they leave alone.  Scores far below the best."""
import pytest
import torch

from test_gpu_head import TYPES, check_distill, gen, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [20, 700, 3000, 70000])
def test_distillation_gradient_of_a_row_that_is_nan(classes, dtype):
    """The row's loss and its whole gradient are NaN, every other row is what it is without the bad entry."""
    import cgnet_b200 as cg
    g = gen(classes)
    z = (2 * randn(g, 6, classes)).to(dtype)
    ids = torch.randint(0, classes, (6, 5), generator=g, device=z.device)
    scores = randn(g, 6, 5)
    g_loss = randn(g, 6)
    bad_ids, bad_scores = ids.clone(), scores.clone()
    bad_ids[1, 3] = classes                     # one of five
    bad_ids[2] = torch.tensor([1 << 40, -1, -1, -1, -1], device=z.device)        # the only one
    bad_scores[4, 2] = float("nan")
    leaf = z.clone().requires_grad_()
    want_loss = cg.distillation_loss(leaf, ids, scores, 2.0)
    (want,) = torch.autograd.grad(want_loss, leaf, g_loss)
    loss = cg.distillation_loss(leaf, bad_ids, bad_scores, 2.0)
    (dz,) = torch.autograd.grad(loss, leaf, g_loss)
    good = [0, 3, 5]
    assert torch.isnan(loss[[1, 2, 4]]).all() and torch.isnan(dz[[1, 2, 4]]).all()
    assert torch.equal(loss[good], want_loss[good]) and torch.equal(dz[good], want[good])
    for row in (1, 2, 4):                       # a row by itself: several blocks share it
        leaf = z[row:row + 1].clone().requires_grad_()
        (dz,) = torch.autograd.grad(cg.distillation_loss(leaf, bad_ids[row:row + 1], bad_scores[row:row + 1].to(dtype), 2.0), leaf, g_loss[:1])
        assert torch.isnan(dz).all()
    check_distill(z[good], ids[good], scores[good], 2.0, g_loss[good])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [20, 3000])
def test_entropy_gradient_of_a_row_whose_target_is_beyond_the_last_class(classes, dtype):
    """The log probability is NaN and so is a gradient through it; the entropy does not depend on the target."""
    import cgnet_b200 as cg
    g = gen(classes)
    z = (2 * randn(g, 4, classes)).to(dtype).requires_grad_()
    target = torch.tensor([1, classes, 1 << 40, -1], device=z.device)
    g_ent = randn(g, 4)
    out = cg.log_probs(z, target)
    (want,) = torch.autograd.grad(cg.log_probs(z).entropy, z, g_ent)
    (dz,) = torch.autograd.grad(out.entropy, z, g_ent, retain_graph=True)
    assert torch.isfinite(want).all() and torch.equal(dz, want)
    (dz,) = torch.autograd.grad(out.log_prob, z, g_ent)
    assert torch.isnan(dz[1:3]).all() and torch.isfinite(dz[[0, 3]]).all()


@pytest.mark.parametrize("entries", [1, 40, 300])
@pytest.mark.parametrize("classes", [20, 3000])
def test_a_class_beyond_the_last_counts_whatever_its_score(classes, entries):
    """Scores of -inf have weight 0 and a row of nothing else loss 0, but not where a class does not exist."""
    import cgnet_b200 as cg
    g = gen(classes + entries)
    z = randn(g, 3, classes).requires_grad_()
    ids = torch.randint(0, classes, (3, entries), generator=g, device=z.device)
    ids[1, entries - 1] = classes
    loss = cg.distillation_loss(z, ids, torch.full((3, entries), float("-inf"), device=z.device))
    (dz,) = torch.autograd.grad(loss.sum(), z)
    assert torch.isnan(loss[1]) and torch.isnan(dz[1]).all()
    assert not loss[[0, 2]].any() and not dz[[0, 2]].any()


@pytest.mark.parametrize("classes, entries", [(50, 12), (700, 100), (3000, 500), (90000, 300)])
def test_distillation_of_scores_far_below_the_best(classes, entries):
    """Weights down to e^-80: each is off by a few roundings of its own, not by its exponent's."""
    g = gen(classes)
    z = 2 * randn(g, 40, classes)
    ids = torch.stack([torch.randperm(classes, generator=g, device=z.device)[:entries] for _ in range(40)])
    scores = -40 * torch.rand(40, entries, generator=g, device=z.device)
    for temp in (0.5, 1.0, 3.0):
        check_distill(z, ids, scores, temp, 1 + randn(g, 40).abs())
