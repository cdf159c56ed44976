"""Infinite log-probabilities and coefficients of zero: a term that is switched off adds
nothing to the loss and nothing to the gradient, however large it is."""

import math

import pytest
import torch

from llm_training_b200 import ops

pytestmark = pytest.mark.gpu


def batch(V, dtype, sequences=4):
    """(logits, targets) whose token (0, 1) has a target without probability."""
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(sequences, 3, V, generator=g) * 2).to(dtype)
    t = torch.randint(0, V, (sequences, 3), generator=g)
    x[0, 1, t[0, 1]] = -math.inf
    return x.cuda(), t.cuda()


DTYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
VOCABULARIES = pytest.mark.parametrize("V", [9, 5003])


@DTYPES
@VOCABULARIES
@pytest.mark.parametrize("far", [math.nan, math.inf, 1000.0, -math.inf])
def test_kl_for_logging_only(far, V, dtype):
    """kl_coef = 0 with ref_logps: the loss and the gradient are those without them."""
    x, t = batch(V, dtype)
    adv = torch.linspace(-1, 2, 4, device="cuda")
    old = torch.full(t.shape, -2.0, device="cuda")
    ref = old.clone()
    ref[1, 2] = far  # and a -inf log-probability against a finite one at (0, 1)
    got = []
    for r in (ref, None):
        leaf = x.clone().requires_grad_(True)
        loss, logps, stats = ops.policy_loss(leaf, t, adv, old, r)
        (g,) = torch.autograd.grad(loss, leaf)
        one, grad, _, _ = ops.policy_loss_and_grad(x, t, adv, old, r)
        assert loss.isfinite() and g.isfinite().all() and grad.isfinite().all()
        got.append([loss.detach(), logps, stats[0], stats[2], g, one, grad])
    assert all(torch.equal(a, b) for a, b in zip(*got))


@DTYPES
@VOCABULARIES
@pytest.mark.parametrize("smooth", [0.0, 1.0])
def test_preference_term_of_coefficient_zero(smooth, V, dtype):
    """A pair's z is +inf or -inf where one of its answers has no probability.  The term that
    counts is then 0 or +inf, the other one is not there."""
    for rejected in (False, True):
        x, t = batch(V, dtype, 2)
        if rejected:
            x, t = x.flip(0), t.flip(0)
        x = x.clone().requires_grad_(True)
        loss, chosen, lost = ops.preference_loss(x, t, label_smoothing=smooth)
        (g,) = torch.autograd.grad(loss, x)
        assert float((lost if rejected else chosen)[0]) == -math.inf
        assert float(loss) == (0.0 if rejected == (smooth == 0.0) else math.inf)
        assert g.isfinite().all()
        # the loss's slope: 0 where it is flat, -beta or beta where it is straight
        assert bool(g.any()) == (float(loss) == math.inf)
