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


@DTYPES
@VOCABULARIES
@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_ratio_without_old_logps_is_one(reduction, V, dtype):
    """Also for a token without probability: its term is -A, its gradient that of the
    log-probability."""
    x, t = batch(V, dtype)
    adv = torch.linspace(-1, 2, 4, device="cuda")
    leaf = x.clone().requires_grad_(True)
    loss, logps, stats = ops.policy_loss(leaf, t, adv, reduction=reduction)
    (g,) = torch.autograd.grad(loss, leaf)
    one, grad, _, _ = ops.policy_loss_and_grad(x, t, adv, reduction=reduction)
    want = -adv.double().mean()  # as many tokens in every sequence
    for v in (loss, one, stats[0]):
        # weights, advantages and the result rounded to fp32, of terms up to 2
        assert abs(float(v) - float(want)) <= 2 * 4 * 2.0**-24
    assert float(logps[0, 1]) == -math.inf
    for v in (g, grad):
        p = torch.softmax(x[0, 1].double(), -1)
        p[t[0, 1]] -= 1.0
        exact = float(adv[0]) / 12 * p
        # V / 32 + 100 roundings in a row's sum at most, as for the other losses
        room = exact.abs() * (torch.finfo(dtype).eps / 2 * 1.01 + (V / 32 + 100) * 2.0**-24)
        assert ((v[0, 1].double() - exact).abs() <= room + 2.0**-126).all()
        assert v.isfinite().all()


def test_nan_log_probabilities_stay_nan_without_old_logps():
    x, t = batch(9, torch.float32)
    x[1, 0] = math.nan
    t[2, 1] = 9  # past the vocabulary
    loss, grad, logps, _ = ops.policy_loss_and_grad(x, t, torch.ones(4, device="cuda"))
    assert loss.isnan() and grad[1, 0].isnan().all() and grad[2, 1].isnan().all()
    assert logps[1, 0].isnan() and logps[2, 1].isnan() and int(logps.isnan().sum()) == 2
