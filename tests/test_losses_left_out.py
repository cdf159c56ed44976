"""Rows of a packed batch outside every sequence, and rows without a target: whatever they
hold, whatever their target is and whatever reaches the loss from above, they add nothing
and their gradient is zero."""

import math

import pytest
import torch

from llm_training_b200 import ops

pytestmark = pytest.mark.gpu

FIRST, LAST = 3, 15  # rows [0, 3) and [15, 20) lie outside the sequences
CU = [FIRST, 7, 9, 9, LAST]


def batch(V, dtype):
    """(logits, targets, targets with the rows outside set to -1, cu_seqlens, outside)"""
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(LAST + 5, V, generator=g) * 3).to(dtype)
    t = torch.randint(0, V, (LAST + 5,), generator=g)
    t[[5, 12]] = -100  # left out inside a sequence, too
    x[5], x[12, V // 2] = math.nan, math.inf
    x[0], t[1], x[2, V // 2] = math.nan, V, math.inf
    x[LAST], t[LAST] = math.nan, V + 5
    x[LAST + 1], t[LAST + 2], t[LAST + 3] = -math.inf, 2**31 + 3, 2**62
    outside = torch.ones(LAST + 5, dtype=torch.bool)
    outside[FIRST:LAST] = False
    masked = torch.where(outside, -1, t)
    cu = torch.tensor(CU, device="cuda")
    return x.cuda(), t.cuda(), masked.cuda(), cu, (masked < 0).cuda()


LOSSES = {
    "preference": lambda x, t, cu: ops.preference_loss(x, t, label_smoothing=0.1, cu_seqlens=cu),
    "policy": lambda x, t, cu: ops.policy_loss(x, t, torch.linspace(-1, 2, 4, device="cuda"),
                                               cu_seqlens=cu),
    "policy, a sequence's mean": lambda x, t, cu: ops.policy_loss(
        x, t, torch.ones(t.shape, device="cuda"), reduction="sequence", cu_seqlens=cu),
}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [9, 1500, 5003])
@pytest.mark.parametrize("up", [1.0, math.inf, math.nan])
@pytest.mark.parametrize("kind", LOSSES)
def test_rows_outside_every_sequence(kind, up, V, dtype):
    x, t, masked, cu, left = batch(V, dtype)
    got = []
    for targets in (t, masked):
        leaf = x.clone().requires_grad_(True)
        loss, *others = LOSSES[kind](leaf, targets, cu)
        (g,) = torch.autograd.grad(loss, leaf, torch.tensor(up, device="cuda"))
        assert loss.isfinite() and torch.count_nonzero(g[left]) == 0
        assert g[~left].isfinite().all() == math.isfinite(up)
        got.append([loss.detach(), *others, g.nan_to_num(7.0, 8.0, 9.0)])
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [9, 1500, 5003])
def test_both_policy_forms_leave_the_same_rows_out(V, dtype):
    x, t, masked, cu, left = batch(V, dtype)
    adv = torch.linspace(-1, 2, 4, device="cuda")
    loss, grad, logps, stats = ops.policy_loss_and_grad(x, t, adv, cu_seqlens=cu)
    want = ops.policy_loss_and_grad(x, masked, adv, cu_seqlens=cu)
    assert loss.isfinite() and grad.isfinite().all()
    assert torch.count_nonzero(grad[left]) == 0 and torch.count_nonzero(logps[left]) == 0
    assert all(torch.equal(a, b) for a, b in zip((loss, grad, logps, stats), want))


@pytest.mark.parametrize("V", [9, 5003])
def test_a_counted_target_past_the_vocabulary_stays_nan(V):
    """Whatever its factor: an upstream gradient of 0 does not make it a number."""
    x = torch.randn(4, V, device="cuda", requires_grad=True)
    t = torch.tensor([1, V, 2**40 + 1, -1], device="cuda")
    lp = ops.token_log_probs(x, t)
    for up in (torch.ones(4, device="cuda"), torch.zeros(4, device="cuda")):
        (g,) = torch.autograd.grad(lp, x, up, retain_graph=True)
        assert g[1:3].isnan().all() and g[[0, 3]].isfinite().all()
        assert torch.count_nonzero(g[3]) == 0
    (g,) = torch.autograd.grad(lp, x, torch.full((4,), math.nan, device="cuda"))
    assert g[:3].isnan().all() and torch.count_nonzero(g[3]) == 0
