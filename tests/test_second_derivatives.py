"""The post-training operators are differentiable once.  A second derivative is refused on
every path that reaches it, also where the rest of the expression has one of its own: a
gradient penalty must not lose its second-order part silently."""

import pytest
import torch

from llm_training_b200 import ops

pytestmark = pytest.mark.gpu


def losses():
    t = torch.randint(0, 9, (4, 3), generator=torch.Generator().manual_seed(0)).cuda()
    one = torch.ones(4, device="cuda")
    return {
        "token_log_probs": lambda x: ops.token_log_probs(x, t).square().sum(),
        "preference_loss": lambda x: ops.preference_loss(x, t)[0],
        "policy_loss": lambda x: ops.policy_loss(x, t, one)[0],
    }


@pytest.mark.parametrize("kind", ["token_log_probs", "preference_loss", "policy_loss"])
def test_gradient_penalty_on_logits(kind):
    loss_of = losses()[kind]
    w = torch.randn(4, 3, 9, device="cuda", requires_grad=True)
    x = 2 * w  # the logits are no leaf
    loss = loss_of(x)
    for wanted in (w, x):
        (g,) = torch.autograd.grad(loss, wanted, create_graph=True)
        total = loss + g.square().sum()
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(total, w, retain_graph=True)
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(g.sum(), wanted, allow_unused=True, retain_graph=True)
        with pytest.raises(RuntimeError, match="second derivative"):
            total.backward(retain_graph=True)
    # and through the upstream gradient
    up = torch.tensor(1.5, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(loss, x, up, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(g.sum(), up, allow_unused=True)


def test_gradient_penalty_through_the_residual_step():
    C = 64
    v = {k: torch.randn(2, 5, C, device="cuda") for k in ("x", "h")}
    v.update({k: torch.randn(C, device="cuda") for k in ("weight", "bias", "gate")})
    v["post_weight"] = torch.randn(C, device="cuda")
    v = {k: t.requires_grad_(True) for k, t in v.items()}
    kw = {k: t for k, t in v.items() if k not in ("x", "h", "weight")}
    xo, y = ops.residual_norm(v["x"], v["h"], v["weight"], **kw)
    loss = (xo * xo).sum() + y.square().sum()
    for first in v:
        (g,) = torch.autograd.grad(loss, v[first], create_graph=True)
        for k, other in v.items():
            with pytest.raises(RuntimeError, match="second derivative"):
                torch.autograd.grad(g.square().sum() + other.sum(), other, retain_graph=True,
                                    allow_unused=True)


def test_a_gradient_kept_for_later_can_be_used():
    """create_graph alone refuses nothing."""
    x = torch.randn(4, 3, 9, device="cuda", requires_grad=True)
    loss_of = losses()["preference_loss"]
    (g,) = torch.autograd.grad(loss_of(x), x, create_graph=True)
    (plain,) = torch.autograd.grad(loss_of(x), x)
    assert torch.equal(g, plain) and g.requires_grad
    k = torch.tensor(2.0, device="cuda", requires_grad=True)
    (d,) = torch.autograd.grad((g.detach() * k).sum(), k)
    assert torch.allclose(d, plain.sum())
