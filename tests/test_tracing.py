"""The post-training operators in calls that something else records or transforms: torch.jit's
tracer, torch.compile, fake tensors, torch.func.  Such a call must reach the registered ops - a
launch of the C++ binding leaves no trace."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from llm_training_b200 import _lib, ops


class Wrapped(torch.Tensor):
    """A tensor that something intercepts."""


def test_what_runs_where_it_is_called():
    x, t = torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64)
    assert _lib.plain(x, t) and _lib.plain(torch.nn.Parameter(x), None, t)
    assert not _lib.plain(x.as_subclass(Wrapped)) and not _lib.plain(x, t.as_subclass(Wrapped))
    seen = []

    def f(x):
        seen.append((torch.jit.is_tracing(), _lib.plain(x)))
        return x + 1

    torch.jit.trace(f, x)
    assert (True, False) in seen and (True, True) not in seen
    with FakeTensorMode():
        assert not _lib.eager()
    torch.func.grad(lambda x: (seen.append(_lib.plain(x)), x.sum())[1])(x)
    assert seen[-1] is False and _lib.eager()


def test_clipping_of_fake_gradients():
    with FakeTensorMode():
        g = [torch.empty(3, 5, device="cuda"), torch.empty(7, device="cuda", dtype=torch.bfloat16)]
        assert ops.grad_norm(g).shape == () and ops.grad_norm(g).dtype == torch.float32
        out, norm = ops.clip_grads(g, 1.0)
        assert [o.shape for o in out] == [v.shape for v in g] and norm.shape == ()
        assert [o.dtype for o in out] == [v.dtype for v in g]
        p = torch.nn.Parameter(torch.empty(3, 5, device="cuda"))
        p.grad = g[0]
        assert ops.clip_grad_norm_([p], 1.0).device.type == "cuda"


# ---- GPU: the operators as functions of one tensor ---------------------------------------


def cases():
    g = torch.Generator().manual_seed(0)
    t = torch.randint(-1, 33, (4, 6), generator=g).cuda()
    ref = (-10 * torch.rand(4, generator=g)).cuda()
    old = (-3.5 * torch.rand(4, 6, generator=g)).cuda()
    adv = torch.randn(4, generator=g).cuda()
    w, h = torch.rand(33, generator=g).cuda(), torch.randn(4, 6, 33, generator=g).cuda()
    p = torch.nn.Parameter(torch.zeros(4, 6, 33, device="cuda"))
    p.grad = torch.zeros_like(p)

    def clip(x):
        out, norm = ops.clip_grads([x.detach() * 2, x.detach()[0].bfloat16()], 0.5)
        return out[0].sum() + out[1].float().sum() + norm

    def clip_into(x):
        a, b = x.detach() * 2, torch.empty(4, 6, 33, device="cuda", dtype=torch.bfloat16)
        _, norm = ops.clip_grads([a, a[1:]], 0.5, out=[b, torch.empty_like(a[1:])])
        ops.clip_grads([a], 0.25, out=[a])  # in place
        return a.sum() + b.float().sum() + norm

    def in_place(x):
        with torch.no_grad():
            p.grad.copy_(x.detach() * 2)
        return ops.clip_grad_norm_([p], 0.5) + p.grad.sum()

    return {
        "token_log_probs": lambda x: ops.token_log_probs(x, t).sum(),
        "preference_loss": lambda x: ops.preference_loss(x, t, ref)[0],
        "policy_loss": lambda x: ops.policy_loss(x, t, adv, old, old, kl_coef=0.1)[0],
        "policy_loss_and_grad": lambda x: (h * ops.policy_loss_and_grad(x, t, adv, old)[1]).sum(),
        "residual_norm": lambda x: sum(v.square().sum() for v in ops.residual_norm(
            x, h, w, post_weight=w, gate=w, kind="rms")),
        "grad_norm": lambda x: ops.grad_norm([x.detach(), x.detach()[1:, ::2]]),
        "clip_grads": clip,
        "clip_grads, out": clip_into,
        "clip_grad_norm_": in_place,
    }


DIFFERENTIABLE = ["token_log_probs", "preference_loss", "policy_loss", "residual_norm"]
KINDS = [*DIFFERENTIABLE, "policy_loss_and_grad", "grad_norm", "clip_grads", "clip_grads, out",
         "clip_grad_norm_"]


def inputs():
    g = torch.Generator().manual_seed(1)
    return [torch.randn(4, 6, 33, generator=g).cuda().requires_grad_(True) for _ in range(2)]


def value_and_grad(f, x, kind):
    v = f(x)
    return (v.detach(), *(torch.autograd.grad(v, x) if kind in DIFFERENTIABLE else ()))


def same(got, want):
    assert len(got) == len(want)
    for a, b in zip(got, want):
        # the same kernels; what stands around them may add up in another order
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_jit_trace_replays_on_new_inputs(kind):
    f, (x, y) = cases()[kind], inputs()
    traced = torch.jit.trace(f, x)
    assert any("sqrtblock::" in n.kind() for n in traced.inlined_graph.nodes())
    for v in (y, x):
        same(value_and_grad(traced, v, kind), value_and_grad(f, v, kind))


@pytest.mark.gpu
@pytest.mark.parametrize("backend", ["aot_eager", "inductor"])
@pytest.mark.parametrize("kind", KINDS)
def test_compiles_without_a_break(kind, backend):
    f, (x, y) = cases()[kind], inputs()
    torch._dynamo.reset()
    compiled = torch.compile(f, backend=backend, fullgraph=True)
    for v in (x, y, x):
        same(value_and_grad(compiled, v, kind), value_and_grad(f, v, kind))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", DIFFERENTIABLE)
def test_transforms_are_refused(kind):
    """Reverse and forward mode by torch.func, forward mode by dual tensors: an error, not a
    derivative of zero."""
    f, (x, y) = cases()[kind], inputs()
    with pytest.raises(RuntimeError):
        torch.func.grad(f)(x.detach())
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(f, (x.detach(),), (y.detach(),))
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda v: torch.func.vmap(f)(v[None]), (x.detach(),), (y.detach(),))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x.detach(), y.detach())
        with pytest.raises((RuntimeError, NotImplementedError)):
            f(dual)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", DIFFERENTIABLE)
def test_vmap_calls_once_for_each(kind):
    f, (x, y) = cases()[kind], inputs()
    got = torch.func.vmap(f)(torch.stack([x.detach(), y.detach()]))
    same(got, [f(v).detach() for v in (x, y)])


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("how", ["jit.trace", "compile"])
def test_a_model_with_a_norm_and_a_gate_behind_its_blocks(how):
    from llm_training_b200.config import ModelConfig
    from llm_training_b200.model.gpt import GPT

    torch.manual_seed(0)
    m = GPT(ModelConfig(block_size=64, vocab_size=97, n_layer=2, n_head=2, n_embd=128, bias=False,
                        attention="sqrt_block", post_norm=True, layer_scale=0.5)).cuda()
    a, b = torch.randint(0, 97, (2, 2, 64), device="cuda")
    if how == "compile":
        torch._dynamo.reset()
        traced = torch.compile(m, backend="aot_eager", fullgraph=True)
    else:
        traced = torch.jit.trace(m, a)
        kinds = [n.kind() for n in traced.inlined_graph.nodes()]
        assert kinds.count("sqrtblock::residual_norm_fwd") == 4
    for tokens in (b, a):
        # fp32 throughout, the same kernels
        torch.testing.assert_close(traced(tokens), m(tokens), rtol=1e-5, atol=1e-5)
