"""The post-training operators as they are used together: a GPT whose blocks have a norm and
a gate behind them, trained on answers by the preference and the policy loss, its gradients
clipped."""

import pytest
import torch

from llm_training_b200 import ops
from llm_training_b200.config import ModelConfig
from llm_training_b200.model.gpt import GPT
from llm_training_b200.train import Trainer, configure_optimizers, synthetic_batch

CPU_ATTN = "tests.cpu_attention:CausalAttentionCPU"


def config(**kw):
    base = dict(block_size=64, vocab_size=97, n_layer=2, n_head=2, n_embd=32, bias=False,
                attention=CPU_ATTN)
    base.update(kw)
    return ModelConfig(**base)


def test_default_model_has_no_new_parameters():
    torch.manual_seed(0)
    keys = set(GPT(config()).state_dict())
    assert not any("lp1" in k or "lp2" in k or "gate" in k for k in keys)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("post,scale", [(True, None), (False, 0.1), (True, 0.1)])
def test_post_norm_and_layer_scale_on_cpu(post, scale, bias):
    torch.manual_seed(0)
    m = GPT(config(post_norm=post, layer_scale=scale, bias=bias))
    b = m.transformer.attn_blocks[0]
    assert (b.lp1 is not None) == post and (b.gate1 is not None) == (scale is not None)
    decay, rest = configure_optimizers(m, 0.1, 1e-3, device_type="cpu").param_groups
    if scale is not None:
        assert torch.all(b.gate1 == scale)
        assert any(p is b.gate1 for p in rest["params"])
    x, _ = synthetic_batch(torch.Generator().manual_seed(0), 2, 16, 97, torch.device("cpu"))
    # the stream unrolled over the blocks is the blocks one after another
    t = m.transformer
    h = t.wte(x) + t.wpe(torch.arange(16))
    for block in t.attn_blocks:
        h = block(h)
    torch.testing.assert_close(m(x), m.lm_head(t.ln_(h)))
    loss = m(x).square().mean()
    loss.backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in m.parameters())


def gpu_model(**kw):
    torch.manual_seed(0)
    m = GPT(config(attention="sqrt_block", block_size=256, n_embd=256, n_head=4,
                   vocab_size=1001, **kw)).cuda()
    with torch.no_grad():
        for p in m.parameters():
            if p.dim() == 1:
                p.add_(0.1 * torch.randn_like(p))
    return m


def same_direction(got, want):
    """bf16 operands of the GEMMs differ by an ulp here and there where a kernel's sum is taken
    in another order: gradients are compared by direction and length, as the trainer's other
    fused operators are."""
    for n in want:
        if n.endswith("Wk.bias"):
            # a constant added to every key moves all of a query's scores alike: the exact
            # gradient is 0, and rounding has no direction
            continue
        a, b = got[n].flatten().float(), want[n].flatten().float()
        cos = float(torch.dot(a, b) / (a.norm() * b.norm() + 1e-30))
        assert cos > 0.999, (n, cos)
        assert float((a.norm() - b.norm()).abs() / (b.norm() + 1e-30)) < 1e-2, n


@pytest.mark.gpu
@pytest.mark.parametrize("bias", [False, True])
def test_fused_residual_step_is_the_models_own(bias, monkeypatch):
    import llm_training_b200.model.gpt as gpt

    m = gpu_model(post_norm=True, layer_scale=0.5, bias=bias)
    x, y = synthetic_batch(torch.Generator().manual_seed(1), 2, 256, 1001,
                           torch.device("cuda", 0))

    def run():
        m.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss = ops.cross_entropy(m(x, pad_vocab=True), y)
        loss.backward()
        return loss.detach(), {n: p.grad.clone() for n, p in m.named_parameters()}

    calls = []
    real = gpt.residual_norm
    monkeypatch.setattr(gpt, "residual_norm", lambda *a, **k: calls.append(1) or real(*a, **k))
    loss, grads = run()
    assert len(calls) == 4  # two residual adds in each of two blocks
    monkeypatch.setattr(gpt, "residual_step_fused", lambda x, h: False)
    want_loss, want = run()
    torch.testing.assert_close(loss, want_loss, rtol=2e-3, atol=2e-3)
    same_direction(grads, want)


def plain_logps(logits, targets):
    lp = torch.log_softmax(logits.float(), -1)
    got = lp.gather(-1, targets.clamp_min(0)[..., None])[..., 0]
    return torch.where(targets >= 0, got, 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["preference", "policy", "policy, one pass"])
def test_a_step_on_answers(kind):
    """Loss, every parameter's gradient, the norm and the clipped gradients against the same
    step on torch operations."""
    m = gpu_model(post_norm=True, layer_scale=0.5)
    g = torch.Generator().manual_seed(2)
    tok = torch.randint(0, 1001, (4, 129), generator=g).cuda()
    x, y = tok[:, :-1].contiguous(), tok[:, 1:].clone()
    y[:, :40] = -100  # the prompt
    y[1, 100:] = -100  # padding
    adv = torch.tensor([1.0, -0.5, 0.3, -1.2], device="cuda")
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        ref = ops.token_log_probs(m(x, pad_vocab=True), y)
    old = ref + 0.1 * torch.randn(ref.shape, generator=g).cuda()
    count = (y >= 0).sum()

    def loss_of(logits, fused):
        if kind == "preference":
            if fused:
                return ops.preference_loss(logits, y, ref.sum(1), beta=0.1)[0]
            s = plain_logps(logits, y).sum(1) - ref.sum(1)
            return -torch.nn.functional.logsigmoid(0.1 * (s[:2] - s[2:])).mean()
        if fused:
            return ops.policy_loss(logits, y, adv, old, ref, kl_coef=0.1)[0]
        lp = plain_logps(logits, y)
        r = (lp - old).exp()
        each = -torch.minimum(r * adv[:, None], r.clamp(0.8, 1.2) * adv[:, None])
        each = each + 0.1 * ((ref - lp).exp() - (ref - lp) - 1)
        return torch.where(y >= 0, each, 0.0).sum() / count

    def step(fused):
        m.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            logits = m(x, pad_vocab=True)
        if fused and kind == "policy, one pass":
            loss, grad, logps, stats = ops.policy_loss_and_grad(logits, y, adv, old, ref,
                                                                kl_coef=0.1)
            logits.backward(grad)
            torch.testing.assert_close(logps, ref, rtol=0, atol=1e-5)
            assert float(stats[2]) > 0
        else:
            loss = loss_of(logits, fused)
            loss.backward()
        params = list(m.parameters())
        before = {n: p.grad.clone() for n, p in m.named_parameters()}
        bound = 0.5 * float(torch.stack([p.grad.norm() for p in params]).norm())
        norm = (ops.clip_grad_norm_(params, bound) if fused
                else torch.nn.utils.clip_grad_norm_(params, bound))
        after = float(torch.stack([p.grad.norm() for p in params]).norm())
        assert after == pytest.approx(bound, rel=1e-4)
        return loss.detach(), norm, before

    loss, norm, grads = step(True)
    want_loss, want_norm, want = step(False)
    torch.testing.assert_close(loss, want_loss, rtol=1e-4, atol=1e-5)
    torch.testing.assert_close(norm, want_norm, rtol=1e-2, atol=0)
    same_direction(grads, want)


@pytest.mark.gpu
def test_trainer_clips_with_the_library():
    tr = Trainer(config(attention="sqrt_block", block_size=256, n_embd=128, n_head=2,
                        vocab_size=512, post_norm=True, layer_scale=0.1),
                 torch.device("cuda", 0), lr=0.0, seed=0)
    gen = torch.Generator().manual_seed(0)
    x, y = synthetic_batch(gen, 4, 256, 512, torch.device("cuda", 0))
    loss, norm = tr.step(x, y)
    grads = [p.grad for p in tr.model.parameters()]
    assert loss.isfinite() and float(norm) > 1.0
    assert float(ops.grad_norm(grads)) == pytest.approx(1.0, rel=1e-5)
