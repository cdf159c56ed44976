"""The trainer's clipping: the library's where it takes the gradients, torch's for others (a
plugin's fp16 or fp64 parameters, sparse gradients), as it did for all of them."""

import pytest
import torch
import torch.nn as nn

from llm_training_b200 import ops
from llm_training_b200.config import ModelConfig
from llm_training_b200.train import Trainer, synthetic_batch
from tests.cpu_attention import CausalAttentionCPU


class HalfGain(CausalAttentionCPU):
    """Attention with a gain for each channel that is kept in half precision."""

    dtype = torch.float16

    def __init__(self, config):
        super().__init__(config)
        self.gain = nn.Parameter(torch.ones(config.n_embd, dtype=self.dtype))

    def forward(self, X):
        return super().forward(X) * self.gain.float()


class DoubleGain(HalfGain):
    dtype = torch.float64


def config(attention):
    return ModelConfig(block_size=64, vocab_size=512, n_layer=2, n_head=2, n_embd=128, bias=False,
                       attention=f"tests.test_trainer_clipping:{attention}")


def test_what_the_library_takes():
    p, q, r = (nn.Parameter(torch.zeros(3)) for _ in range(3))
    assert not ops.clip_grad_norm_supported([p, q])  # nothing to look at
    p.grad = torch.zeros(3)
    assert not ops.clip_grad_norm_supported([p])  # on the CPU
    assert not ops.clip_grad_norm_supported(iter([p, q]))
    r.grad = torch.zeros(3).to_sparse()
    assert not ops.clip_grad_norm_supported([r])


def test_trainer_step_on_the_cpu():
    tr = Trainer(config("HalfGain"), torch.device("cpu"), lr=0.0)
    x, y = synthetic_batch(torch.Generator().manual_seed(0), 2, 32, 512, torch.device("cpu"))
    loss, norm = tr.step(x, y)
    assert loss.isfinite() and norm.isfinite()


@pytest.mark.gpu
def test_what_the_library_takes_on_the_gpu():
    def param(dtype, device="cuda"):
        p = nn.Parameter(torch.zeros(3, dtype=dtype, device=device))
        p.grad = torch.ones_like(p)
        return p

    f32, bf16 = param(torch.float32), param(torch.bfloat16)
    assert ops.clip_grad_norm_supported([f32, bf16]) and ops.clip_grad_norm_supported(f32)
    for dtype in (torch.float16, torch.float64):
        assert not ops.clip_grad_norm_supported([f32, param(dtype)])
    assert not ops.clip_grad_norm_supported([f32, param(torch.float32, "cpu")])
    none = nn.Parameter(torch.zeros(3, dtype=torch.float64, device="cuda"))
    assert ops.clip_grad_norm_supported([f32, none])  # it has no gradient


@pytest.mark.gpu
@pytest.mark.parametrize("attention", ["HalfGain", "DoubleGain"])
def test_trainer_with_other_dtypes(attention):
    tr = Trainer(config(attention), torch.device("cuda", 0), lr=0.0, seed=0)
    x, y = synthetic_batch(torch.Generator().manual_seed(0), 2, 64, 512, torch.device("cuda", 0))
    loss, norm = tr.step(x, y)
    grads = [p.grad for p in tr.model.parameters()]
    assert {g.dtype for g in grads} == {torch.float32, globals()[attention].dtype}
    after = float(torch.stack([g.double().norm() for g in grads]).norm())
    assert loss.isfinite() and float(norm) > 1.0
    # the half gradients are rounded to 2^-11, the factor to fp32
    assert after == pytest.approx(1.0, rel=2.0**-11 + 1e-5)
