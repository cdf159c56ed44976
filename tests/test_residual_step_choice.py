"""When a GPT block's residual step runs as the library's kernel; other calls are torch's."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from llm_training_b200.model.gpt import LayerNorm, residual_step_fused


def test_what_runs_as_the_kernel():
    with FakeTensorMode():
        x = torch.empty(2, 5, 64, device="cuda")
        assert residual_step_fused(x, x) and residual_step_fused(x, x.bfloat16())
        assert not residual_step_fused(x, x.double()) and not residual_step_fused(x.half(), x)
        assert not residual_step_fused(x, x[:1])  # added to every sample
        assert not residual_step_fused(x, x.cpu())
        wide = torch.empty(2, 4097, device="cuda")
        assert not residual_step_fused(wide, wide)


@pytest.mark.gpu
def test_an_output_that_is_shared_by_the_samples():
    torch.manual_seed(0)
    norm, post = LayerNorm(64).cuda(), LayerNorm(64).cuda()
    gate = torch.randn(64, device="cuda")
    x, h = torch.randn(2, 5, 64, device="cuda"), torch.randn(1, 5, 64, device="cuda")
    got = norm.add_forward(x, h, post, gate)
    want = norm.add_forward(x, h.expand(2, 5, 64).contiguous(), post, gate)
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-5)
