"""The residual step between two norms (csrc/sqb_residual_norm.cu)."""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib

__all__ = ["residual_norm"]

_DTYPES = (torch.float32, torch.bfloat16)
MAX_WIDTH = 4096
MAX_GATES = 65530


# ---- the operator: contiguous x, h (..., C), gate (..., C) with each of its rows shared by
# as many rows of x in turn.  An eager call goes to the C++ binding, which has the autograd
# node; these are the same launches registered as custom ops, for traced calls.


@torch.library.custom_op("sqrtblock::residual_norm_fwd", mutates_args=())
def _fwd(x: torch.Tensor, h: torch.Tensor, w: torch.Tensor, b: Optional[torch.Tensor],
         wp: Optional[torch.Tensor], bp: Optional[torch.Tensor], gate: Optional[torch.Tensor],
         scale: float, eps: float, rms: bool, out_dtype: torch.dtype
         ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(x', y, row statistics)"""
    return _lib.binding().residual_fwd(x, h, w, b, wp, bp, gate, scale, eps, rms,
                                       out_dtype == torch.bfloat16)


@_fwd.register_fake
def _(x, h, w, b, wp, bp, gate, scale, eps, rms, out_dtype):
    return (torch.empty_like(x), torch.empty_like(x, dtype=out_dtype),
            x.new_empty(4 * (x.numel() // x.shape[-1]), dtype=torch.float32))


@torch.library.custom_op("sqrtblock::residual_norm_bwd", mutates_args=())
def _bwd(dy: torch.Tensor, dxo: Optional[torch.Tensor], x: torch.Tensor, h: torch.Tensor,
         w: torch.Tensor, b: Optional[torch.Tensor], wp: Optional[torch.Tensor],
         bp: Optional[torch.Tensor], gate: Optional[torch.Tensor], scale: float, eps: float,
         rms: bool, stats: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dh, the gradients of w, b, wp, bp and gate - those that are there - end to end)."""
    return _lib.binding().residual_bwd(dy, dxo, x, h, w, b, wp, bp, gate, scale, eps, rms, stats)


@_bwd.register_fake
def _(dy, dxo, x, h, w, b, wp, bp, gate, scale, eps, rms, stats):
    n = sum(p.numel() for p in (w, b, wp, bp, gate) if p is not None)
    return torch.empty_like(x), torch.empty_like(h), x.new_empty(n, dtype=torch.float32)


def _setup(ctx, inputs, output):
    _, y, stats = output
    ctx.save_for_backward(*inputs[:7], stats)
    ctx.cfg = inputs[7:10]
    ctx.y_dtype = y.dtype
    ctx.mark_non_differentiable(stats)
    ctx.set_materialize_grads(False)


def _grad(ctx, dxo, dy, _dstats):
    x, h, w, b, wp, bp, gate, stats = ctx.saved_tensors
    if dxo is None and dy is None:
        return (None,) * 11
    if dy is None:
        dy = torch.zeros(x.shape, dtype=ctx.y_dtype, device=x.device)
    dxo = dxo.contiguous() if dxo is not None else None
    dx, dh, dp = _bwd(dy.contiguous(), dxo, x, h, w, b, wp, bp, gate, *ctx.cfg, stats)
    given, at = [], 0
    for p in (w, b, wp, bp, gate):
        given.append(dp[at:at + p.numel()].view(p.shape) if p is not None else None)
        at += p.numel() if p is not None else 0
    return (dx, dh, *given, None, None, None, None)


_fwd.register_autograd(_grad, setup_context=_setup)


def _fp32(p):
    if p.dtype != torch.float32:
        p = p.float()
    return p if p.is_contiguous() else p.contiguous()


def _param(name, p, C, device):
    if p is None:
        return None
    if p.shape != (C,) or p.device != device or p.dtype not in _DTYPES:
        raise ValueError(f"residual_norm: {name} must be float32 or bfloat16 ({C},) on x's "
                         f"device, got {p.dtype} {tuple(p.shape)}")
    return _fp32(p)


def _gates(gate, x, C, device):
    if gate is None:
        return None
    if gate.device != device or gate.dtype not in _DTYPES:
        raise ValueError("residual_norm: gate must be float32 or bfloat16 on x's device, got "
                         f"{gate.dtype}")
    shape, B = gate.shape, x.shape[0]
    if shape != (C,) and (x.dim() < 2 or not 0 < B <= MAX_GATES
                          or shape not in ((B, *(1,) * (x.dim() - 2), C), (B, C))):
        raise ValueError(f"residual_norm: gate must be (C,) or one row for each of the first "
                         f"dimension's entries (at most {MAX_GATES}), got {tuple(shape)} for x "
                         f"{tuple(x.shape)}")
    return _fp32(gate)


def residual_norm(x, h, weight, bias=None, *, post_weight=None, post_bias=None, gate=None,
                  scale=1.0, eps=1e-5, kind="layer", out_dtype=torch.float32):
    """The residual step after a block and the norm before the next -> (x', y).

        n  = Norm(h; post_weight, post_bias)     (h itself without a post_weight)
        x' = x + scale * gate * n                (no gate: ones)
        y  = Norm(x'; weight, bias)

    ``x`` (the residual stream) and ``h`` (a block's output) are CUDA (..., C), C <= 4096,
    each float32 or bfloat16; x' has x's dtype and y ``out_dtype``.  ``kind`` "layer" is
    LayerNorm, "rms" an RMS norm (no mean).  ``gate`` is (C,), or one row for each sample
    of x's first dimension: (B, C) or (B, 1, ..., C).  All math is fp32, each output
    rounded once (y is the norm of x' before x' is rounded to bfloat16); weights and gates
    may be bfloat16.  Differentiable, once, in every tensor (``sqrtblock::residual_norm_fwd/bwd``);
    parameter gradients are summed in a fixed order (bit-reproducible)."""
    if not x.is_cuda:
        raise RuntimeError("residual_norm: x must be a CUDA tensor (the op has no CPU "
                           "implementation)")
    if x.dtype not in _DTYPES or h.dtype not in _DTYPES or out_dtype not in _DTYPES:
        raise TypeError("residual_norm supports float32 and bfloat16, got "
                        f"{x.dtype}, {h.dtype}, {out_dtype}")
    if x.dim() == 0 or h.shape != x.shape or h.device != x.device:
        raise ValueError(f"residual_norm: x and h must have one shape (..., C) and device, got "
                         f"{tuple(x.shape)} and {tuple(h.shape)}")
    C = x.shape[-1]
    if not 0 < C <= MAX_WIDTH:
        raise ValueError(f"residual_norm: rows of 1 to {MAX_WIDTH} columns, got {C}")
    if kind not in ("layer", "rms"):
        raise ValueError(f"residual_norm: kind must be 'layer' or 'rms', got {kind!r}")
    if weight is None:
        raise ValueError("residual_norm: weight is needed")
    if post_bias is not None and post_weight is None:
        raise ValueError("residual_norm: a post_bias needs a post_weight")
    scale, eps = float(scale), float(eps)
    if not abs(scale) <= 1e30 or not 0 <= eps <= 1e30:  # float32 arguments of the kernels
        raise ValueError(f"residual_norm: scale must be finite and eps finite and not negative, "
                         f"got {scale}, {eps}")
    if x.numel() // C > 2**31 - 1:
        raise ValueError("residual_norm: at most 2**31 - 1 rows")
    device = x.device
    w, b = _param("weight", weight, C, device), _param("bias", bias, C, device)
    wp = _param("post_weight", post_weight, C, device)
    bp = _param("post_bias", post_bias, C, device)
    args = (x.contiguous(), h.contiguous(), w, b, wp, bp, _gates(gate, x, C, device), scale, eps,
            kind == "rms")
    if _lib.plain(*args[:7]):
        return _lib.binding().residual(*args, out_dtype == torch.bfloat16)
    return _fwd(*args, out_dtype)[:2]
