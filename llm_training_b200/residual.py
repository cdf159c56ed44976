"""The residual step between two norms (csrc/sqb_residual_norm.cu)."""

from __future__ import annotations

import math
from typing import Optional

import torch

from torch.autograd.function import once_differentiable

from . import _lib

__all__ = ["residual_norm"]

_DTYPES = {torch.float32: _lib.SQB_F32, torch.bfloat16: _lib.SQB_BF16}
MAX_WIDTH = 4096
MAX_GATES = 65530


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _fwd_raw(x: torch.Tensor, h: torch.Tensor, w: torch.Tensor, b: Optional[torch.Tensor],
             wp: Optional[torch.Tensor], bp: Optional[torch.Tensor],
             gate: Optional[torch.Tensor], scale: float, eps: float, rms: bool,
             out_dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Contiguous x, h (..., C) and gate (... , C), each of its rows shared by as many rows
    of x in turn -> (x', y, row statistics)."""
    C = x.shape[-1]
    N = x.numel() // C
    xo = torch.empty_like(x)
    y = torch.empty_like(x, dtype=out_dtype)
    stats = torch.empty(4 * N, dtype=torch.float32, device=x.device)
    if N:
        with _lib.on_device(x.device):
            _lib.check("sqb_residual_norm_fwd", _lib.lib().sqb_residual_norm_fwd(
                x.data_ptr(), _DTYPES[x.dtype], h.data_ptr(), _DTYPES[h.dtype], w.data_ptr(),
                _ptr(b), _ptr(wp), _ptr(bp), _ptr(gate),
                gate.numel() // C if gate is not None else 0, scale, eps, rms, xo.data_ptr(),
                y.data_ptr(), _DTYPES[out_dtype], stats.data_ptr(), N, C,
                _lib.stream(x.device)))
    return xo, y, stats


_fwd = torch.library.custom_op("sqrtblock::residual_norm_fwd", _fwd_raw, mutates_args=())


@_fwd.register_fake
def _(x, h, w, b, wp, bp, gate, scale, eps, rms, out_dtype):
    return (torch.empty_like(x), torch.empty_like(x, dtype=out_dtype),
            x.new_empty(4 * (x.numel() // x.shape[-1]), dtype=torch.float32))


def _bwd_raw(dy: torch.Tensor, dxo: Optional[torch.Tensor], x: torch.Tensor, h: torch.Tensor,
             w: torch.Tensor, b: Optional[torch.Tensor], wp: Optional[torch.Tensor],
             bp: Optional[torch.Tensor], gate: Optional[torch.Tensor], scale: float, eps: float,
             rms: bool, stats: torch.Tensor
             ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dh, the gradients of w, b, wp, bp and gate - those that are there - end to end)."""
    C = x.shape[-1]
    N = x.numel() // C
    sizes = [p.numel() if p is not None else 0 for p in (w, b, wp, bp, gate)]
    dx, dh = torch.empty_like(x), torch.empty_like(h)
    dp = torch.empty(sum(sizes), dtype=torch.float32, device=x.device)
    if N == 0:
        return dx, dh, dp.zero_()
    at, ptrs = dp.data_ptr(), []
    for n in sizes:
        ptrs.append(at if n else None)
        at += 4 * n
    gates = sizes[4] // C
    lib = _lib.lib()
    nbytes = lib.sqb_residual_norm_workspace_bytes(N, C, gates)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    with _lib.on_device(x.device):
        _lib.check("sqb_residual_norm_bwd", lib.sqb_residual_norm_bwd(
            dy.data_ptr(), _DTYPES[dy.dtype], _ptr(dxo), x.data_ptr(), _DTYPES[x.dtype],
            h.data_ptr(), _DTYPES[h.dtype], w.data_ptr(), _ptr(b), _ptr(wp), _ptr(bp),
            _ptr(gate), gates, scale, eps, rms, stats.data_ptr(), dx.data_ptr(), dh.data_ptr(),
            *ptrs, ws.data_ptr(), nbytes, N, C,
            _lib.stream(x.device)))
    return dx, dh, dp


_bwd = torch.library.custom_op("sqrtblock::residual_norm_bwd", _bwd_raw, mutates_args=())


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
    dx, dh, dp = (_bwd_raw if _lib.plain(x) else _bwd)(
        dy.contiguous(), dxo, x, h, w, b, wp, bp, gate, *ctx.cfg, stats)
    C = x.shape[-1]
    rows = dp.view(-1, C)
    if gate is not None and gate.numel() != C:  # its rows are the last
        k = rows.shape[0] - gate.numel() // C
        parts = iter((*rows[:k].unbind(0), rows[k:].view(gate.shape)))
    else:
        parts = iter(rows.unbind(0))
    given = [next(parts) if p is not None else None for p in (w, b, wp, bp, gate)]
    if gate is not None and given[4].shape != gate.shape:
        given[4] = given[4].view(gate.shape)
    return (dx, dh, *given, None, None, None, None)


_fwd.register_autograd(_grad, setup_context=_setup)


class _Residual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *args):
        out = _fwd_raw(*args)
        _setup(ctx, args, out)
        return out

    backward = staticmethod(once_differentiable(_grad))


def _run(*args):
    """An eager call skips the dispatcher, a traced one is the custom op."""
    if not _lib.plain(args[0]):
        return _fwd(*args)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args[:7]):
        return _Residual.apply(*args)
    return _fwd_raw(*args)


def _param(name, p, shape, device):
    if p is None:
        return None
    if tuple(p.shape) != shape or p.device != device or p.dtype not in _DTYPES:
        raise ValueError(f"residual_norm: {name} must be float32 or bfloat16 {shape} on x's "
                         f"device, got {p.dtype} {tuple(p.shape)}")
    return p.float().contiguous()


def _gates(gate, x):
    if gate is None:
        return None
    C, B = x.shape[-1], x.shape[0]
    if gate.device != x.device or gate.dtype not in _DTYPES:
        raise ValueError("residual_norm: gate must be float32 or bfloat16 on x's device, got "
                         f"{gate.dtype}")
    shape = tuple(gate.shape)
    if shape != (C,) and (x.dim() < 2 or not 0 < B <= MAX_GATES
                          or shape not in ((B, *(1,) * (x.dim() - 2), C), (B, C))):
        raise ValueError(f"residual_norm: gate must be (C,) or one row for each of the first "
                         f"dimension's entries (at most {MAX_GATES}), got {shape} for x "
                         f"{tuple(x.shape)}")
    return gate.float().contiguous()


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
    if not math.isfinite(scale) or not (math.isfinite(eps) and eps >= 0):
        raise ValueError(f"residual_norm: scale must be finite and eps finite and not negative, "
                         f"got {scale}, {eps}")
    if x.numel() // C > 2**31 - 1:
        raise ValueError("residual_norm: at most 2**31 - 1 rows")
    w, b = (_param(n, p, (C,), x.device) for n, p in (("weight", weight), ("bias", bias)))
    wp, bp = (_param(n, p, (C,), x.device) for n, p in (("post_weight", post_weight),
                                                        ("post_bias", post_bias)))
    xo, y, _ = _run(x.contiguous(), h.contiguous(), w, b, wp, bp, _gates(gate, x), scale, eps,
                    kind == "rms", out_dtype)
    return xo, y
