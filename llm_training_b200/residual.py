"""The residual step between two norms (csrc/sqb_residual_norm.cu)."""

from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib

__all__ = ["residual_norm"]

_DTYPES = {torch.float32: _lib.SQB_F32, torch.bfloat16: _lib.SQB_BF16}
MAX_WIDTH = 4096
MAX_GATES = 65531


def _ptr(t):
    return t.data_ptr() if t is not None else None


@torch.library.custom_op("sqrtblock::residual_norm_fwd", mutates_args=())
def _fwd(x: torch.Tensor, h: torch.Tensor, w: torch.Tensor, b: Optional[torch.Tensor],
         wp: Optional[torch.Tensor], bp: Optional[torch.Tensor], gate: Optional[torch.Tensor],
         scale: float, eps: float, rms: bool, out_dtype: torch.dtype
         ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Rows x, h (N, C), gate (G, C) or None -> (x' (N, C), y (N, C), row statistics)."""
    N, C = x.shape
    xo = torch.empty_like(x)
    y = torch.empty((N, C), dtype=out_dtype, device=x.device)
    stats = torch.empty((N, 4), dtype=torch.float32, device=x.device)
    if N:
        with _lib.on_device(x.device):
            _lib.check("sqb_residual_norm_fwd", _lib.lib().sqb_residual_norm_fwd(
                x.data_ptr(), _DTYPES[x.dtype], h.data_ptr(), _DTYPES[h.dtype], w.data_ptr(),
                _ptr(b), _ptr(wp), _ptr(bp), _ptr(gate), gate.shape[0] if gate is not None else 0,
                scale, eps, int(rms), xo.data_ptr(), y.data_ptr(), _DTYPES[out_dtype],
                stats.data_ptr(), N, C, torch.cuda.current_stream(x.device).cuda_stream))
    return xo, y, stats


@_fwd.register_fake
def _(x, h, w, b, wp, bp, gate, scale, eps, rms, out_dtype):
    N, C = x.shape
    return (x.new_empty((N, C)), x.new_empty((N, C), dtype=out_dtype),
            x.new_empty((N, 4), dtype=torch.float32))


@torch.library.custom_op("sqrtblock::residual_norm_bwd", mutates_args=())
def _bwd(dy: torch.Tensor, dxo: Optional[torch.Tensor], x: torch.Tensor, h: torch.Tensor,
         w: torch.Tensor, b: Optional[torch.Tensor], wp: Optional[torch.Tensor],
         bp: Optional[torch.Tensor], gate: Optional[torch.Tensor], scale: float, eps: float,
         rms: bool, stats: torch.Tensor
         ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor,
                    torch.Tensor, torch.Tensor]:
    """(dx, dh, dw, db, dwp, dbp, dgate), empty for a parameter that is not there."""
    N, C = x.shape
    gates = gate.shape[0] if gate is not None else 0
    dx, dh = torch.empty_like(x), torch.empty_like(h)

    def grad_of(p, *shape):
        return torch.empty(shape if p is not None else 0, dtype=torch.float32, device=x.device)

    dw, db, dwp, dbp = grad_of(w, C), grad_of(b, C), grad_of(wp, C), grad_of(bp, C)
    dgate = grad_of(gate, gates, C)
    if N == 0:
        for g in (dw, db, dwp, dbp, dgate):
            g.zero_()
        return dx, dh, dw, db, dwp, dbp, dgate
    lib = _lib.lib()
    nbytes = lib.sqb_residual_norm_workspace_bytes(N, C, gates)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    with _lib.on_device(x.device):
        _lib.check("sqb_residual_norm_bwd", lib.sqb_residual_norm_bwd(
            dy.data_ptr(), _DTYPES[dy.dtype], _ptr(dxo), x.data_ptr(), _DTYPES[x.dtype],
            h.data_ptr(), _DTYPES[h.dtype], w.data_ptr(), _ptr(b), _ptr(wp), _ptr(bp),
            _ptr(gate), gates, scale, eps, int(rms), stats.data_ptr(), dx.data_ptr(),
            dh.data_ptr(), dw.data_ptr(), _ptr(db), _ptr(dwp), _ptr(dbp), _ptr(dgate),
            ws.data_ptr(), nbytes, N, C, torch.cuda.current_stream(x.device).cuda_stream))
    return dx, dh, dw, db, dwp, dbp, dgate


@_bwd.register_fake
def _(dy, dxo, x, h, w, b, wp, bp, gate, scale, eps, rms, stats):
    def grad_of(p):
        return x.new_empty(p.shape if p is not None else 0, dtype=torch.float32)

    return (torch.empty_like(x), torch.empty_like(h), grad_of(w), grad_of(b), grad_of(wp),
            grad_of(bp), grad_of(gate))


def _setup(ctx, inputs, output):
    x, h, w, b, wp, bp, gate, scale, eps, rms, _ = inputs
    xo, y, stats = output
    ctx.save_for_backward(x, h, w, b, wp, bp, gate, stats)
    ctx.cfg = (scale, eps, rms)
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
    dx, dh, dw, db, dwp, dbp, dgate = _bwd(dy.contiguous(), dxo, x, h, w, b, wp, bp, gate,
                                           *ctx.cfg, stats)
    given = (dw, db if b is not None else None, dwp if wp is not None else None,
             dbp if bp is not None else None, dgate if gate is not None else None)
    return (dx, dh, *given, None, None, None, None)


_fwd.register_autograd(_grad, setup_context=_setup)


def _param(name, p, shape, device):
    if p is None:
        return None
    if tuple(p.shape) != shape or p.device != device or p.dtype not in _DTYPES:
        raise ValueError(f"residual_norm: {name} must be float32 or bfloat16 {shape} on x's "
                         f"device, got {p.dtype} {tuple(p.shape)}")
    return p.float().contiguous()


def _gates(gate, x):
    """The gate as (G, C) rows, each shared by N / G rows of x in turn."""
    if gate is None:
        return None
    C = x.shape[-1]
    if gate.device != x.device or gate.dtype not in _DTYPES:
        raise ValueError("residual_norm: gate must be float32 or bfloat16 on x's device, got "
                         f"{gate.dtype}")
    if tuple(gate.shape) == (C,):
        return gate.float().reshape(1, C).contiguous()
    one_per_sample = [(x.shape[0], *(1,) * (x.dim() - 2), C), (x.shape[0], C)]
    if x.dim() >= 2 and tuple(gate.shape) in one_per_sample and 0 < x.shape[0] <= MAX_GATES:
        return gate.float().reshape(x.shape[0], C).contiguous()
    raise ValueError(f"residual_norm: gate must be (C,) or one row for each of the first "
                     f"dimension's entries (at most {MAX_GATES}), got {tuple(gate.shape)} for x "
                     f"{tuple(x.shape)}")


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
    may be bfloat16.  Differentiable in every tensor (``sqrtblock::residual_norm_fwd/bwd``);
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
    xo, y, _ = _fwd(x.reshape(-1, C).contiguous(), h.reshape(-1, C).contiguous(), w, b, wp, bp,
                    _gates(gate, x), scale, eps, kind == "rms", out_dtype)
    return xo.view(x.shape), y.view(x.shape)
