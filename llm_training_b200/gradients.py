"""Global gradient norm over many tensors, and clipping (csrc/sqb_gradclip.cu)."""

from __future__ import annotations

import math

import torch

from . import _lib

__all__ = ["grad_norm", "clip_grads", "clip_grad_norm_", "clip_grad_norm_supported"]

_DTYPES = {torch.float32, torch.bfloat16}


def _dense(t):
    """Whether t's elements fill one run of memory, in whatever order."""
    at = 1
    for stride, size in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n > 1):
        if stride != at:
            return False
        at *= size
    return True


def _overlap(tensors, more=()):
    """Whether two of `tensors`, or one of them and one of `more`, have memory in common (all
    without gaps)."""
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), mine)
                   for group, mine in ((tensors, True), (more, False)) for t in group if t.numel())
    reach = {True: 0, False: 0}  # how far the spans so far go, of either kind
    for start, end, mine in spans:
        if start < reach[True] or (mine and start < reach[False]):
            return True
        reach[mine] = max(reach[mine], end)
    return False


def _checked(fn, tensors, what="gradients"):
    """The device of `tensors`, all of them strided CUDA float32 or bfloat16 on it."""
    device = tensors[0].device
    if ({t.layout for t in tensors} != {torch.strided}
            or not {t.dtype for t in tensors} <= _DTYPES
            or {t.device for t in tensors} != {device}):
        for t in tensors:
            if t.layout != torch.strided:
                raise ValueError(f"{fn}: {what} must be strided tensors, got layout {t.layout}")
            if t.dtype not in _DTYPES:
                raise TypeError(f"{fn} supports float32 and bfloat16, got {t.dtype}")
            if t.device != device:
                raise ValueError(f"{fn}: {what} are on {device} and {t.device}: one call takes "
                                 "one device")
    if device.type != "cuda":
        raise RuntimeError(f"{fn}: {what} must be CUDA tensors (the op has no CPU "
                           "implementation)")
    return device


def _done(fn, result):
    if result is None:
        raise RuntimeError(f"{fn}: needs ordinary CUDA tensors that do not share memory")
    return result


# ---- the operators, on tensors that fill one run of memory each.  An eager call goes to the
# C++ binding; these are the same launches registered as custom ops, for traced calls.


@torch.library.custom_op("sqrtblock::grad_norm", mutates_args=())
def _grad_norm(tensors: list[torch.Tensor]) -> torch.Tensor:
    return _done("grad_norm", _lib.binding().grad_norm(tensors))


@torch.library.custom_op("sqrtblock::clip_grads", mutates_args=())
def _clip_grads(grads: list[torch.Tensor], bf16: list[int], max_norm: float
                ) -> list[torch.Tensor]:
    """The clipped gradients, contiguous, bfloat16 where `bf16` is 1 and else float32; last
    the norm.  (It writes to none of its inputs: torch.jit loses track of lists that an op
    writes to.)"""
    out = [torch.empty(g.shape, dtype=torch.bfloat16 if b else torch.float32, device=g.device)
           for g, b in zip(grads, bf16)]
    grads = [g.contiguous() for g in grads]
    return [*out, _done("clip_grads", _lib.binding().clip(grads, out, max_norm, False))[1]]


@_grad_norm.register_fake
def _(tensors):
    return tensors[0].new_empty((), dtype=torch.float32)


@_clip_grads.register_fake
def _(grads, bf16, max_norm):
    out = [g.new_empty(g.shape, dtype=torch.bfloat16 if b else torch.float32)
           for g, b in zip(grads, bf16)]
    return [*out, grads[0].new_empty((), dtype=torch.float32)]


def _clip_traced(grads, out, max_norm):
    """(out, norm) of a traced call; out is written by ordinary copies."""
    *clipped, norm = _clip_grads(grads, [int(o.dtype == torch.bfloat16) for o in out], max_norm)
    with torch.no_grad():
        for o, c in zip(out, clipped):
            o.copy_(c)
    return out, norm


def _in_one_run(t):
    return t if t.is_contiguous() or _dense(t) else t.contiguous()


def grad_norm(tensors):
    """2-norm of all elements of ``tensors`` (CUDA float32 or bfloat16, any mixture, one
    device) as a float32 scalar on their device.  The squares are summed in 64 bits in a
    fixed order: no overflow, and the same bits on every run.  No tensors: 0."""
    fn, tensors = "grad_norm", list(tensors)
    if not tensors:
        return torch.tensor(0.0)
    eager = _lib.eager()
    norm = _lib.binding().grad_norm(tensors) if eager and tensors[0].is_cuda else None
    if norm is None:
        _checked(fn, tensors, "tensors")
        tensors = [_in_one_run(t) for t in tensors]
        norm = (_done(fn, _lib.binding().grad_norm(tensors)) if eager else _grad_norm(tensors))
    return norm


def _bound(fn, max_norm):
    max_norm = float(max_norm)
    if math.isnan(max_norm) or max_norm < 0:
        raise ValueError(f"{fn}: max_norm must not be negative, got {max_norm}")
    return max_norm


def clip_grads(grads, max_norm, out=None):
    """(out, norm): the ``grads`` (CUDA float32 or bfloat16, any mixture, one device)
    times min(1, max_norm / (norm + 1e-6)), norm their global 2-norm as ``grad_norm``
    computes it, written to ``out``: one tensor for each gradient, of its shape, float32
    or bfloat16 (an optimizer's fp32 buffers for bf16 gradients: the factor is applied
    before the only rounding), sharing no memory with any gradient unless it is the same
    tensor (any overlap is refused).  None: new tensors like the gradients."""
    fn = "clip_grads"
    grads, max_norm = list(grads), _bound(fn, max_norm)
    if not grads:
        return [], torch.tensor(0.0)
    out, eager = list(out) if out is not None else None, _lib.eager()
    done = _lib.binding().clip(grads, out, max_norm, False) if eager and grads[0].is_cuda else None
    if done is None:
        device = _checked(fn, grads)
        if out is not None:
            _check_out(fn, grads, out, device)
            if eager:
                _check_memory(fn, grads, out)
        if not eager and out is not None:
            return _clip_traced(grads, out, max_norm)
        if not eager:
            *out, norm = _clip_grads(grads, [int(g.dtype == torch.bfloat16) for g in grads], max_norm)
            return out, norm
        grads = [g.contiguous() for g in grads]
        done = _done(fn, _lib.binding().clip(grads, out, max_norm, False))
    return out if out is not None else done[0], done[1]


def _check_out(fn, grads, out, device):
    if [o.shape for o in out] != [g.shape for g in grads]:
        raise ValueError(f"{fn}: out must hold one tensor of each gradient's shape")
    if _checked(fn, out, "out") != device:
        raise ValueError(f"{fn}: out must be on the gradients' device, {device}")
    if not all([o.is_contiguous() for o in out]):
        raise ValueError(f"{fn}: out must be contiguous")


def _check_memory(fn, grads, out):
    at = {o.data_ptr(): i for i, o in enumerate(out) if o.numel()}
    if len(at) < sum(o.numel() > 0 for o in out):
        raise ValueError(f"{fn}: out holds one tensor twice")
    if any([at.get(g.data_ptr(), i) != i for i, g in enumerate(grads)]):
        raise ValueError(f"{fn}: out holds another gradient's memory")
    if any([o.data_ptr() == g.data_ptr() and (o.dtype != g.dtype or not g.is_contiguous())
            for g, o in zip(grads, out) if o.numel()]):
        raise ValueError(f"{fn}: out holds a gradient's memory in another layout or dtype")
    if _overlap(out):
        raise ValueError(f"{fn}: out holds tensors that overlap")
    runs = [g for g in grads if g.is_contiguous()]  # others are copied first
    ours = {o.data_ptr() for o in out}
    placed = [g for g in runs if g.data_ptr() in ours]
    if _overlap([o for o in out if o.data_ptr() not in {g.data_ptr() for g in placed}], runs) or (
            _overlap(placed, [g for g in runs if g.data_ptr() not in ours])):
        raise ValueError(f"{fn}: out overlaps a gradient that it is not")


def clip_grad_norm_supported(parameters) -> bool:
    """Whether ``clip_grad_norm_`` takes the gradients of ``parameters`` (an iterable of tensors,
    or one): ordinary strided CUDA float32 and bfloat16 tensors on one device, one at least."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    return (bool(grads) and grads[0].is_cuda and {type(g) for g in grads} == {torch.Tensor}
            and {g.dtype for g in grads} <= _DTYPES and {g.layout for g in grads} == {torch.strided}
            and len({g.device for g in grads}) == 1)


def clip_grad_norm_(parameters, max_norm):
    """Scales the gradients of ``parameters`` (an iterable of tensors, or one) in place so
    that their global 2-norm is at most ``max_norm``, and returns the norm before, a
    float32 scalar: ``torch.nn.utils.clip_grad_norm_`` for CUDA float32 and bfloat16
    gradients on one device, with the norm of ``grad_norm``.  A parameter listed twice
    counts once; parameters that share one gradient tensor, and gradients that overlap, are
    refused.  Gradients below the bound are not written.  A NaN norm makes every
    gradient NaN, as there.  No gradients: 0."""
    fn = "clip_grad_norm_"
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    # a parameter listed twice is counted and scaled once
    grads = [p.grad for p in dict.fromkeys(parameters) if p.grad is not None]
    max_norm = _bound(fn, max_norm)
    if not grads:
        return torch.tensor(0.0)
    eager = _lib.eager()
    done = _lib.binding().clip(grads, None, max_norm, True) if eager and grads[0].is_cuda else None
    if done is not None:
        return done[1]
    _checked(fn, grads)
    if not eager:
        return _clip_traced(grads, grads, max_norm)[1]
    at = [g.data_ptr() for g in grads if g.numel()]
    if len(set(at)) < len(at):
        raise ValueError(f"{fn}: two parameters share one gradient")
    if _overlap([g for g in grads if g.is_contiguous() or _dense(g)]):
        raise ValueError(f"{fn}: two gradients overlap")
    # a gradient with gaps (a view of a larger buffer) goes through a copy
    for g in grads:
        if any(s == 0 and n > 1 for n, s in zip(g.shape, g.stride())):
            raise ValueError(f"{fn}: a gradient expanded over its own memory cannot be scaled "
                             "in place")
    work = [_in_one_run(g) for g in grads]
    _, norm = _done(fn, _lib.binding().clip(work, None, max_norm, True))
    with torch.no_grad():
        for g, w in zip(grads, work):
            if w is not g:
                g.copy_(w)
    return norm
