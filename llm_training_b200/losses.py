"""Losses that train on a model's answers: token log-probabilities, a preference loss
over pairs of answers and a clipped policy loss with a KL term (csrc/sqb_logits.cu).

All take CUDA float32 or bfloat16 logits with unit stride on the vocabulary (any other
strides that do not overlap) and integer targets, where a negative target leaves its
token out (the prompt, the padding): such a row of logits is not read and its gradient
is zero.  A batch of S sequences is padded, logits (S, T, V) with targets (S, T), or
packed, logits (N, V) with targets (N,) and ``cu_seqlens`` (S + 1,), the sequences'
first rows and their end, non-decreasing; rows outside ``[cu_seqlens[0],
cu_seqlens[S])`` are left out too.  A target past the vocabulary is never read: its
log-probability and gradient row are NaN, as is everything summed from them.  Gradients
reach the logits only, once (a second derivative is refused), in the logits' dtype and, as
far as those leave no large gaps, with their strides.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib

__all__ = ["token_log_probs", "preference_loss", "policy_loss", "policy_loss_and_grad"]

_DTYPES = (torch.float32, torch.bfloat16)
_INTEGERS = (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8)


def _grad_strides(x):
    """Strides of the gradient, as the binding makes it: x's, or where x's rows lie far apart
    (a few tokens of a longer batch) ones without the gaps, that keep every row's place
    between 16-byte boundaries."""
    strides = x.stride()
    if x.numel() == 0 or 1 + sum((n - 1) * s for n, s in zip(x.shape, strides)) <= 2 * x.numel():
        return strides
    step, got = 16 // x.element_size(), [1]
    span = x.shape[-1]
    for n, s in zip(reversed(x.shape[:-1]), reversed(strides[:-1])):
        span += (s - span) % step
        got.append(span)
        span *= n
    return tuple(reversed(got))


def _fake_grad(x):
    return torch.empty_strided(x.shape, _grad_strides(x), dtype=x.dtype, device=x.device)


# ---- the operators --------------------------------------------------------------------
# x is (S, T, V), or (N, V) as one sequence; t int64, contiguous, one target a row.  An eager
# call goes to the C++ binding, which has the autograd nodes; these are the same launches
# registered as custom ops, for traced calls.


def _dims(x):
    """(S, T, V, sequence stride, token stride)"""
    if x.dim() == 2:
        return (1, *x.shape, 0, x.stride(0))
    return (*x.shape, x.stride(0), x.stride(1))


@torch.library.custom_op("sqrtblock::logp_fwd", mutates_args=())
def _logp_fwd(x: torch.Tensor, t: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(logp in t's shape, row statistics (2 S T,))."""
    return _lib.binding().logp_fwd(x, t)


@_logp_fwd.register_fake
def _(x, t):
    return (x.new_empty(t.shape, dtype=torch.float32),
            x.new_empty(2 * t.numel(), dtype=torch.float32))


@torch.library.custom_op("sqrtblock::logp_bwd", mutates_args=())
def _logp_bwd(x: torch.Tensor, t: torch.Tensor, stats: torch.Tensor,
              g_row: Optional[torch.Tensor], scale: Optional[torch.Tensor]) -> torch.Tensor:
    """g_row[r] * scale * ([c == t] - softmax) in x's dtype; without a g_row the factors follow
    the row statistics."""
    return _lib.binding().logp_bwd(x, t, stats, g_row, scale)


@_logp_bwd.register_fake
def _(x, t, stats, g_row, scale):
    return _fake_grad(x)


def _logp_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs, output[1])
    ctx.mark_non_differentiable(output[1])


def _logp_grad(ctx, dlogp, _dstats):
    return _logp_bwd(*ctx.saved_tensors, dlogp.to(torch.float32).contiguous(), None), None


_logp_fwd.register_autograd(_logp_grad, setup_context=_logp_setup)


@torch.library.custom_op("sqrtblock::preference_fwd", mutates_args=())
def _preference_fwd(x: torch.Tensor, t: torch.Tensor, ref: Optional[torch.Tensor],
                    cu: Optional[torch.Tensor], pairs: int, beta: float, label_smoothing: float
                    ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(loss, rewards (2, P), row statistics and d loss / d logp of each row (3 S T floats, and
    scratch))."""
    return _lib.binding().preference_fwd(x, t, ref, cu, pairs, beta, label_smoothing)


@_preference_fwd.register_fake
def _(x, t, ref, cu, pairs, beta, label_smoothing):
    f32, N = torch.float32, t.numel()
    up = lambda n: -(-n // 256) * 256  # noqa: E731
    scratch = up(8 * N) + 8 * pairs  # sqb_preference_workspace_bytes
    return (x.new_empty((), dtype=f32), x.new_empty((2, pairs), dtype=f32),
            x.new_empty((up(12 * N) + scratch + 3) // 4, dtype=f32))


def _loss_setup(ctx, inputs, output):
    _, *others, last = output
    ctx.save_for_backward(*inputs[:2], last)
    ctx.mark_non_differentiable(*others, last)
    ctx.arguments = len(inputs)


def _loss_grad(ctx, dloss, *_):
    x, t, rows = ctx.saved_tensors
    return (_logp_bwd(x, t, rows, None, dloss.to(torch.float32)),) + (None,) * (
        ctx.arguments - 1)


_preference_fwd.register_autograd(_loss_grad, setup_context=_loss_setup)


@torch.library.custom_op("sqrtblock::policy_fwd", mutates_args=())
def _policy_fwd(x: torch.Tensor, t: torch.Tensor, adv: torch.Tensor,
                old: Optional[torch.Tensor], ref: Optional[torch.Tensor],
                cu: Optional[torch.Tensor], seqs: int, adv_by_seq: bool, per_seq: bool,
                clip_low: float, clip_high: float, kl_coef: float, grad_scale: Optional[float]
                ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(loss, logps, (policy term, KL, clipped share), last): `last` is the logits' gradient
    times grad_scale, or for None the row statistics and d loss / d logp (3 S T,)."""
    return _lib.binding().policy_fwd(x, t, adv, old, ref, cu, seqs, adv_by_seq, per_seq,
                                     clip_low, clip_high, kl_coef, grad_scale)


@_policy_fwd.register_fake
def _(x, t, adv, old, ref, cu, seqs, adv_by_seq, per_seq, clip_low, clip_high, kl_coef,
      grad_scale):
    f32 = torch.float32
    last = _fake_grad(x) if grad_scale is not None else x.new_empty(3 * t.numel(), dtype=f32)
    return (x.new_empty((), dtype=f32), x.new_empty(t.shape, dtype=f32),
            x.new_empty(3, dtype=f32), last)


_policy_fwd.register_autograd(_loss_grad, setup_context=_loss_setup)


# ---- public entry points --------------------------------------------------------------


def _disjoint(x):
    """Whether the rows of x, unit stride on V, occupy different memory."""
    S, T, V, ss, st = _dims(x)
    if S <= 1 or T <= 1:
        return (S <= 1 or ss >= V) and (T <= 1 or st >= V)
    return (st >= V and ss >= (T - 1) * st + V) or (ss >= V and st >= (S - 1) * ss + V)


def _rows(fn, logits, targets):
    """Logits as (S, T, V) or (N, V) and int64 targets, checked."""
    if not logits.is_cuda:
        raise RuntimeError(f"{fn}: logits must be a CUDA tensor (the op has no CPU "
                           "implementation)")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"{fn} supports float32 and bfloat16 logits, got {logits.dtype}")
    shape = logits.shape
    if len(shape) < 2 or shape[-1] == 0:
        raise ValueError(f"{fn}: logits must be (..., tokens, V), got {tuple(shape)}")
    if targets.shape != shape[:-1] or targets.device != logits.device:
        raise ValueError(f"{fn}: one target per row of logits on their device, got targets "
                         f"{tuple(targets.shape)} for logits {tuple(shape)}")
    if targets.dtype not in _INTEGERS:
        raise TypeError(f"{fn}: targets must be integers, got {targets.dtype}")
    x, t = logits, targets
    if len(shape) > 3:
        x = x.reshape(math.prod(shape[:-2]), *shape[-2:])
    if t.numel() > 2**31 - 1 or shape[-1] > 2**30:
        raise ValueError(f"{fn}: at most 2**31 - 1 rows of at most 2**30 logits")
    if (x.stride(-1) != 1 and shape[-1] > 1) or not _disjoint(x):
        x = x.contiguous()
    return x, t.to(torch.int64).contiguous()


def _sequences(fn, logits, targets, cu_seqlens):
    """(x, t, cu_seqlens as int64 or None, sequences)."""
    if cu_seqlens is None:
        if logits.dim() != 3:
            raise ValueError(f"{fn}: logits must be (sequences, tokens, V), or (rows, V) with "
                             f"cu_seqlens, got {tuple(logits.shape)}")
        x, t = _rows(fn, logits, targets)
        return x, t, None, x.shape[0]
    if logits.dim() != 2:
        raise ValueError(f"{fn}: with cu_seqlens logits must be (rows, V), got "
                         f"{tuple(logits.shape)}")
    if (cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2
            or cu_seqlens.dtype not in (torch.int32, torch.int64)
            or cu_seqlens.device != logits.device):
        raise ValueError(f"{fn}: cu_seqlens must be int32 or int64 (sequences + 1,) on the "
                         "logits' device")
    x, t = _rows(fn, logits, targets)
    return x, t, cu_seqlens.to(torch.int64).contiguous(), cu_seqlens.numel() - 1


def _given(fn, name, v, shapes, device):
    """A fixed input as contiguous float32 of one of `shapes`."""
    if v is None:
        return None
    if tuple(v.shape) not in shapes or v.device != device or not v.dtype.is_floating_point:
        raise ValueError(f"{fn}: {name} must be floating point of shape "
                         f"{' or '.join(map(str, shapes))} on the logits' device, got {v.dtype} "
                         f"{tuple(v.shape)}")
    if v.requires_grad:
        raise ValueError(f"{fn}: no gradient reaches {name}: pass it detached")
    return v.to(torch.float32).contiguous()


def _number(fn, name, v, least=0.0, most=math.inf):
    v = float(v)
    if not least <= v <= most:
        raise ValueError(f"{fn}: {name} must be in [{least}, {most}], got {v}")
    return v


def token_log_probs(logits, targets):
    """Log-probability of each target under its row of logits (..., tokens, V), float32 in
    the targets' shape; 0 where the target is negative.  Differentiable in the logits
    (``sqrtblock::logp_fwd/bwd``): one read of the logits forward, and one read and one
    write backward, with no softmax kept in between."""
    x, t = _rows("token_log_probs", logits, targets)
    return _lib.binding().logp(x, t) if _lib.plain(x, t) else _logp_fwd(x, t)[0]


def preference_loss(logits, targets, ref_logps=None, *, beta=0.1, label_smoothing=0.0,
                    cu_seqlens=None):
    """Preference loss over P pairs of answers -> (loss, chosen rewards, rejected rewards).

    Of the 2P sequences the first P are the chosen answers and the last P the rejected
    ones, in the same order.  With s the sum of a sequence's token log-probabilities and
    ``ref_logps`` (2P,) the same sums under the reference model (None: zeros),

        z = beta * ((s_chosen - ref_chosen) - (s_rejected - ref_rejected))
        loss = mean of -(1 - label_smoothing) log sigmoid(z) - label_smoothing log sigmoid(-z)

    and the rewards (P,) are beta * (s - ref), for logging (not differentiable).  Sums
    and the loss are computed in 64 bits.  One read of the logits forward, one read and
    one write backward: a pair's factor is known only after its last token."""
    fn = "preference_loss"
    x, t, cu, seqs = _sequences(fn, logits, targets, cu_seqlens)
    if seqs == 0 or seqs % 2:
        raise ValueError(f"{fn}: {seqs} sequences are no pairs")
    ref = _given(fn, "ref_logps", ref_logps, [(seqs,)], x.device)
    beta = _number(fn, "beta", beta, most=1e30)
    label_smoothing = _number(fn, "label_smoothing", label_smoothing, most=1.0)
    args = (x, t, ref, cu, seqs // 2, beta, label_smoothing)
    if _lib.plain(*args[:4]):
        return _lib.binding().preference(*args)
    loss, rewards, _ = _preference_fwd(*args)
    return (loss, *rewards.unbind(0))


def _policy_args(fn, logits, targets, advantages, old_logps, ref_logps, clip, clip_high, kl_coef,
                 reduction, cu_seqlens):
    x, t, cu, seqs = _sequences(fn, logits, targets, cu_seqlens)
    if reduction not in ("token", "sequence"):
        raise ValueError(f"{fn}: reduction must be 'token' or 'sequence', got {reduction!r}")
    if seqs == 0:
        raise ValueError(f"{fn}: no sequences")
    shape = tuple(targets.shape)
    by_seq = [(seqs,)] if cu is not None else [(seqs,), (seqs, 1)]
    adv = _given(fn, "advantages", advantages, [shape] + [s for s in by_seq if s != shape],
                 x.device)
    if adv is None:
        raise ValueError(f"{fn}: advantages are needed")
    old = _given(fn, "old_logps", old_logps, [shape], x.device)
    ref = _given(fn, "ref_logps", ref_logps, [shape], x.device)
    clip = _number(fn, "clip", clip)
    clip_high = clip if clip_high is None else _number(fn, "clip_high", clip_high)
    kl_coef = _number(fn, "kl_coef", kl_coef, most=1e30)
    if kl_coef and ref is None:
        raise ValueError(f"{fn}: a KL term needs ref_logps")
    return (x, t, adv, old, ref, cu, seqs, tuple(adv.shape) != shape, reduction == "sequence",
            clip, clip_high, kl_coef)


def policy_loss(logits, targets, advantages, old_logps=None, ref_logps=None, *, clip=0.2,
                clip_high=None, kl_coef=0.0, reduction="token", cu_seqlens=None):
    """Clipped policy loss with a KL term -> (loss, log-probabilities, statistics).

    Per counted token, with logp its log-probability, r = exp(logp - old_logps) (1 where
    ``old_logps`` is None: the sampling policy is this one) and A its advantage,

        -min(r A, min(max(r, 1 - clip), 1 + clip_high) A)
            + kl_coef (exp(ref_logps - logp) - (ref_logps - logp) - 1)

    averaged over the counted tokens (``reduction="token"``), or over each sequence's
    counted tokens and then over the sequences that have any (``"sequence"``); 0 where no
    token is counted.  ``clip_high`` None is ``clip``; with a ``kl_coef`` of 0 ``ref_logps``
    serve the statistics alone, whatever they hold.  ``old_logps`` and ``ref_logps``
    have the targets' shape, ``advantages`` that or one value per sequence (a 1-D tensor
    of as many values as a packed batch has rows is one per token).  The gradient of a
    token on the clip's border is the unclipped one.  What the inputs hold at tokens that
    are left out is not looked at.

    The log-probabilities (float32, the targets' shape, 0 at tokens left out) and the
    statistics - (mean policy term, mean KL, share of clipped tokens), averaged as the
    loss - are for logging and for the next step's ``old_logps``, not differentiable."""
    args = _policy_args("policy_loss", logits, targets, advantages, old_logps, ref_logps, clip,
                        clip_high, kl_coef, reduction, cu_seqlens)
    if _lib.plain(*args[:6]):
        return _lib.binding().policy(*args)
    return _policy_fwd(*args, None)[:3]


def policy_loss_and_grad(logits, targets, advantages, old_logps=None, ref_logps=None, *,
                         clip=0.2, clip_high=None, kl_coef=0.0, reduction="token",
                         cu_seqlens=None, grad_scale=1.0):
    """``policy_loss`` and its gradient in one pass over the logits -> (loss, gradient,
    log-probabilities, statistics).

    The gradient (the logits' shape and dtype) is that of ``grad_scale * loss``;
    hand it on with ``logits.backward(gradient)``.  A token's factor needs its own row
    only, so each row is read from HBM once and its gradient written once, where the
    autograd form reads the logits a second time."""
    fn = "policy_loss_and_grad"
    args = _policy_args(fn, logits.detach(), targets, advantages, old_logps, ref_logps, clip,
                        clip_high, kl_coef, reduction, cu_seqlens)
    grad_scale = _number(fn, "grad_scale", grad_scale, least=-1e30, most=1e30)
    run = _lib.binding().policy_fwd if _lib.plain(*args[:6]) else _policy_fwd
    loss, logps, stats, grad = run(*args, grad_scale)
    return loss, grad, logps, stats
