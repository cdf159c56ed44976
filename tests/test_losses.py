"""Token log-probabilities, the preference loss and the clipped policy loss.

CPU: refusals, argument checks of the C entry points, fake implementations.  GPU: values
and gradients against the definition in 64 bits (log_softmax and autograd in float64),
with bounds that count the roundings:

* a row's sum s of exp(x - m) is added up in fp32 over V / threads terms a thread (at
  most V / 32 + 8) and a tree of at most 10 levels; each exponential is off by two units
  (2^-22) and by at most the rounding of its argument, |x - m| * 2^-23.  Terms further
  than 30 below the maximum weigh nothing, so relative error of s <= rel(V) below, and
  log s is off by as much;
* a log-probability stored in fp32 is off by 2^-24 of itself more;
* a gradient element g ([c == t] - exp / s) is off by rel(V) of g p, 2^-23 of g at the
  target (the sum) and, rounded to its type, by half a step: finfo.eps / 2."""

import ctypes
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from llm_training_b200 import _lib, ops

ERR_ARG, ERR_DTYPE, ERR_ALIGN, ERR_WORKSPACE = 1, 2, 3, 5  # include/sqrtblock.h
U = 2.0**-24  # half a step of fp32, relative


def rel(V):
    return (V / 32 + 8 + 10 + 4 + 60 + 8) * U if V <= 4096 else (V / 256 + 90) * U


# ---- CPU: refusals ----------------------------------------------------------------


def _cuda(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="cuda")


def test_cpu_logits_are_refused():
    x, t = torch.zeros(2, 3, 5), torch.zeros(2, 3, dtype=torch.int64)
    for call in (lambda: ops.token_log_probs(x, t), lambda: ops.preference_loss(x, t),
                 lambda: ops.policy_loss(x, t, torch.zeros(2)),
                 lambda: ops.policy_loss_and_grad(x, t, torch.zeros(2))):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


def test_bad_arguments_are_refused():
    i64 = torch.int64
    with FakeTensorMode():
        x, t = _cuda(4, 3, 5), _cuda(4, 3, dtype=i64)
        packed, tp, cu = _cuda(12, 5), _cuda(12, dtype=i64), _cuda(5, dtype=i64)
        adv = _cuda(4)
        cases = [
            (TypeError, "float32 and bfloat16", lambda: ops.token_log_probs(x.half(), t)),
            (TypeError, "integers", lambda: ops.token_log_probs(x, t.float())),
            (ValueError, "one target per row", lambda: ops.token_log_probs(x, t[:, :2])),
            (ValueError, "must be", lambda: ops.token_log_probs(_cuda(5), _cuda(dtype=i64))),
            (ValueError, "must be", lambda: ops.token_log_probs(_cuda(4, 3, 0), t)),
            (ValueError, "no pairs", lambda: ops.preference_loss(x[:3], t[:3])),
            (ValueError, "no pairs", lambda: ops.preference_loss(x[:0], t[:0])),
            (ValueError, "with cu_seqlens", lambda: ops.preference_loss(packed, tp)),
            (ValueError, "with cu_seqlens", lambda: ops.preference_loss(x, t, cu_seqlens=cu)),
            (ValueError, "cu_seqlens must", lambda: ops.preference_loss(
                packed, tp, cu_seqlens=cu.float())),
            (ValueError, "cu_seqlens must", lambda: ops.preference_loss(
                packed, tp, cu_seqlens=cu[:1])),
            (ValueError, "ref_logps", lambda: ops.preference_loss(x, t, _cuda(2))),
            (ValueError, "detached", lambda: ops.preference_loss(
                x, t, _cuda(4).requires_grad_(True))),
            (ValueError, "beta", lambda: ops.preference_loss(x, t, beta=-1.0)),
            (ValueError, "beta", lambda: ops.preference_loss(x, t, beta=math.nan)),
            (ValueError, "label_smoothing", lambda: ops.preference_loss(
                x, t, label_smoothing=1.5)),
            (ValueError, "advantages", lambda: ops.policy_loss(x, t, _cuda(3))),
            (ValueError, "advantages", lambda: ops.policy_loss(x, t, None)),
            (ValueError, "advantages", lambda: ops.policy_loss(
                packed, tp, _cuda(4, 1), cu_seqlens=cu)),
            (ValueError, "old_logps", lambda: ops.policy_loss(x, t, adv, _cuda(4))),
            (ValueError, "ref_logps", lambda: ops.policy_loss(x, t, adv, kl_coef=0.1)),
            (ValueError, "clip", lambda: ops.policy_loss(x, t, adv, clip=-0.1)),
            (ValueError, "clip_high", lambda: ops.policy_loss(x, t, adv, clip_high=math.nan)),
            (ValueError, "reduction", lambda: ops.policy_loss(x, t, adv, reduction="sum")),
            (ValueError, "grad_scale", lambda: ops.policy_loss_and_grad(
                x, t, adv, grad_scale=math.inf)),
            (ValueError, "grad_scale", lambda: ops.policy_loss_and_grad(
                x, t, adv, grad_scale=-1e39)),
        ]
        for kind, text, call in cases:
            with pytest.raises(kind, match=text):
                call()


def test_c_entry_points_reject_bad_arguments_without_a_device():
    lib, p = _lib.lib(), ctypes.c_void_p(16)
    assert lib.sqb_logp_fwd(None, p, p, p, 1, 4, 8, 32, 8, 1, None) == ERR_ARG
    assert lib.sqb_logp_fwd(p, p, p, p, 0, 4, 8, 32, 8, 1, None) == ERR_ARG
    assert lib.sqb_logp_fwd(p, p, p, p, 2**20, 2**12, 8, 32, 8, 1, None) == ERR_ARG
    assert lib.sqb_logp_fwd(p, p, p, p, 1, 4, 2**31, 32, 8, 1, None) == ERR_ARG
    assert lib.sqb_logp_fwd(p, p, p, p, 1, 4, 8, 32, 8, 7, None) == ERR_DTYPE
    assert lib.sqb_logp_bwd(p, p, p, None, p, p, 1, 4, 8, 32, 8, 32, 8, 1, None) == ERR_ARG
    assert lib.sqb_logp_bwd(p, p, p, p, p, p, 1, 4, 8, 32, 8, 32, 8, 9, None) == ERR_DTYPE

    def preference(x=p, cu=None, P=2, S=4, T=3, dtype=1, ws=p, nbytes=1 << 20, loss=p):
        return lib.sqb_preference_fwd(x, p, cu, p, P, .1, 0., loss, p, p, p, S, T, 8, 24, 8, dtype,
                                      ws, nbytes, None)

    assert preference(x=None) == ERR_ARG and preference(loss=None) == ERR_ARG
    assert preference(P=0) == ERR_ARG and preference(P=3) == ERR_ARG and preference(T=-1) == ERR_ARG
    assert preference(cu=p) == ERR_ARG and preference(dtype=4) == ERR_DTYPE
    assert preference(ws=None) == ERR_WORKSPACE and preference(nbytes=64) == ERR_WORKSPACE
    assert preference(ws=ctypes.c_void_p(20)) == ERR_ALIGN

    def policy(adv=p, cu=None, seqs=4, S=4, dtype=1, ws=p, nbytes=1 << 20, logp=p):
        return lib.sqb_policy_fwd(p, p, cu, seqs, None, None, adv, 1, .2, .2, 0., 0, p, p, logp, p,
                                  p, None, 1., S, 3, 8, 24, 8, 24, 8, dtype, ws, nbytes, None)

    assert policy(adv=None) == ERR_ARG and policy(logp=None) == ERR_ARG
    assert policy(seqs=3) == ERR_ARG and policy(cu=p) == ERR_ARG and policy(seqs=0) == ERR_ARG
    assert policy(dtype=4) == ERR_DTYPE
    assert policy(ws=None) == ERR_WORKSPACE and policy(nbytes=64) == ERR_WORKSPACE
    assert policy(ws=ctypes.c_void_p(20)) == ERR_ALIGN


def test_fakes_keep_shapes_dtypes_and_strides():
    with FakeTensorMode():
        x = _cuda(4, 3, 40, dtype=torch.bfloat16)[..., :37].requires_grad_(True)
        t = _cuda(4, 3, dtype=torch.int32)
        lp = ops.token_log_probs(x, t)
        assert lp.shape == (4, 3) and lp.dtype == torch.float32
        loss, a, b = ops.preference_loss(x, t, _cuda(4))
        assert loss.shape == () and a.shape == b.shape == (2,)
        loss, logps, stats = ops.policy_loss(x, t, _cuda(4, 1), lp.detach(), lp.detach(),
                                             kl_coef=0.1)
        assert logps.shape == (4, 3) and stats.shape == (3,) and not logps.requires_grad
        loss, grad, logps, _ = ops.policy_loss_and_grad(x, t, _cuda(4))
        assert grad.shape == x.shape and grad.dtype == x.dtype and grad.stride() == x.stride()


# ---- GPU: inputs ----------------------------------------------------------------------


def batch(S, T, V, dtype, layout, seed=0, masked=0.3):
    """(logits, targets, cu_seqlens or None, sequences' rows): `layout` says how they lie."""
    g = torch.Generator().manual_seed(seed)
    lens = [T] * S
    if layout == "packed":
        lens = [int(n) for n in torch.randint(0, T + 1, (S,), generator=g)]
        lens[0], lens[-1] = T, min(1, T)
        rows = sum(lens) + 2  # two rows behind the last sequence
        shape = (rows,)
    else:
        shape = (S, T)
    x = torch.randn(*shape, V, generator=g) * 3
    t = torch.randint(0, V, shape, generator=g)
    x.scatter_add_(-1, t[..., None], 4 * torch.rand(*shape, 1, generator=g))
    if layout == "inf":  # columns that take no probability, and some of the lowest value
        dead = V // 3
        x[..., V - dead:] = -math.inf
        x[..., V - dead - 1] = torch.finfo(dtype).min
        t.remainder_(max(1, V - dead - 1))
    x = x.to(dtype)
    keep = torch.rand(shape, generator=g) >= masked
    if layout == "none":
        keep[:] = False
    elif layout == "nan":  # nothing that is left out may be looked at
        x[~keep] = math.nan
    t = torch.where(keep, t, -100)
    x, t, cu = x.cuda(), t.cuda(), None
    if layout == "pitch":
        buf = torch.full((S, T, V + 13), 5.0, dtype=dtype, device="cuda")
        buf[..., :V] = x
        x = buf[..., :V]
    elif layout == "phase":  # rows that start between two 16-byte boundaries
        buf = torch.zeros(S * T * V + 3, dtype=dtype, device="cuda")
        buf[3:] = x.reshape(-1)
        x = buf[3:].view(S, T, V)
    elif layout == "slice":  # all but the last token
        buf = torch.cat([x, torch.full_like(x[:, :1], 9.0)], 1)
        x = buf[:, :-1]
    elif layout == "transposed":
        x = x.transpose(0, 1).contiguous().transpose(0, 1)
    elif layout == "strided":
        buf = torch.zeros(S, T, 2 * V, dtype=dtype, device="cuda")
        buf[..., ::2] = x
        x = buf[..., ::2]
    if layout == "packed":
        at = [sum(lens[:i]) for i in range(S + 1)]
        cu = torch.tensor(at, device="cuda", dtype=torch.int32 if seed % 2 else torch.int64)
        spans = list(zip(at[:-1], at[1:]))
        t[-2:] = 0  # behind the last sequence: left out all the same
    else:
        spans = [(i * T, (i + 1) * T) for i in range(S)]
    return x, t, cu, spans


def exact_logps(x, t, spans):
    """(x in 64 bits as a leaf, log-probabilities (rows,) with 0 where left out, counted)."""
    x64 = x.detach().double().requires_grad_(True)
    V = x.shape[-1]
    rows, tt = x64.reshape(-1, V), t.reshape(-1)
    inside = torch.zeros_like(tt, dtype=torch.bool)
    for a, b in spans:
        inside[a:b] = True
    keep = inside & (tt >= 0)
    lp = torch.zeros(tt.shape, dtype=torch.float64, device=x.device)
    at = keep.nonzero()[:, 0]
    picked = torch.log_softmax(rows[at], -1).gather(1, tt[at, None].long())[:, 0]
    return x64, lp.index_put((at,), picked), keep


def assert_within(got, want, bound, what):
    got, want, bound = got.detach().double(), want.detach().double(), torch.as_tensor(bound, dtype=torch.float64)
    bound = bound.to(got.device).expand(got.shape)
    ok = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), ok), what
    over = ((got - want).abs() - bound)[ok]
    assert over.numel() == 0 or float(over.max()) <= 0, (
        what, float(over.max()), float(bound[ok].max()))


def check_grad(got, want, x, t, g_exact, g_err):
    """Gradient rows against the exact ones; g: exact factor of each row, g_err: how far the
    kernel's may be from it."""
    V = x.shape[-1]
    assert got.shape == x.shape and got.dtype == x.dtype
    g, ge = (v.reshape(*t.shape, 1).abs() for v in (g_exact, g_err))
    p = torch.softmax(x.detach().double(), -1).nan_to_num(0.0)
    hot = torch.zeros_like(p).scatter_(-1, t.clamp_min(0).long()[..., None], 1.0)
    bound = g * (p * (rel(V) + 4 * U) + hot * 2 * U) + ge * (p + hot)
    bound = bound + want.abs() * (torch.finfo(x.dtype).eps / 2) * 1.01 + 2.0**-126
    assert_within(got, want, bound, "gradient")


LAYOUTS = ["plain", "packed", "pitch", "phase", "slice", "transposed", "strided", "inf", "nan",
           "none"]
SHAPES = [(2, 3, 1), (2, 1, 2), (4, 9, 7), (4, 33, 65), (2, 17, 1003), (4, 5, 5000),
          (2, 3, 50257)]
DTYPES = [torch.float32, torch.bfloat16]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", [v for v in LAYOUTS if v != "packed"])
@pytest.mark.parametrize("S,T,V", SHAPES)
def test_token_log_probs(S, T, V, layout, dtype):
    x, t, _, spans = batch(S, T, V, dtype, layout)
    x = x.detach().requires_grad_(True)
    lp = ops.token_log_probs(x, t)
    x64, want, keep = exact_logps(x, t, spans)
    want = want.view(t.shape)
    assert_within(lp, want, rel(V) + want.detach().abs() * 2 * U, "logp")
    assert torch.equal(lp[t < 0], torch.zeros_like(lp[t < 0]))
    up = torch.randn(t.shape, generator=torch.Generator().manual_seed(5)).cuda()
    (got,) = torch.autograd.grad(lp, x, up)
    (gx,) = torch.autograd.grad(want, x64, up.double())
    gx = torch.where((t >= 0)[..., None], gx, 0.0)
    check_grad(got, gx, x, t, torch.where(t >= 0, up, 0.0).double(), torch.zeros_like(up))
    if layout != "strided" and x.stride(1) <= 2 * V:
        assert got.stride() == x.stride() or 1 in x.shape


def _preference_exact(x, t, spans, ref, beta, smooth):
    x64, lp, keep = exact_logps(x, t, spans)
    lp.retain_grad()
    sums = torch.stack([lp[a:b].sum() for a, b in spans])
    r = sums - (ref.double() if ref is not None else 0.0)
    P = len(spans) // 2
    z = beta * (r[:P] - r[P:])
    ls = torch.nn.functional.logsigmoid
    loss = -((1 - smooth) * ls(z) + smooth * ls(-z)).mean()
    loss.backward()
    return loss.detach(), beta * r.detach(), z.detach(), lp, x64.grad, keep


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("S,T,V,beta,smooth,with_ref", [
    (2, 1, 2, 0.1, 0.0, True), (4, 9, 7, 0.5, 0.1, False), (8, 33, 65, 0.1, 0.0, True),
    (6, 17, 1003, 0.2, 0.25, True), (2, 300, 50, 0.1, 1.0, True), (2, 3, 50257, 0.1, 0.0, False),
])
def test_preference_loss(S, T, V, beta, smooth, with_ref, layout, dtype):
    x, t, cu, spans = batch(S, T, V, dtype, layout, seed=S + T)
    g = torch.Generator().manual_seed(1)
    ref = (-3.0 * T * torch.rand(S, generator=g)).cuda() if with_ref else None
    x = x.detach().requires_grad_(True)
    loss, chosen, rejected = ops.preference_loss(x, t, ref, beta=beta, label_smoothing=smooth,
                                                 cu_seqlens=cu)
    (got,) = torch.autograd.grad(loss, x, torch.tensor(1.5, device="cuda"))
    w_loss, w_rewards, z, lp, gx, keep = _preference_exact(x, t, spans, ref, beta, smooth)
    # each log-probability is off by rel(V): the sums by that times their lengths
    off = beta * max(b - a for a, b in spans) * rel(V)
    assert_within(torch.cat([chosen, rejected]), w_rewards, off + w_rewards.abs() * 2 * U,
                  "rewards")
    assert_within(loss, w_loss, 2 * off + w_loss.abs() * 2 * U, "loss")
    g_row = torch.where(keep, lp.grad, 0.0) * 1.5
    # sigmoid's slope is at most a quarter
    g_err = torch.where(keep, 1.5 * beta / (S // 2) * 2 * off / 4 + g_row.abs() * 4 * U, 0.0)
    gx = torch.where(keep.view(t.shape)[..., None], gx, 0.0) * 1.5
    check_grad(got, gx, x, torch.where(keep.view(t.shape), t, -1), g_row, g_err)
    assert torch.count_nonzero(got[~keep.view(t.shape)]) == 0


CLIPS = (0.2, 0.3)


def _policy_inputs(x, t, spans, per_token, kl, seed):
    g = torch.Generator().manual_seed(seed)
    _, lp, keep = exact_logps(x, t, spans)
    lp = lp.detach().cpu()
    old = lp + 0.25 * torch.randn(lp.shape, generator=g)
    ratio = (lp - old).exp()
    edge = ((ratio - 1 + CLIPS[0]).abs() < 1e-2) | ((ratio - 1 - CLIPS[1]).abs() < 1e-2)
    old = torch.where(edge, old - 0.05, old)  # a border has two one-sided gradients
    ref = lp + 0.5 * torch.randn(lp.shape, generator=g) if kl else None
    adv = torch.randn(lp.shape if per_token else len(spans), generator=g)
    left_out = ~keep.cpu()
    old[left_out] = math.nan
    if kl:
        ref[left_out] = math.inf
    if per_token:
        adv[left_out] = math.nan
    put = lambda v: v.float().cuda().view(t.shape) if v is not None else None  # noqa: E731
    return put(old), put(ref), put(adv) if per_token else adv.cuda()


def _policy_exact(x, t, spans, adv, old, ref, kl, reduction):
    """(loss, statistics, logp leaf, gradient, counted, bound on the loss, bound on each row's
    factor) from the definition, with every |d term / d logp| for the bounds."""
    x64, lp, keep = exact_logps(x, t, spans)
    lp.retain_grad()
    seq = torch.zeros(lp.shape, dtype=torch.long, device=lp.device)
    for i, (a, b) in enumerate(spans):
        seq[a:b] = i
    A = adv.double().reshape(-1) if adv.shape == t.shape else adv.double().reshape(-1)[seq]
    each, kls, cut, w, err = [], [], [], [], []
    counts = [int(keep[a:b].sum()) for a, b in spans]
    full = sum(c > 0 for c in counts)
    for i, (a, b) in enumerate(spans):
        k = keep[a:b].nonzero()[:, 0] + a
        r = torch.exp(lp[k] - old.double().reshape(-1)[k]) if old is not None else torch.exp(
            lp[k] - lp[k].detach())
        free, held = r * A[k], r.clamp(1 - CLIPS[0], 1 + CLIPS[1]) * A[k]
        each.append(-torch.minimum(free, held))
        cut.append((held < free).double())
        gap = ref.double().reshape(-1)[k] - lp[k] if ref is not None else 0.0 * lp[k]
        kls.append(torch.exp(gap) - gap - 1)
        err.append((free.abs() + kl * torch.exp(gap)).detach())
        share = sum(counts) if reduction == "token" else counts[i] * full
        share = 1 / share if share else 0.0
        w.append(torch.full(k.shape, share, dtype=torch.float64, device=k.device))
    each, kls, cut, w, err = (torch.cat(v) for v in (each, kls, cut, w, err))
    stats = torch.stack([(w * each).sum(), (w * kls).sum(), (w * cut).sum()])
    loss = stats[0] + kl * stats[1]
    if w.numel():
        loss.backward()
    at = torch.cat([keep[a:b].nonzero()[:, 0] + a for a, b in spans])
    row_err = torch.zeros_like(lp)
    row_err[at] = w * err
    grad = x64.grad if x64.grad is not None else torch.zeros_like(x64)
    g_row = lp.grad if lp.grad is not None else torch.zeros_like(lp)
    # |logp error| <= rel(V): a term moves by err times that, and its slope by as much; the
    # terms themselves and the weights are rounded in fp32
    V = x.shape[-1]
    e = rel(V)
    loss_err = (w * (err + kl * kls.abs())).sum().detach() * (e + 4 * U) + 2 * U * loss.detach().abs()
    stat_err = torch.stack([(w * (each.abs() * 1.5 + 1)).sum(), (w * (kls + 1) * 4).sum(),
                            w.sum()]).detach() * (e + 8 * U)
    return (loss.detach(), stats.detach(), lp.detach(), grad, keep, loss_err, stat_err, g_row,
            row_err * (e + 8 * U))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("S,T,V,per_token,kl,reduction,with_old", [
    (1, 1, 2, False, 0.0, "token", True), (3, 9, 7, True, 0.1, "sequence", True),
    (8, 33, 65, False, 0.05, "token", True), (5, 17, 1003, True, 0.0, "sequence", False),
    (3, 2, 50257, False, 0.02, "sequence", True),
])
def test_policy_loss(S, T, V, per_token, kl, reduction, with_old, layout, dtype):
    x, t, cu, spans = batch(S, T, V, dtype, layout, seed=S + T)
    if cu is not None and not per_token and t.numel() == S:
        per_token = True  # as many rows as sequences: a 1-D tensor is one per token
    old, ref, adv = _policy_inputs(x, t, spans, per_token, kl, seed=7)
    old = old if with_old else None
    x = x.detach().requires_grad_(True)
    kw = dict(clip=CLIPS[0], clip_high=CLIPS[1], kl_coef=kl, reduction=reduction, cu_seqlens=cu)
    loss, logps, stats = ops.policy_loss(x, t, adv, old, ref, **kw)
    (got,) = torch.autograd.grad(loss, x, torch.tensor(0.5, device="cuda"))
    (w_loss, w_stats, lp, gx, keep, loss_err, stat_err, g_row, g_err) = _policy_exact(
        x, t, spans, adv, old, ref, kl, reduction)
    assert_within(loss, w_loss, loss_err + 1e-30, "loss")
    assert_within(stats, w_stats, stat_err + 1e-30, "statistics")
    lp = lp.view(t.shape)
    assert_within(logps, lp, torch.where(keep.view(t.shape), rel(V) + lp.abs() * 2 * U, 0.0),
                  "logps")
    shown = keep.view(t.shape)[..., None]
    tt = torch.where(keep.view(t.shape), t, -1)
    check_grad(got, torch.where(shown, gx, 0.0) * 0.5, x, tt, g_row * 0.5, g_err * 0.5)
    one, grad, logps1, stats1 = ops.policy_loss_and_grad(x, t, adv, old, ref, grad_scale=2.0,
                                                         **kw)
    assert not grad.requires_grad
    check_grad(grad, torch.where(shown, gx, 0.0) * 2, x, tt, g_row * 2, g_err * 2)
    # (the two forms may give a row to different numbers of threads: not the same bits)
    assert_within(one, w_loss, loss_err + 1e-30, "loss, one pass")
    assert_within(stats1, w_stats, stat_err + 1e-30, "statistics, one pass")
    assert_within(logps1, lp, torch.where(keep.view(t.shape), rel(V) + lp.abs() * 2 * U, 0.0),
                  "logps, one pass")


@pytest.mark.gpu
def test_target_past_the_vocabulary_is_nan_in_its_own_row():
    x, t, _, _ = batch(2, 4, 65, torch.float32, "plain", masked=0.0)
    t[1, 2] = 65
    x.requires_grad_(True)
    lp = ops.token_log_probs(x, t)
    (g,) = torch.autograd.grad(lp, x, torch.ones_like(lp))
    bad = torch.zeros(2, 4, dtype=torch.bool, device="cuda")
    bad[1, 2] = True
    assert torch.equal(lp.isnan(), bad)
    assert torch.equal(g.isnan(), bad[..., None].expand(g.shape))
    loss, grad, logps, _ = ops.policy_loss_and_grad(x, t, torch.ones(2, device="cuda"))
    assert loss.isnan() and torch.equal(logps.isnan(), bad)
    assert torch.equal(grad.isnan(), bad[..., None].expand(g.shape))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [40, 1000, 20_000])
def test_target_far_past_the_vocabulary(V):
    """Targets whose low 32 bits lie inside: their rows are NaN, nothing else is written."""
    far = [2**31, 2**31 + 8, 2**32, 2**32 + 5, 2**32 + V - 1, 2**40 + 33, 2**63 - 1]
    t = torch.tensor([3] + [k for f in far for k in (f, 3)], device="cuda")
    inside = t < V
    gen = torch.Generator("cuda").manual_seed(5)
    x = torch.randn(t.numel(), V, device="cuda", generator=gen).bfloat16().requires_grad_()

    def both(t):
        lp = ops.token_log_probs(x, t)
        return lp.detach(), torch.autograd.grad(lp, x, torch.ones_like(lp))[0]

    for got, want in zip(both(t), both(torch.where(inside, t, -1))):
        assert torch.equal(got[inside], want[inside])
        assert got[~inside].isnan().all()
    cu = torch.tensor([0, t.numel()], device="cuda")
    grad = ops.policy_loss_and_grad(x, t, torch.ones(t.numel(), device="cuda"), cu_seqlens=cu)[1]
    assert grad[inside].isfinite().all() and grad[~inside].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [33, 5003, 40001])
def test_rows_without_a_softmax_are_nan(V, dtype):
    """All -inf, a +inf, a NaN: log_softmax has no value there either."""
    x, t, _, _ = batch(1, 4, V, dtype, "plain", masked=0.0)
    x[0, 0], x[0, 1, 5], x[0, 2, V // 2] = -math.inf, math.inf, math.nan
    x.requires_grad_(True)
    lp = ops.token_log_probs(x, t)
    (g,) = torch.autograd.grad(lp, x, torch.zeros_like(lp))
    assert lp[0, :3].isnan().all() and lp[0, 3].isfinite()
    assert g[0, :3].isnan().any(-1).all() and torch.count_nonzero(g[0, 3]) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [50, 5003])
@pytest.mark.parametrize("shift", [-1e30, -60000.0, -3000.0, 2500.0, 2900.0, 70000.0, 1e30])
def test_logits_far_from_zero(shift, V, dtype):
    """Rows whose maximum lies where the sum takes its other form, and rows of the type's
    lowest value alone, which are uniform.  x and m are exact; their difference is rounded."""
    x, t, _, spans = batch(1, 6, V, dtype, "plain", masked=0.0)
    x = (x.float() * max(1.0, abs(shift) * 2.0**-6) + shift).to(dtype)
    x[0, 5] = torch.finfo(dtype).min
    x.requires_grad_(True)
    lp = ops.token_log_probs(x, t)
    x64, want, _ = exact_logps(x, t, spans)
    want = want.view(t.shape)
    assert_within(lp, want, rel(V) + want.detach().abs() * 2 * U, "logp")
    (g,) = torch.autograd.grad(lp, x, torch.ones_like(lp))
    (gx,) = torch.autograd.grad(want, x64, torch.ones_like(want))
    check_grad(g, gx, x, t, torch.ones_like(want), torch.zeros_like(want))


@pytest.mark.gpu
def test_more_dimensions_and_tokens_cut_from_a_longer_batch():
    x, t, _, spans = batch(6, 7, 65, torch.bfloat16, "plain")
    four = x.view(2, 3, 7, 65).detach().requires_grad_(True)
    lp = ops.token_log_probs(four, t.view(2, 3, 7))
    assert torch.equal(lp.view(6, 7), ops.token_log_probs(x, t))
    (g,) = torch.autograd.grad(lp.sum(), four)
    long = torch.zeros(6, 400, 65, dtype=torch.bfloat16, device="cuda")
    long[:, -7:] = x
    cut = long[:, -7:].detach().requires_grad_(True)
    (g2,) = torch.autograd.grad(ops.token_log_probs(cut, t).sum(), cut)
    assert torch.equal(g.view(6, 7, 65), g2)
    # no memory for the tokens that are not there, and rows at the logits' phase
    assert g2.untyped_storage().nbytes() < 4 * x.numel() * 2
    assert all((g2[i, j].data_ptr() - cut[i, j].data_ptr()) % 16 == 0
               for i in range(6) for j in range(7))
    _, g3, _, _ = ops.policy_loss_and_grad(cut, t, torch.ones(6, device="cuda"))
    leaf = x.detach().requires_grad_(True)
    _, g4, _, _ = ops.policy_loss_and_grad(leaf, t, torch.ones(6, device="cuda"))
    assert torch.equal(g3, g4)


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    x, t, _, _ = batch(2, 3, 9, torch.float32, "plain")
    x.requires_grad_(True)
    for loss in (ops.token_log_probs(x, t).sum(), ops.preference_loss(x, t)[0],
                 ops.policy_loss(x, t, torch.ones(2, device="cuda"))[0]):
        (g,) = torch.autograd.grad(loss, x, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), x)


@pytest.mark.gpu
def test_target_without_probability():
    """A -inf target: log-probability -inf, loss +inf, and a finite gradient."""
    x, t, _, _ = batch(2, 3, 9, torch.float32, "plain", masked=0.0)
    x[0, 1, t[0, 1]] = -math.inf
    x.requires_grad_(True)
    loss, chosen, _ = ops.preference_loss(x, t)
    (g,) = torch.autograd.grad(loss, x)
    assert float(loss) == math.inf and float(chosen[0]) == -math.inf
    assert g.isfinite().all() and float(g[0, 1, t[0, 1]]) == pytest.approx(-0.1, rel=1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [3, 3000])
def test_no_row_waits_for_weights(V):
    """A batch of nothing but left-out rows: its kernel has nothing to wait for, and what the
    memory of the weights held before does not show in the sums."""
    N = 30_000
    x = torch.zeros(N, V, device="cuda")
    t, adv = torch.full((N,), -1, device="cuda"), torch.ones(N, device="cuda")
    cu = torch.tensor([0, N // 3, N], device="cuda")
    for _ in range(10):
        old = [torch.full((n,), math.nan, device="cuda") for n in (N, 8 * N + 66, 9 * N)]
        del old
        loss, logps, stats = ops.policy_loss(x, t, adv, cu_seqlens=cu)
        assert not loss and not stats.any() and not logps.any()
        loss, grad, logps, stats = ops.policy_loss_and_grad(x, t, adv, cu_seqlens=cu)
        assert not loss and not stats.any() and not grad.any()


@pytest.mark.gpu
def test_empty_sequences_and_batches():
    x = torch.randn(5, 11, device="cuda", requires_grad=True)
    t = torch.randint(0, 11, (5,), device="cuda")
    cu = torch.tensor([0, 0, 5, 5, 5], device="cuda")  # 2 pairs: (0, 5 rows), (0, 0)
    loss, chosen, rejected = ops.preference_loss(x, t, cu_seqlens=cu)
    assert float(chosen[0]) == 0.0 and torch.count_nonzero(rejected) == 0
    x64, lp, _ = exact_logps(x, t, [(0, 5)])
    r = torch.tensor([0.0, float(lp.sum()), 0.0, 0.0], dtype=torch.float64)
    z = 0.1 * (r[:2] - r[2:])
    want = torch.nn.functional.softplus(-z).mean()
    assert float(loss) == pytest.approx(float(want), rel=1e-6)
    empty = torch.empty(4, 0, 7, device="cuda", requires_grad=True)
    none = torch.empty(4, 0, dtype=torch.int64, device="cuda")
    loss, _, _ = ops.preference_loss(empty, none, torch.tensor([1., 0, 0, 0], device="cuda"))
    want = (math.log1p(math.exp(0.1)) + math.log(2)) / 2
    assert float(loss) == pytest.approx(want, rel=1e-6)
    assert torch.autograd.grad(loss, empty)[0].shape == empty.shape
    loss, logps, stats = ops.policy_loss(empty, none, torch.ones(4, device="cuda"))
    assert float(loss) == 0.0 and logps.shape == (4, 0) and torch.count_nonzero(stats) == 0
    loss, grad, _, _ = ops.policy_loss_and_grad(empty, none, torch.ones(4, device="cuda"))
    assert grad.shape == empty.shape and ops.token_log_probs(empty, none).shape == (4, 0)


@pytest.mark.gpu
def test_gradients_against_differences():
    """Central differences of the kernels' own losses along a direction; how far they may be
    from the gradient is what the 64-bit loss's differences are, and the rounding of both
    fp32 losses over the step."""
    x, t, _, spans = batch(4, 12, 65, torch.float32, "plain", seed=3)
    old, ref, adv = _policy_inputs(x, t, spans, False, 0.1, seed=3)
    d = torch.randn(x.shape, generator=torch.Generator().manual_seed(9)).cuda()
    h = 2.0**-6
    kw = dict(clip=CLIPS[0], clip_high=CLIPS[1], kl_coef=0.1)

    def exact_pref(v):
        return float(_preference_exact(v, t, spans, None, 0.1, 0.0)[0])

    def exact_policy(v):
        return float(_policy_exact(v, t, spans, adv, old, ref, 0.1, "token")[0])

    for mine, exact in ((lambda v: ops.preference_loss(v, t)[0], exact_pref),
                        (lambda v: ops.policy_loss(v, t, adv, old, ref, **kw)[0], exact_policy)):
        leaf = x.clone().requires_grad_(True)
        (g,) = torch.autograd.grad(mine(leaf), leaf)
        slope = float((g.double() * d.double()).sum())
        up, down = x + h * d, x - h * d
        diff = (float(mine(up)) - float(mine(down))) / (2 * h)
        # the same differences in 64 bits against the slope there: the curvature (the slope is
        # itself a difference, over 2^-16: its own curvature is 2^-20 of the first one's)
        e64 = (exact(up) - exact(down)) / (2 * h)
        tiny = 2.0**-16
        x64 = x.double()
        s64 = (exact(x64 + tiny * d) - exact(x64 - tiny * d)) / (2 * tiny)
        loss_off = 12 * 2 * rel(65) + abs(exact(x)) * 2 * U
        assert abs(diff - slope) <= abs(e64 - s64) + loss_off / h + 1e-5 * abs(s64) + 1e-7


@pytest.mark.gpu
def test_same_bits_twice_and_on_two_streams():
    x, t, _, _ = batch(6, 40, 1003, torch.bfloat16, "plain", seed=2)
    x2, t2, _, _ = batch(6, 40, 1003, torch.bfloat16, "plain", seed=4)

    def step(x, t):
        x = x.detach().requires_grad_(True)
        loss, a, b = ops.preference_loss(x, t)
        (g,) = torch.autograd.grad(loss, x)
        return [loss, a, b, g, *ops.policy_loss_and_grad(x, t, torch.ones(6, device="cuda"))]

    first, second = step(x, t), step(x2, t2)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(5):
        for s, args in zip(streams, ((x, t), (x2, t2))):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(step(*args))
    torch.cuda.synchronize()
    for i, v in enumerate(got):
        for a, b in zip(v, (first, second)[i % 2]):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_captured_and_replayed_on_new_inputs():
    x, t, cu, _ = batch(4, 20, 130, torch.bfloat16, "packed", seed=2)
    x2, _, _, _ = batch(4, 20, 130, torch.bfloat16, "packed", seed=2)
    x2 = x2 * 0.5
    leaf = x.clone().requires_grad_(True)
    adv = torch.randn(4, device="cuda")

    def step(v):
        loss, _, _ = ops.preference_loss(v, t, cu_seqlens=cu)
        (g,) = torch.autograd.grad(loss, v)
        return [loss, g, *ops.policy_loss_and_grad(v, t, adv, cu_seqlens=cu)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(leaf)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(leaf)
    for v in (x2, x):
        with torch.no_grad():
            leaf.copy_(v)
        graph.replay()
        want = step(v.clone().requires_grad_(True))
        for a, b in zip(out, want):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_more_logits_than_32_bits_count():
    """Rows behind 2**31 logits, and rows that lie that far apart."""
    V, n = 32_768, 6
    N = 2**31 // V + 100
    x = torch.empty(N, V, device="cuda", dtype=torch.bfloat16).normal_(
        generator=torch.Generator("cuda").manual_seed(4))
    t = torch.full((N,), -1, device="cuda")
    t[-n:] = torch.arange(n, device="cuda") * 5000
    adv = torch.linspace(-1, 2, N, device="cuda")
    old = torch.linspace(-10, -11, N, device="cuda")

    def everything(x, t, adv, old):
        x = x.detach().requires_grad_()
        cu = torch.tensor([0, t.numel() - n // 2, t.numel()], device="cuda")
        got = []
        for loss, *others in (ops.preference_loss(x, t, cu_seqlens=cu),
                              ops.policy_loss(x, t, adv, old, cu_seqlens=cu),
                              (ops.token_log_probs(x, t),)):
            got += [loss.detach(), *others]
            got.append(torch.autograd.grad(loss, x, torch.ones_like(loss))[0][-n:])
        loss, grad, logps, stats = ops.policy_loss_and_grad(x, t, adv, old, cu_seqlens=cu)
        assert not grad[: -n].any()
        return got + [loss, grad[-n:], logps[-n:], stats]

    def same(a, b):
        for p, q in zip(a, b):
            if p.dim() == 1 and p.numel() == N:
                p = p[-n:]
            assert torch.equal(p, q)

    few = everything(x[-n:].clone(), t[-n:], adv[-n:], old[-n:])
    same(everything(x, t, adv, old), few)
    apart = x.flatten().as_strided((n, V), ((N - 1) // (n - 1) * V, 1))
    apart.copy_(x[-n:].clone())
    same(everything(apart, t[-n:], adv[-n:], old[-n:]), few)


@pytest.mark.gpu
def test_retained_graph_and_compile():
    x, t, _, _ = batch(2, 6, 65, torch.float32, "plain", masked=0.1)
    x.requires_grad_(True)
    loss, _, _ = ops.preference_loss(x, t)
    (a,) = torch.autograd.grad(loss, x, retain_graph=True)
    (b,) = torch.autograd.grad(loss, x)
    assert torch.equal(a, b)

    def f(x):
        loss, _, _ = ops.preference_loss(x, t)
        return loss + ops.policy_loss(x, t, torch.ones(2, device="cuda"))[0]

    (want,) = torch.autograd.grad(f(x), x)
    compiled = torch.compile(f, backend="aot_eager", fullgraph=True)
    (got,) = torch.autograd.grad(compiled(x), x)
    assert torch.equal(got, want)
