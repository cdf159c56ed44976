"""Measured cases of the post-training operators: preference loss, clipped policy loss,
global gradient norm and clipping, and the gated residual step between two norms.

``run`` computes one pass either in its plain form (elementary torch operations, the
definition written out) or, where ``own`` is true, by the calls a training program makes
of ``llm_training_b200.ops``.  ``exact`` is the definition in 64 bits, differentiated by
autograd where the operator has a gradient.
"""

import random

import torch

own = False

GRAD_EPS = 1e-6  # the clip factor's: max_norm / (norm + 1e-6), at most 1


# ---- cases ----------------------------------------------------------------------


def listed():
    return [
        # one pair of short answers of a character-level model: all latency
        dict(name="preference, one short pair", op="preference", pairs=1, T=40, V=97,
             dtype="float32", packed=False, ref=True, smooth=0.0, kept=0.6),
        # answers of different lengths back to back, the unpadded GPT-2 vocabulary
        dict(name="preference, packed, odd vocab", op="preference", pairs=6, T=509, V=50257,
             dtype="bfloat16", packed=True, ref=True, smooth=0.1, kept=0.7),
        # a full padded batch of pairs, the padded GPT-2 vocabulary
        dict(name="preference, padded batch", op="preference", pairs=8, T=512, V=50304,
             dtype="bfloat16", packed=False, ref=True, smooth=0.0, kept=0.8),
        # a few short samples with one advantage each, no KL term
        dict(name="policy, short samples", op="policy", seqs=4, T=33, V=1000, dtype="float32",
             packed=False, per_token=False, kl=0.0, reduction="token", fused=False, kept=0.7),
        # packed samples with per-token advantages and a KL term, through autograd
        dict(name="policy, packed, KL", op="policy", seqs=9, T=257, V=50257, dtype="bfloat16",
             packed=True, per_token=True, kl=0.05, reduction="token", fused=False, kept=0.8),
        # a group of samples per prompt, mean over samples, loss and gradient in one call
        dict(name="policy, group, one call", op="policy", seqs=16, T=512, V=50304,
             dtype="bfloat16", packed=False, per_token=False, kl=0.02, reduction="sequence",
             fused=True, kept=0.85),
        # the gradients of a two-layer test model, below the bound: nothing to scale
        dict(name="clip, tiny model, in place", op="clip", layers=2, C=32, V=97, ctx=64,
             bias=False, dtype="float32", out="", bounded=False),
        # GPT-2 small's fp32 gradients, clipped into the optimizer's buffer
        dict(name="clip, GPT-2 small", op="clip", layers=12, C=768, V=50257, ctx=1024,
             bias=False, dtype="float32", out="float32", bounded=True),
        # GPT-2 medium's bf16 gradients, clipped and cast to fp32
        dict(name="clip, GPT-2 medium, bf16", op="clip", layers=24, C=1024, V=50257, ctx=8192,
             bias=False, dtype="bfloat16", out="float32", bounded=True),
        # a handful of tokens: all latency
        dict(name="residual, few tokens", op="residual", B=1, T=5, C=768, kind="layer",
             post=True, gate="channel", bias=True, x="float32", h="bfloat16", y="bfloat16"),
        # GPT-2 small's stream at its training batch
        dict(name="residual, GPT-2 small", op="residual", B=16, T=1024, C=768, kind="layer",
             post=True, gate="channel", bias=False, x="float32", h="bfloat16", y="bfloat16"),
        # RMS norms, a gate for each sample, an odd width, a bf16 stream
        dict(name="residual, odd width, per sample", op="residual", B=6, T=1501, C=1999,
             kind="rms", post=True, gate="sample", bias=False, x="bfloat16", h="bfloat16",
             y="bfloat16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["preference", "policy", "clip", "residual"])
    dtype = rng.choice(["float32", "bfloat16"])
    if op in ("preference", "policy"):
        V = _log_int(rng, 60, 60000)
        T = _log_int(rng, 3, 1100)
        room = (7_000 * 50_000 if dtype == "bfloat16" else 3_500 * 50_000) // (V * T)
        kept = round(rng.uniform(0.3, 1.0), 2)
        packed = rng.random() < 0.5
        if op == "preference":
            return dict(op=op, pairs=_log_int(rng, 1, max(1, min(24, room // 2))), T=T, V=V,
                        dtype=dtype, packed=packed, ref=rng.random() < 0.7,
                        smooth=rng.choice([0.0, 0.1]), kept=kept)
        return dict(op=op, seqs=_log_int(rng, 1, max(1, min(48, room))), T=T, V=V, dtype=dtype,
                    packed=packed, per_token=rng.random() < 0.5,
                    kl=rng.choice([0.0, 0.04]), reduction=rng.choice(["token", "sequence"]),
                    fused=rng.random() < 0.5, kept=kept)
    if op == "clip":
        out = rng.choice(["", dtype, "float32"])
        return dict(op=op, layers=_log_int(rng, 1, 20), C=_log_int(rng, 16, 900),
                    V=_log_int(rng, 60, 50000), ctx=_log_int(rng, 16, 4096),
                    bias=rng.random() < 0.5, dtype=dtype, out=out, bounded=bool(out))
    C = _log_int(rng, 30, 4096)
    rows = _log_int(rng, 1, max(2, 12_000_000 // C))
    B = _log_int(rng, 1, min(rows, 32))
    return dict(op=op, B=B, T=max(1, rows // B), C=C, kind=rng.choice(["layer", "rms"]),
                post=rng.random() < 0.8, gate=rng.choice(["", "channel", "sample"]),
                bias=rng.random() < 0.5, x=rng.choice(["float32", "bfloat16"]), h=dtype,
                y=rng.choice(["float32", "bfloat16"]))


# ---- what a case holds ------------------------------------------------------------


def _lengths(case, n):
    """Answer lengths: each between a third of T and T (the longest has T)."""
    r = random.Random(f"{case['T']},{n}")
    T = case["T"]
    got = [max(1, round(T * r.uniform(0.33, 1.0))) for _ in range(n)]
    got[r.randrange(n)] = T
    return got


def _counted(case, n):
    """(first, last + 1) counted token of each sequence: the prompt comes first."""
    return [(min(k - 1, int(k * (1 - case["kept"]))), k) for k in _lengths(case, n)]


def _shapes(case):
    C, bias, got = case["C"], case["bias"], [(case["V"], case["C"]), (case["ctx"], case["C"])]
    block = [(C,), (C, C), (C, C), (C, C), (C, C), (C,), (4 * C, C), (C, 4 * C)]
    block += [(C,)] * 6 + [(4 * C,), (C,)] if bias else []
    return got + block * case["layers"] + [(C,)] * (2 if bias else 1)


def _numels(case):
    return [s[0] * (s[1] if len(s) > 1 else 1) for s in _shapes(case)]


def work(case):
    elt = {"float32": 4, "bfloat16": 2}
    if case["op"] in ("preference", "policy"):
        n = 2 * case["pairs"] if case["op"] == "preference" else case["seqs"]
        counted = sum(b - a for a, b in _counted(case, n))
        rows = sum(_lengths(case, n)) if case["packed"] else n * case["T"]
        e = elt[case["dtype"]]
        # counted rows of logits in, every row of the gradient out
        return {"bytes": (counted + rows) * case["V"] * e + rows * 24,
                "flops": 8 * counted * case["V"]}
    if case["op"] == "clip":
        n = sum(_numels(case))
        return {"bytes": n * (elt[case["dtype"]] + (elt[case["out"]] if case["out"] else 0)),
                "flops": 3 * n}
    n = case["B"] * case["T"] * case["C"]
    x, h, y = elt[case["x"]], elt[case["h"]], elt[case["y"]]
    # inputs (x, h, both upstream gradients) and outputs (sum, norm, both gradients)
    return {"bytes": n * 2 * (2 * x + h + y), "flops": 40 * n}


# ---- inputs -------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _answers(case, n, g):
    """Logits of n answers (a peak on most targets, as a trained model has), targets with the
    prompt and the padding left out, and each token's log-probability."""
    dtype = getattr(torch, case["dtype"])
    lens, counted, V = _lengths(case, n), _counted(case, n), case["V"]
    if case["packed"]:
        starts = [sum(lens[:i]) for i in range(n)]
        rows = sum(lens)
        cu = torch.tensor(starts + [rows], device="cuda")
    else:
        starts = [i * case["T"] for i in range(n)]
        rows, cu = n * case["T"], None
    logits = torch.randn(rows, V, device="cuda", dtype=dtype, generator=g).mul_(2)
    targets = torch.randint(0, V, (rows,), device="cuda", generator=g)
    peak = 9 * torch.rand(rows, 1, device="cuda", generator=g)
    logits.scatter_add_(1, targets[:, None], peak.to(dtype))
    keep = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for at, (a, b) in zip(starts, counted):
        keep[at + a:at + b] = True
    logp = torch.empty(rows, device="cuda", dtype=torch.float64)
    for a in range(0, rows, 1024):
        x = logits[a:a + 1024].float()
        logp[a:a + 1024] = (x.gather(1, targets[a:a + 1024, None])[:, 0].double()
                            - torch.logsumexp(x, 1).double())
    targets = torch.where(keep, targets, -100)
    logp = torch.where(keep, logp, 0.0)
    if not case["packed"]:
        logits, targets = logits.view(n, case["T"], V), targets.view(n, case["T"])
    return logits, targets, cu, logp


def _by_sequence(values, n, cu):
    """Sums of a float64 (rows,) over each of the n sequences."""
    if cu is None:
        return values.view(n, -1).sum(1)
    run_sum = torch.cat([values.new_zeros(1), values.cumsum(0)])
    return run_sum[cu[1:]] - run_sum[cu[:-1]]


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case=case)
    if case["op"] == "preference":
        n = 2 * case["pairs"]
        s["logits"], s["targets"], s["cu"], logp = _answers(case, n, g)
        sums = _by_sequence(logp, n, s["cu"])
        # the reference model's sums: near this model's
        off = 6 * torch.randn(n, device="cuda", generator=g)
        s["ref"] = (sums + off).float() if case["ref"] else None
        s["logits"].requires_grad_(True)
    elif case["op"] == "policy":
        n = case["seqs"]
        s["logits"], s["targets"], s["cu"], logp = _answers(case, n, g)
        shape = s["targets"].shape
        old = logp + 0.15 * torch.randn(logp.shape, device="cuda", generator=g)
        # on the clip's border the loss has two one-sided gradients: keep off it
        ratio = (logp - old).exp()
        edge = ((ratio - 0.8).abs() < 1e-3) | ((ratio - 1.25).abs() < 1e-3)
        s["old"] = torch.where(edge, old - 0.01, old).float().view(shape)
        ref = logp + 0.3 * torch.randn(logp.shape, device="cuda", generator=g)
        s["ref"] = ref.float().view(shape) if case["kl"] else None
        # mostly above the baseline, so that the loss is no difference of near-equal sums
        s["adv"] = 0.8 + 0.6 * torch.randn(shape if case["per_token"] else n, device="cuda",
                                           generator=g)
        s["logits"].requires_grad_(True)
    elif case["op"] == "clip":
        sizes = _numels(case)
        dtype = getattr(torch, case["dtype"])
        # gradients as views of one bucket, as data parallel training keeps them
        s["flat"] = torch.randn(sum(sizes), device="cuda", dtype=dtype, generator=g).mul_(1e-2)
        s["grads"] = [v.view(k) for v, k in zip(s["flat"].split(sizes), _shapes(case))]
        if case["out"]:
            s["flat_out"] = torch.empty(sum(sizes), device="cuda",
                                        dtype=getattr(torch, case["out"]))
            s["out"] = [v.view(k) for v, k in zip(s["flat_out"].split(sizes), _shapes(case))]
        s["max_norm"] = 1e-2 * sum(sizes) ** 0.5 * (0.37 if case["bounded"] else 1.5)
        if not case["out"]:
            s["params"] = [torch.nn.Parameter(torch.empty_like(v)) for v in s["grads"]]
            for p, v in zip(s["params"], s["grads"]):
                p.grad = v
    else:
        B, T, C = case["B"], case["T"], case["C"]

        def normal(*shape, dtype="float32", mean=0.0, std=1.0):
            v = torch.randn(*shape, device="cuda", generator=g) * std + mean
            return v.to(getattr(torch, dtype))

        s["x"] = normal(B, T, C, dtype=case["x"], std=3.0, mean=0.2)
        s["h"] = normal(B, T, C, dtype=case["h"], std=0.5, mean=-0.1)
        s["w"] = normal(C, mean=1.0, std=0.1)
        s["wp"] = normal(C, mean=1.0, std=0.1) if case["post"] else None
        s["b"] = normal(C, std=0.1) if case["bias"] else None
        s["bp"] = normal(C, std=0.1) if case["bias"] and case["post"] else None
        shape = {"": None, "channel": (C,), "sample": (B, 1, C)}[case["gate"]]
        s["gate"] = normal(*shape, mean=0.3, std=0.2) if shape else None
        s["leaves"] = [k for k in ("x", "h", "w", "b", "wp", "bp", "gate") if s[k] is not None]
        for k in s["leaves"]:
            s[k].requires_grad_(True)
        s["dxo"] = normal(B, T, C, dtype=case["x"])
        s["dy"] = normal(B, T, C, dtype=case["y"])
    return s


SCALE = 0.7071  # the residual cases' scale on the block's output
EPS = 1e-5
BETA = 0.1
CLIP = (0.2, 0.25)


# ---- the framework's calls ------------------------------------------------------------


def _own(s):
    from llm_training_b200 import ops

    case = s["case"]
    if case["op"] == "preference":
        loss, chosen, rejected = ops.preference_loss(
            s["logits"], s["targets"], s["ref"], beta=BETA, label_smoothing=case["smooth"],
            cu_seqlens=s["cu"])
        (grad,) = torch.autograd.grad(loss, s["logits"])
        return dict(loss=loss, chosen=chosen, rejected=rejected, grad=grad)
    if case["op"] == "policy":
        args = (s["logits"], s["targets"], s["adv"], s["old"], s["ref"])
        kw = dict(clip=CLIP[0], clip_high=CLIP[1], kl_coef=case["kl"],
                  reduction=case["reduction"], cu_seqlens=s["cu"])
        if case["fused"]:
            loss, grad, logps, _ = ops.policy_loss_and_grad(*args, **kw)
        else:
            loss, logps, _ = ops.policy_loss(*args, **kw)
            (grad,) = torch.autograd.grad(loss, s["logits"])
        return dict(loss=loss, logps=logps, grad=grad)
    if case["op"] == "clip":
        if case["out"]:
            _, norm = ops.clip_grads(s["grads"], s["max_norm"], out=s["out"])
            return dict(norm=norm, grads=s["flat_out"])
        norm = ops.clip_grad_norm_(s["params"], s["max_norm"])
        return dict(norm=norm, grads=s["flat"])
    xo, y = ops.residual_norm(s["x"], s["h"], s["w"], s["b"], post_weight=s["wp"],
                              post_bias=s["bp"], gate=s["gate"], scale=SCALE, eps=EPS,
                              kind=case["kind"], out_dtype=s["dy"].dtype)
    grads = torch.autograd.grad((xo, y), [s[k] for k in s["leaves"]], (s["dxo"], s["dy"]))
    return dict(sum=xo, norm=y, **{"d" + k: v for k, v in zip(s["leaves"], grads)})


# ---- the plain form ---------------------------------------------------------------------


def _rows(s):
    """exp(x - max), its sum, and the log-probability (in 64 bits) of each row's target."""
    x = s["logits"].detach().reshape(-1, s["case"]["V"]).float()
    t = s["targets"].reshape(-1)
    top = x.max(1, keepdim=True).values
    picked = (x.gather(1, t.clamp_min(0)[:, None]) - top)[:, 0].double()
    e = (x - top).exp_()
    total = e.sum(1)
    logp = torch.where(t >= 0, picked - total.double().log(), 0.0)
    return e, total, logp, t


def _logits_grad(s, e, total, t, coef):
    """coef (rows,) * ([column is the target] - softmax), in the logits' type and shape."""
    grad = e.mul_((-coef / total)[:, None])
    grad.scatter_add_(1, t.clamp_min(0)[:, None], coef[:, None])
    return grad.to(s["logits"].dtype).view(s["logits"].shape)


def _row_sequence(s):
    """The sequence each row belongs to."""
    if s["cu"] is None:
        n, T = s["targets"].shape
        return torch.arange(n, device=s["targets"].device).repeat_interleave(T)
    rows = torch.arange(s["targets"].numel(), device=s["cu"].device)
    return (rows[:, None] >= s["cu"][None, 1:]).sum(1)


def _softplus(z):
    return z.clamp_min(0) + (1 + (-z.abs()).exp()).log()


def _plain_preference(s):
    case = s["case"]
    P, n = case["pairs"], 2 * case["pairs"]
    e, total, logp, t = _rows(s)
    ratio = _by_sequence(logp, n, s["cu"])
    if s["ref"] is not None:
        ratio = ratio - s["ref"].double()
    z = BETA * (ratio[:P] - ratio[P:])
    a = case["smooth"]
    loss = ((1 - a) * _softplus(-z) + a * _softplus(z)).sum() / P
    dz = (a / (1 + (-z).exp()) - (1 - a) / (1 + z.exp())) * BETA / P
    coef = torch.where(t >= 0, torch.cat([dz, -dz])[_row_sequence(s)], 0.0).float()
    return dict(loss=loss.float(), chosen=(BETA * ratio[:P]).float(),
                rejected=(BETA * ratio[P:]).float(), grad=_logits_grad(s, e, total, t, coef))


def _plain_policy(s):
    case = s["case"]
    e, total, logp, t = _rows(s)
    keep = t >= 0
    count = keep.double()
    if case["reduction"] == "token":
        weight = count / count.sum().clamp_min(1)
    else:
        per = _by_sequence(count, case["seqs"], s["cu"])
        share = 1 / (per.clamp_min(1) * (per > 0).sum().clamp_min(1))
        weight = count * share[_row_sequence(s)]
    adv = s["adv"].double().reshape(-1)
    if not case["per_token"]:
        adv = adv[_row_sequence(s)]
    ratio = (logp - s["old"].reshape(-1).double()).exp()
    free = ratio * adv
    held = ratio.clamp(1 - CLIP[0], 1 + CLIP[1]) * adv
    each = -torch.minimum(free, held)
    slope = torch.where(free <= held, -free, 0.0)
    if case["kl"]:
        d = s["ref"].reshape(-1).double() - logp
        each = each + case["kl"] * (d.exp() - d - 1)
        slope = slope + case["kl"] * (1 - d.exp())
    loss = torch.where(keep, each * weight, 0.0).sum()
    coef = torch.where(keep, slope * weight, 0.0).float()
    return dict(loss=loss.float(), logps=logp.float().view(s["targets"].shape),
                grad=_logits_grad(s, e, total, t, coef))


def _plain_clip(s):
    norm = torch.stack([v.double().square().sum() for v in s["grads"]]).sum().sqrt().float()
    factor = (s["max_norm"] / (norm + GRAD_EPS)).clamp_max(1.0)
    into = s["out"] if s["case"]["out"] else s["grads"]
    [o.copy_(v.float() * factor) for o, v in zip(into, s["grads"])]
    return dict(norm=norm, grads=s["flat_out"] if s["case"]["out"] else s["flat"])


def _normed(v, kind):
    """(v - mean) / sqrt(var + eps) over the last axis (mean 0 for an RMS norm), 1 / sqrt."""
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    rstd = (v.square().mean(-1, keepdim=True) + EPS).rsqrt()
    return v * rstd, rstd


def _normed_grad(d, hat, rstd, kind):
    d = d - hat * (d * hat).mean(-1, keepdim=True) - (
        d.mean(-1, keepdim=True) if kind == "layer" else 0.0)
    return d * rstd


def _plain_residual(s):
    kind = s["case"]["kind"]
    v = {k: s[k].detach().float() for k in s["leaves"]}
    n = h = v["h"]
    if "wp" in v:
        hat, rstd_h = _normed(h, kind)
        n = hat * v["wp"] + (v["bp"] if "bp" in v else 0.0)
    gate = SCALE * (v["gate"] if "gate" in v else torch.ones_like(v["w"]))
    xo = v["x"] + gate * n
    xo_hat, rstd = _normed(xo, kind)
    y = xo_hat * v["w"] + (v["b"] if "b" in v else 0.0)
    dy = s["dy"].float()
    dxo = s["dxo"].float() + _normed_grad(dy * v["w"], xo_hat, rstd, kind)
    dn = dxo * gate
    rows = (0, 1)
    got = dict(sum=xo.to(s["x"].dtype), norm=y.to(s["dy"].dtype), dx=dxo.to(s["x"].dtype),
               dw=(dy * xo_hat).sum(rows))
    if "b" in v:
        got["db"] = dy.sum(rows)
    if "gate" in v:
        each = dxo * n * SCALE
        got["dgate"] = each.sum(rows) if v["gate"].dim() == 1 else each.sum(1, keepdim=True)
    if "wp" in v:
        got["dwp"] = (dn * hat).sum(rows)
        if "bp" in v:
            got["dbp"] = dn.sum(rows)
        dn = _normed_grad(dn * v["wp"], hat, rstd_h, kind)
    return dict(got, dh=dn.to(s["h"].dtype))


def run(state):
    if own:
        return _own(state)
    plain = dict(preference=_plain_preference, policy=_plain_policy, clip=_plain_clip,
                 residual=_plain_residual)
    return plain[state["case"]["op"]](state)


# ---- the definition in 64 bits --------------------------------------------------------------


def _chunks(s):
    """Each sequence's (first row, last row + 1)."""
    if s["cu"] is not None:
        at = s["cu"].tolist()
        return list(zip(at[:-1], at[1:]))
    n, T = s["targets"].shape
    return [(i * T, (i + 1) * T) for i in range(n)]


def _exact_answers(s, loss_of):
    """loss_of(per-sequence lists of token log-probabilities) and its gradient: the softmax's
    chain rule a sequence at a time, everything above the log-probabilities by autograd."""
    V = s["case"]["V"]
    x, t = s["logits"].detach().reshape(-1, V), s["targets"].reshape(-1)
    parts = []
    for a, b in _chunks(s):
        lp = torch.log_softmax(x[a:b].double(), 1)
        keep = t[a:b] >= 0
        lp = lp[keep].gather(1, t[a:b][keep][:, None])[:, 0]
        parts.append(lp.requires_grad_(True))
    loss, more = loss_of(parts)
    slopes = torch.autograd.grad(loss, parts)
    grad = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for (a, b), slope in zip(_chunks(s), slopes):
        keep = t[a:b] >= 0
        per_row = torch.zeros(b - a, dtype=torch.float64, device=x.device)
        per_row[keep] = slope
        one_hot = torch.zeros(b - a, V, dtype=torch.float64, device=x.device)
        one_hot[keep, t[a:b][keep]] = 1.0
        grad[a:b] = per_row[:, None] * (one_hot - torch.softmax(x[a:b].double(), 1))
    return dict(loss=loss.detach(), grad=grad.view(s["logits"].shape), **more)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "preference":
        P = case["pairs"]

        def loss_of(parts):
            r = torch.stack([p.sum() for p in parts])
            if s["ref"] is not None:
                r = r - s["ref"].double()
            win = torch.sigmoid(BETA * (r[:P] - r[P:]))
            lose = torch.sigmoid(BETA * (r[P:] - r[:P]))
            loss = -((1 - case["smooth"]) * win.log() + case["smooth"] * lose.log()).mean()
            return loss, dict(chosen=BETA * r[:P].detach(), rejected=BETA * r[P:].detach())

        return _exact_answers(s, loss_of)
    if case["op"] == "policy":
        t = s["targets"].reshape(-1)

        def loss_of(parts):
            logps = torch.zeros(t.shape, dtype=torch.float64, device=t.device)
            losses = []
            for i, ((a, b), lp) in enumerate(zip(_chunks(s), parts)):
                keep = t[a:b] >= 0
                logps[a:b][keep] = lp.detach()
                adv = (s["adv"].reshape(-1)[a:b][keep] if case["per_token"]
                       else s["adv"][i]).double()
                ratio = torch.exp(lp - s["old"].reshape(-1)[a:b][keep].double())
                each = torch.where(adv >= 0, -adv * ratio.clamp(max=1 + CLIP[1]),
                                   -adv * ratio.clamp(min=1 - CLIP[0]))
                if case["kl"]:
                    gap = s["ref"].reshape(-1)[a:b][keep].double() - lp
                    each = each + case["kl"] * (torch.expm1(gap) - gap)
                losses.append(each)
            if case["reduction"] == "token":
                loss = torch.cat(losses).mean()
            else:
                loss = torch.stack([v.mean() for v in losses if v.numel()]).mean()
            return loss, dict(logps=logps.view(s["targets"].shape))

        return _exact_answers(s, loss_of)
    if case["op"] == "clip":
        norm = torch.linalg.vector_norm(s["flat"].double())
        over = float(norm) + GRAD_EPS > s["max_norm"]
        return dict(norm=norm, grads=s["flat"].double() * (
            s["max_norm"] / (norm + GRAD_EPS) if over else 1.0))
    F = torch.nn.functional
    v = {k: s[k].detach().double().requires_grad_(True) for k in s["leaves"]}
    C = (case["C"],)

    def norm_of(u, w, b):
        if case["kind"] == "layer":
            return F.layer_norm(u, C, w, b, EPS)
        u = F.rms_norm(u, C, w, EPS)
        return u if b is None else u + b

    n = norm_of(v["h"], v["wp"], v.get("bp")) if case["post"] else v["h"]
    xo = v["x"] + SCALE * (v["gate"] * n if "gate" in v else n)
    y = norm_of(xo, v["w"], v.get("b"))
    grads = torch.autograd.grad((xo, y), [v[k] for k in s["leaves"]],
                                (s["dxo"].double(), s["dy"].double()))
    return dict(sum=xo.detach(), norm=y.detach(),
                **{"d" + k: u for k, u in zip(s["leaves"], grads)})
