"""The residual step between two norms (csrc/sqb_residual_norm.cu) against its definition
in 64 bits, differentiated by autograd.

Bounds, u = 2^-24: a mean of C fp32 values summed in a tree of runs of at most 8 is off by
at most (8 + 10) u of the mean magnitude, a variance by twice that, 1/std by as much and
the two units of rsqrt; a normalised element is then off by at most 32 u (1 + |element|)
plus 2 u |value| / std of cancellation (|mean| is below 4 std here).  With the weights'
products, the sum and the second norm a forward value is off by at most k u of the largest
magnitude it is made of, k = 128; a gradient, which goes back through both, by k = 512.
Column sums over N rows add (N / CTAs + CTAs / 8 + 8) u of the sum of magnitudes.  Results
are then rounded to their type: half a step, finfo.eps / 2."""

import ctypes
import math

import pytest
import torch
import torch.nn.functional as F
from torch._subclasses.fake_tensor import FakeTensorMode

from llm_training_b200 import _lib, ops

U = 2.0**-24
F32, BF16 = torch.float32, torch.bfloat16
EPS = 1e-5


def test_refusals():
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.residual_norm(torch.zeros(2, 8), torch.zeros(2, 8), torch.ones(8))
    with FakeTensorMode():
        x, w = torch.empty(3, 4, 8, device="cuda"), torch.empty(8, device="cuda")
        wide = torch.empty(2, 4097, device="cuda")
        for kind, text, args, kw in [
            (TypeError, "float32 and bfloat16", (x.half(), x, w), {}),
            (TypeError, "float32 and bfloat16", (x, x.double(), w), {}),
            (TypeError, "float32 and bfloat16", (x, x, w), dict(out_dtype=torch.float16)),
            (ValueError, "one shape", (x, x[:2], w), {}),
            (ValueError, "columns", (wide, wide, wide[0]), {}),
            (ValueError, "kind", (x, x, w), dict(kind="batch")),
            (ValueError, "weight is needed", (x, x, None), {}),
            (ValueError, "weight", (x, x, w[:7]), {}),
            (ValueError, "post_weight", (x, x, w), dict(post_weight=w[:7])),
            (ValueError, "post_bias", (x, x, w), dict(post_bias=w)),
            (ValueError, "gate", (x, x, w), dict(gate=torch.empty(4, 8, device="cuda"))),
            (ValueError, "gate", (x, x, w), dict(gate=torch.empty(3, 4, 8, device="cuda"))),
            (ValueError, "gate", (x, x, w), dict(gate=w.double())),
            (ValueError, "scale", (x, x, w), dict(scale=math.nan)),
            (ValueError, "scale", (x, x, w), dict(scale=1e39)),
            (ValueError, "eps", (x, x, w), dict(eps=-1.0)),
        ]:
            with pytest.raises(kind, match=text):
                ops.residual_norm(*args, **kw)


def test_c_entry_points_reject_bad_arguments_without_a_device():
    lib, p = _lib.lib(), ctypes.c_void_p(256)

    def fwd(x=p, xt=0, yt=0, w=p, wp=p, bp=None, gate=None, gates=0, N=4, C=8, stats=p):
        return lib.sqb_residual_norm_fwd(x, xt, p, 0, w, None, wp, bp, gate, gates, 1.0, EPS, 0,
                                         p, p, yt, stats, N, C, None)

    assert fwd(x=None) == 1 and fwd(w=None) == 1 and fwd(N=0) == 1 and fwd(stats=None) == 1
    assert fwd(wp=None, bp=p) == 1 and fwd(gate=p, gates=3) == 1 and fwd(gate=p) == 1
    assert fwd(xt=5) == 2 and fwd(yt=5) == 2
    assert fwd(stats=ctypes.c_void_p(264)) == 3
    assert fwd(C=4097) == 4 and fwd(C=0) == 4 and fwd(C=1 << 40) == 4

    def bwd(dy=p, dw=p, wp=None, gates=0, gate=None, dgate=None, ws=p, ws_bytes=1 << 30, N=4):
        return lib.sqb_residual_norm_bwd(dy, 0, None, p, 0, p, 0, p, None, wp, None, gate, gates,
                                         1.0, EPS, 0, p, p, p, dw, None, None, None, dgate, ws,
                                         ws_bytes, N, 8, None)

    assert bwd(dy=None) == 1 and bwd(dw=None) == 1 and bwd(wp=p) == 1
    assert bwd(gate=p, gates=4) == 1 and bwd(ws=None) == 5 and bwd(ws_bytes=64) == 5
    assert bwd(gate=p, gates=65532, dgate=p, N=65532) == 4
    assert lib.sqb_residual_norm_workspace_bytes(4, 8, 4) > lib.sqb_residual_norm_workspace_bytes(
        4, 8, 0) > 0


def test_fakes():
    with FakeTensorMode():
        x = torch.empty(2, 3, 8, device="cuda", dtype=BF16)
        w, g = torch.empty(8, device="cuda"), torch.empty(2, 1, 8, device="cuda", dtype=BF16)
        for v in (x, w, g):
            v.requires_grad_(True)
        xo, y = ops.residual_norm(x, x, w, post_weight=w, gate=g, out_dtype=F32)
        assert xo.shape == y.shape == x.shape and xo.dtype == BF16 and y.dtype == F32


def inputs(shape, xt, ht, yt, gate, bias, post, seed=0, mean=0.3):
    g = torch.Generator().manual_seed(seed)
    C = shape[-1]

    def normal(*s, std=1.0, mean=0.0, dtype=F32):
        return (torch.randn(*s, generator=g) * std + mean).to(dtype).cuda()

    v = dict(x=normal(*shape, std=2.0, mean=mean, dtype=xt),
             h=normal(*shape, std=0.7, mean=-mean, dtype=ht), weight=normal(C, std=0.2, mean=1.0))
    if bias:
        v["bias"] = normal(C, std=0.3)
    if post:
        v["post_weight"] = normal(C, std=0.2, mean=1.0)
        if bias:
            v["post_bias"] = normal(C, std=0.3)
    if gate:
        s = dict(channel=(C,), sample=(shape[0], *(1,) * (len(shape) - 2), C),
                 flat=(shape[0], C))[gate]
        v["gate"] = normal(*s, std=0.4, mean=0.2)
    return v, normal(*shape, dtype=xt), normal(*shape, dtype=yt)


def exact(v, kind, scale):
    C = (v["x"].shape[-1],)

    def norm(u, w, b):
        if kind == "layer":
            return F.layer_norm(u, C, w, b, EPS)
        u = F.rms_norm(u, C, w, EPS)
        return u if b is None else u + b

    n = norm(v["h"], v["post_weight"], v.get("post_bias")) if "post_weight" in v else v["h"]
    gate = v.get("gate")
    if gate is not None and gate.dim() != 1:
        gate = gate.reshape(gate.shape[0], *(1,) * (v["x"].dim() - 2), C[0])
    xo = v["x"] + scale * (n if gate is None else gate * n)
    return xo, norm(xo, v["weight"], v.get("bias"))


def run(v, dxo, dy, kind, scale):
    leaves = {k: t.detach().requires_grad_(True) for k, t in v.items()}
    kw = {k: leaves[k] for k in ("post_weight", "post_bias", "gate") if k in v}
    xo, y = ops.residual_norm(leaves["x"], leaves["h"], leaves["weight"], leaves.get("bias"),
                              scale=scale, kind=kind, out_dtype=dy.dtype, eps=EPS, **kw)
    outs, ups = ((xo, y), (dxo, dy)) if dxo is not None else ((y,), (dy,))
    grads = torch.autograd.grad(outs, list(leaves.values()), ups)
    return xo, y, dict(zip(leaves, grads))


def close(got, want, k, size, what):
    """|got - want| <= k u size + half a step of got's type."""
    err = (got.double() - want).abs()
    bound = k * U * size + torch.finfo(got.dtype).eps / 2 * want.abs() * 1.01
    assert torch.isfinite(got).all(), what
    assert float((err - bound).max()) <= 0, (what, float(err.max()), float((err / bound).max()))


def check(shape, xt, ht, yt, gate, bias, post, kind, with_dxo=True, scale=0.7, seed=0, mean=0.3):
    v, dxo, dy = inputs(shape, xt, ht, yt, gate, bias, post, seed, mean)
    if not with_dxo:
        dxo = None
    xo, y, grads = run(v, dxo, dy, kind, scale)
    assert xo.dtype == xt and y.dtype == yt and xo.shape == y.shape == tuple(shape)
    v64 = {k: t.double().requires_grad_(True) for k, t in v.items()}
    wxo, wy = exact(v64, kind, scale)
    outs, ups = ((wxo, wy), (dxo.double(), dy.double())) if with_dxo else ((wy,), (dy.double(),))
    want = dict(zip(v64, torch.autograd.grad(outs, list(v64.values()), ups)))
    # magnitudes: what values of a row are made of
    N, C = v["x"].numel() // shape[-1], shape[-1]
    row = lambda t: t.detach().abs().amax(-1, keepdim=True).double()  # noqa: E731
    big = row(v["x"]) + row(wxo) + 4.0
    close(xo, wxo.detach(), 128, big, "sum")
    std = wxo.detach().std(-1, unbiased=False, keepdim=True) if C > 1 else 0 * big
    inv = 1 / (std.square() + EPS).sqrt()
    hstd = v["h"].double().std(-1, unbiased=False, keepdim=True) if C > 1 else 0 * big
    hinv = 1 / (hstd.square() + EPS).sqrt() if post else 1 + 0 * big
    if kind == "rms":
        inv = 1 / (wxo.detach().square().mean(-1, keepdim=True) + EPS).sqrt()
        hinv = 1 / (v["h"].double().square().mean(-1, keepdim=True) + EPS).sqrt() if post else hinv
    # hat h is off by k u max|h| / std(h); x' by that times scale and gate
    off_n = row(v["h"]) * hinv + 4.0
    off_x = big + off_n
    off_y = off_x * inv + 4.0
    close(y, wy.detach(), 128, off_y * 2, "norm")
    up = row(dy) * 3 + 1.0
    d_size = ((row(dxo) if with_dxo else 0.0) + up * inv * (1 + off_y) ** 2) * 3 + 1.0
    close(grads["x"], want["x"], 512, d_size, "dx")
    h_size = d_size * (hinv * (1 + off_n) ** 2 if post else 1.0) * 4
    close(grads["h"], want["h"], 512, h_size, "dh")
    ctas = min(N, 592)
    terms = N / ctas + ctas / 8 + 16
    flat = lambda t: t.expand(*shape[:-1], 1).reshape(N, 1)  # noqa: E731

    def summed(name, each, share=N):
        """Column sums over `share` rows each: every term off by 512 u of `each`, added in
        `terms` steps."""
        size = flat(each).reshape(-1, share).sum(1).reshape(-1, 1)
        g = grads[name].reshape(size.shape[0], -1)
        close(g, want[name].reshape(g.shape), 512 + terms, size, name)
        assert grads[name].shape == v[name].shape

    summed("weight", up * (1 + off_y))
    if bias:
        summed("bias", up)
    if post:
        summed("post_weight", d_size * (1 + off_n) * 2)
        if bias:
            summed("post_bias", d_size * 2)
    if gate:
        summed("gate", d_size * (1 + off_n) * 2, N if gate == "channel" else N // shape[0])


SHAPES = [(1, 1), (3, 2), (5, 7), (2, 3, 30), (4, 33), (2, 5, 768), (3, 4, 1000), (1, 2, 1024),
          (3, 1025), (2, 3, 1999), (2, 2, 2052), (2, 4095), (3, 4096), (2, 2, 3, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("xt,ht,yt,gate,bias,post,with_dxo", [
    (F32, BF16, BF16, "channel", True, True, True),
    (F32, F32, F32, "sample", False, True, True),
    (BF16, BF16, BF16, None, False, True, False),
    (BF16, F32, F32, "flat", True, False, True),
    (F32, BF16, F32, None, True, False, True),
])
def test_matches_the_definition(shape, kind, xt, ht, yt, gate, bias, post, with_dxo):
    if gate == "sample" and len(shape) == 2:
        gate = "flat"
    check(shape, xt, ht, yt, gate, bias, post, kind, with_dxo)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,gate", [((7, 400, 48), "sample"), ((1200, 3, 20), "sample"),
                                        ((5003, 36), "flat"), ((3000, 130), "channel"),
                                        ((16, 257, 768), "sample")])
def test_many_rows_and_gates(shape, gate):
    """Runs of rows that end inside a sample, samples that end inside a run."""
    check(shape, F32, BF16, BF16, gate, True, True, "layer")


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(900, 31), (3, 400, 127), (2, 1500, 128), (700, 129), (700, 132),
                                   (500, 256), (500, 257), (400, 2048), (5, 80, 2049),
                                   (400, 2304), (400, 2305), (3, 120, 3333), (350, 4093),
                                   (2, 170, 4096)])
@pytest.mark.parametrize("bias,gate", [(True, "channel"), (False, "sample")])
def test_widths_around_the_layouts_borders(shape, bias, gate):
    """Widths at which another number of warps or columns a lane takes a row."""
    check(shape, BF16, F32, BF16, "flat" if len(shape) == 2 and gate == "sample" else gate, bias,
          True, "layer")


@pytest.mark.gpu
def test_more_elements_than_32_bits_count():
    """The last rows of a stream of more than 2**31 elements are what they are on their own."""
    N, C, n = 2**31 // 2050 + 400, 2050, 300
    gen = torch.Generator("cuda").manual_seed(3)
    x, h, dy, dxo = (torch.empty(N, C, device="cuda", dtype=BF16).normal_(generator=gen)
                     for _ in range(4))
    w, wp = (torch.rand(C, device="cuda", generator=gen) + 0.5 for _ in range(2))

    def grads(x, h, dy, dxo):
        x, h = x.requires_grad_(), h.requires_grad_()
        out = ops.residual_norm(x, h, w, post_weight=wp, out_dtype=BF16)
        return [t.detach() for t in (*out, *torch.autograd.grad(out, (x, h), (dxo, dy)))]

    assert N * C > 2**31
    few = grads(*(t[-n:].clone() for t in (x, h, dy, dxo)))
    for got, want in zip(grads(x, h, dy, dxo), few):
        assert torch.equal(got[-n:], want)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_constant_rows_and_zero_rows(kind):
    """Rows without variance: 1/std is 1/sqrt(eps), nothing is NaN."""
    x = torch.zeros(3, 64, device="cuda")
    x[1] = 7.0
    h = torch.zeros(3, 64, device="cuda", dtype=BF16)
    h[2] = 3.0
    v = dict(x=x, h=h, weight=torch.ones(64, device="cuda"),
             post_weight=torch.ones(64, device="cuda"))
    up = torch.zeros(3, 64, device="cuda")
    xo, y, grads = run(v, up, up, kind, 1.0)
    v64 = {k: t.double() for k, t in v.items()}
    wxo, wy = exact(v64, kind, 1.0)
    torch.testing.assert_close(xo.double(), wxo, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(y.double(), wy, rtol=1e-5, atol=1e-5)
    assert all(torch.count_nonzero(g) == 0 for g in grads.values())


@pytest.mark.gpu
def test_a_nan_row_stays_in_its_row():
    v, dxo, dy = inputs((4, 96), F32, BF16, F32, None, False, True)
    v["h"][2, 5] = math.nan
    xo, y, grads = run(v, dxo, dy, "layer", 1.0)
    bad = torch.tensor([False, False, True, False], device="cuda")[:, None].expand(4, 96)
    for t in (xo, y, grads["x"], grads["h"]):
        assert torch.equal(t.isnan(), bad)


@pytest.mark.gpu
def test_far_mean_keeps_its_digits():
    """A mean of 1000 stds: the variance is of differences, not of squares (whose difference
    would keep no digit: 2^-24 * 1e6 = 6 %)."""
    g = torch.Generator().manual_seed(0)
    x = (1000 + torch.randn(8, 512, generator=g)).cuda()
    h = torch.zeros(8, 512, device="cuda")
    w = torch.ones(512, device="cuda")
    _, y = ops.residual_norm(x, h, w)
    want = F.layer_norm(x.double(), (512,), None, None, EPS)
    # the mean's own rounding, 18 u * 1000, shifts every element alike
    assert float((y.double() - want).abs().max()) <= 20 * U * 1000 + 64 * U * 5


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["offset", "expanded", "transposed"])
def test_layouts(layout):
    v, dxo, dy = inputs((3, 5, 64), F32, BF16, BF16, "sample", True, True)
    want = run(v, dxo, dy, "layer", 0.5)
    if layout == "offset":  # contiguous rows off the 16-byte grid
        for k in ("x", "h", "weight", "gate"):
            buf = torch.empty(v[k].numel() + 1, dtype=v[k].dtype, device="cuda")
            buf[1:] = v[k].reshape(-1)
            v[k] = buf[1:].view(v[k].shape)
    elif layout == "expanded":
        dy = dy[:, :1].expand(3, 5, 64)
        want = run(v, dxo, dy.contiguous(), "layer", 0.5)
    else:
        v["x"] = v["x"].transpose(0, 1).contiguous().transpose(0, 1)
        dxo = dxo.transpose(1, 2).contiguous().transpose(1, 2)
    got = run(v, dxo, dy, "layer", 0.5)
    for a, b in zip([*got[:2], *got[2].values()], [*want[:2], *want[2].values()]):
        torch.testing.assert_close(a.double(), b.double(), rtol=2e-5 if a.dtype == F32 else 2**-7,
                                   atol=2e-5)


@pytest.mark.gpu
def test_bf16_parameters_get_bf16_gradients_and_one_output_unused():
    v, dxo, dy = inputs((2, 5, 64), F32, BF16, BF16, "sample", False, True)
    v["gate"], v["weight"] = v["gate"].bfloat16(), v["weight"].bfloat16()
    _, _, grads = run(v, dxo, dy, "rms", 1.0)
    assert grads["gate"].dtype == grads["weight"].dtype == BF16
    x = v["x"].requires_grad_(True)
    xo, _ = ops.residual_norm(x, v["h"], v["weight"])
    (g,) = torch.autograd.grad(xo, x, dxo)  # the norm is not used: the add's gradient
    assert torch.equal(g, dxo)


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    x = torch.randn(3, 64, device="cuda", requires_grad=True)
    _, y = ops.residual_norm(x, x.detach(), torch.ones(64, device="cuda"))
    (g,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


@pytest.mark.gpu
def test_no_rows():
    x = torch.empty(0, 5, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    xo, y = ops.residual_norm(x, x.detach(), w, post_weight=w)
    gx, gw = torch.autograd.grad(y.sum() + xo.sum(), (x, w))
    assert gx.shape == x.shape and torch.count_nonzero(gw) == 0


@pytest.mark.gpu
def test_gradients_against_differences():
    v, dxo, dy = inputs((2, 3, 48), F32, F32, F32, "sample", True, True)
    _, _, grads = run(v, dxo, dy, "layer", 0.7)
    g = torch.Generator().manual_seed(4)
    h = 2.0**-8

    def value(u, f):
        xo, y = f(u)
        return float((xo.double() * dxo.double()).sum() + (y.double() * dy.double()).sum())

    def mine(u):
        kw = {k: u[k] for k in ("post_weight", "post_bias", "gate")}
        return ops.residual_norm(u["x"], u["h"], u["weight"], u["bias"], scale=0.7, **kw)

    for k in v:
        d = torch.randn(v[k].shape, generator=g).cuda()
        moved = [{**v, k: v[k] + s * h * d} for s in (1, -1)]
        diff = (value(moved[0], mine) - value(moved[1], mine)) / (2 * h)
        wide = [{n: t.double() for n, t in m.items()} for m in moved]
        true = (value(wide[0], lambda u: exact(u, "layer", 0.7))
                - value(wide[1], lambda u: exact(u, "layer", 0.7))) / (2 * h)
        slope = float((grads[k].double() * d.double()).sum())
        v64 = {n: t.double().requires_grad_(True) for n, t in v.items()}
        xo, y = exact(v64, "layer", 0.7)
        (w,) = torch.autograd.grad((xo * dxo.double()).sum() + (y * dy.double()).sum(), v64[k])
        curved = abs(true - float((w * d.double()).sum()))
        # two values, each a sum of 576 products off by 128 u of about 10
        rounding = 576 * 128 * U * 10 / h / 10
        assert abs(diff - slope) <= curved + rounding + 1e-4 * abs(slope), k


@pytest.mark.gpu
def test_same_bits_captured_and_on_two_streams():
    a = inputs((4, 300, 768), F32, BF16, BF16, "sample", False, True)
    b = inputs((4, 300, 768), F32, BF16, BF16, "sample", False, True, seed=5)

    def step(case):
        v, dxo, dy = case
        xo, y, grads = run(v, dxo, dy, "layer", 0.5)
        return [xo, y, *grads.values()]

    want = [step(a), step(b)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(6):
        s = streams[i % 2]
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(step((a, b)[i % 2]))
    torch.cuda.synchronize()
    for i, r in enumerate(got):
        assert all(torch.equal(p, q) for p, q in zip(r, want[i % 2]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(a)
    for src, w in ((b, want[1]),):
        for k in a[0]:
            a[0][k].copy_(src[0][k])
        a[1].copy_(src[1]), a[2].copy_(src[2])
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(out, w))


@pytest.mark.gpu
def test_compiles_without_a_break():
    v, dxo, dy = inputs((2, 5, 64), F32, BF16, BF16, "channel", True, True)
    leaves = {k: t.requires_grad_(True) for k, t in v.items()}

    def f(u):
        xo, y = ops.residual_norm(u["x"], u["h"], u["weight"], u["bias"], gate=u["gate"],
                                  post_weight=u["post_weight"], out_dtype=BF16)
        return (xo * dxo).sum() + (y.float() * dy.float()).sum()

    names = [k for k in leaves if k != "post_bias"]
    want = torch.autograd.grad(f(leaves), [leaves[k] for k in names])
    got = torch.autograd.grad(torch.compile(f, backend="aot_eager", fullgraph=True)(leaves),
                              [leaves[k] for k in names])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
