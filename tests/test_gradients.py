"""Global gradient norm and clipping (csrc/sqb_gradclip.cu).

Bounds: the squares are summed in 64 bits, so the norm is the exact one rounded to fp32
(2^-24 relative, and 2^-50 a term before that); the factor max_norm / (norm + 1e-6) has
the roundings of a sum, a quotient and the norm (3 * 2^-24), the scaled gradient one more,
and half a step of its type."""

import ctypes
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from llm_training_b200 import _lib, ops

U = 2.0**-24
ERR_ARG, ERR_DTYPE, ERR_ALIGN, ERR_WORKSPACE = 1, 2, 3, 5


def test_refusals():
    with FakeTensorMode():
        f = [torch.empty(3, device="cuda"), torch.empty(4, 5, device="cuda")]
        for call, kind, text in [
            (lambda: ops.grad_norm([torch.empty(3)]), RuntimeError, "CUDA"),
            (lambda: ops.grad_norm([f[0].half()]), TypeError, "float32 and bfloat16"),
            (lambda: ops.grad_norm([f[0], torch.empty(3)]), ValueError, "one device"),
            (lambda: ops.clip_grads(f, -1.0), ValueError, "max_norm"),
            (lambda: ops.clip_grads(f, math.nan), ValueError, "max_norm"),
            (lambda: ops.clip_grads(f, 1.0, out=f[:1]), ValueError, "shape"),
            (lambda: ops.clip_grads(f, 1.0, out=[f[0], f[1].t()]), ValueError, "shape"),
            (lambda: ops.clip_grads(f, 1.0, out=[f[0], torch.empty(5, 4, device="cuda").t()]),
             ValueError, "contiguous"),
            (lambda: ops.clip_grads(f, 1.0, out=[f[0].double(), f[1]]), TypeError, "float32"),
        ]:
            with pytest.raises(kind, match=text):
                call()
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.zeros(3)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.clip_grad_norm_([p], 1.0)
    p.grad = torch.zeros(3).to_sparse()
    with pytest.raises(ValueError, match="layout"):
        ops.clip_grad_norm_(p, 1.0)


def test_nothing_to_clip():
    p = torch.nn.Parameter(torch.zeros(3))
    assert float(ops.clip_grad_norm_([p], 1.0)) == 0.0
    assert float(ops.grad_norm([])) == 0.0
    assert ops.clip_grads([], 1.0)[0] == []


def test_c_entry_points_reject_bad_arguments_without_a_device():
    lib = _lib.lib()

    def call(ptr=256, numel=4, dtype=0, out=256, out_dtype=0, n=1, max_norm=1.0, ws=256,
             ws_bytes=1 << 20, norm=256):
        table = lambda kind, v: (kind * 1)(v)  # noqa: E731
        return lib.sqb_grad_clip(table(ctypes.c_void_p, ptr), table(ctypes.c_void_p, out),
                                 table(ctypes.c_int64, numel), table(ctypes.c_int32, dtype),
                                 table(ctypes.c_int32, out_dtype), n, max_norm, ws, ws_bytes,
                                 norm, None)

    assert call(n=0) == ERR_ARG and call(ptr=None) == ERR_ARG and call(out=None) == ERR_ARG
    assert call(numel=-1) == ERR_ARG and call(numel=1 << 46) == ERR_ARG
    assert call(norm=None) == ERR_ARG and call(max_norm=-1.0) == ERR_ARG
    assert call(max_norm=math.nan) == ERR_ARG
    assert call(dtype=3) == ERR_DTYPE and call(out_dtype=3) == ERR_DTYPE
    assert call(ptr=258) == ERR_ALIGN and call(ptr=257, dtype=1) == ERR_ALIGN
    assert call(ws=None) == ERR_WORKSPACE and call(ws_bytes=8) == ERR_WORKSPACE
    assert lib.sqb_grad_norm(None, None, None, 1, None, 0, None, None) == ERR_ARG
    assert lib.sqb_grad_norm_workspace_bytes(0) == 0


def tensors(sizes, dtypes, seed=0, std=1.0, phase=0):
    """Views of one buffer per dtype, back to back from element `phase` on."""
    g = torch.Generator().manual_seed(seed)
    flat = {d: torch.zeros(phase + sum(math.prod(s) for s in sizes), dtype=d, device="cuda")
            for d in set(dtypes)}
    at, got = phase, []
    for i, s in enumerate(sizes):
        d, n = dtypes[i % len(dtypes)], math.prod(s)
        v = flat[d][at:at + n].view(s)
        v.copy_(torch.randn(s, generator=g) * std)
        at += n
        got.append(v)
    return got


def check(outs, grads, norm, max_norm):
    total = torch.cat([g.double().reshape(-1) for g in grads]).square().sum().sqrt()
    assert norm.dtype == torch.float32 and norm.shape == ()
    assert abs(float(norm) - float(total)) <= 1.01 * U * float(total)
    factor = min(1.0, max_norm / (float(total) + 1e-6))
    for o, g in zip(outs, grads):
        want = g.double() * factor
        half = torch.finfo(o.dtype).eps / 2 if o.dtype != g.dtype or factor != 1.0 else 0.0
        assert float(((o.double() - want).abs() - want.abs() * (half + 6 * U)).max()
                     if o.numel() else 0.0) <= 2.0**-126


SIZES = [
    [(1,)], [(7,), (3, 5)], [(0,), (9,)], [(16384,), (16385,), (1,)],
    [(768,)] * 5 + [(768, 768)] * 3, [(1003, 97)] * 2 + [(13,)] * 40,
]
F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("phase", [0, 1, 3])
@pytest.mark.parametrize("dtypes,out", [((F32,), F32), ((BF16,), BF16), ((BF16,), F32),
                                        ((F32,), BF16), ((F32, BF16), F32)])
@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("bound", [0.3, 3.0])
def test_clip_into_other_tensors(sizes, dtypes, out, phase, bound):
    grads = tensors(sizes, dtypes, phase=phase)
    max_norm = bound * math.sqrt(sum(math.prod(s) for s in sizes))
    outs = tensors(sizes, (out,), seed=5, phase=(phase * 2) % 5)
    kept = [g.clone() for g in grads]
    got, norm = ops.clip_grads(grads, max_norm, out=outs)
    assert got[0] is outs[0]
    check(outs, grads, norm, max_norm)
    assert all(torch.equal(a, b) for a, b in zip(grads, kept))
    fresh, norm2 = ops.clip_grads(grads, max_norm)
    check(fresh, grads, norm2, max_norm)
    assert torch.equal(norm, norm2) and torch.equal(norm, ops.grad_norm(grads))
    assert [f.dtype for f in fresh] == [g.dtype for g in grads]


@pytest.mark.gpu
@pytest.mark.parametrize("dtypes", [(F32,), (BF16,), (F32, BF16)])
@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("bound", [0.0, 0.3, 3.0, math.inf])
def test_clip_in_place_and_as_torch_does(sizes, dtypes, bound):
    grads = tensors(sizes, dtypes, phase=1)
    kept = [g.clone() for g in grads]
    params = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
    for p, g in zip(params, grads):
        p.grad = g
    params.append(torch.nn.Parameter(torch.zeros(2, device="cuda")))  # no gradient
    max_norm = bound * math.sqrt(sum(math.prod(s) for s in sizes)) if bound else 0.0
    norm = ops.clip_grad_norm_(iter(params), max_norm)
    check(grads, kept, norm, max_norm)
    others = [torch.nn.Parameter(torch.zeros_like(g)) for g in kept]
    for p, g in zip(others, kept):
        p.grad = g.float().clone() if g.dtype == F32 else g.clone()
    if len(dtypes) == 1 and dtypes[0] == F32 and 0 < bound < math.inf:
        torch.testing.assert_close(norm, torch.nn.utils.clip_grad_norm_(others, max_norm),
                                   rtol=2e-5, atol=0)


@pytest.mark.gpu
def test_more_tensors_than_one_table_holds():
    sizes = [(1 + i % 11,) for i in range(2000)]
    grads = tensors(sizes, (F32, BF16))
    kept = [g.clone() for g in grads]
    outs, norm = ops.clip_grads(grads, 5.0)
    check(outs, kept, norm, 5.0)
    params = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
    for p, g in zip(params, grads):
        p.grad = g
    assert torch.equal(ops.clip_grad_norm_(params, 5.0), norm)
    assert all(torch.equal(a, b) for a, b in zip(grads, outs))


@pytest.mark.gpu
@pytest.mark.parametrize("value", [1e-25, 1e25])
def test_squares_out_of_fp32_range(value):
    """Squares of 1e-50 and 1e50 have no fp32 value; the norm has."""
    g = torch.full((1000,), value, device="cuda")
    assert float(ops.grad_norm([g])) == pytest.approx(value * math.sqrt(1000), rel=1e-6)
    out, _ = ops.clip_grads([g], value)
    if value > 1:  # (below, norm + 1e-6 is 1e-6)
        assert float(out[0][0]) == pytest.approx(value / math.sqrt(1000), rel=1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_non_finite_gradients_as_torch(value):
    def grads():
        g = tensors([(50,), (20000,)], (F32,))
        g[1][19999] = value
        return g

    mine, theirs = ([torch.nn.Parameter(torch.zeros_like(v)) for v in grads()] for _ in range(2))
    for ps in (mine, theirs):
        for p, g in zip(ps, grads()):
            p.grad = g
    a, b = ops.clip_grad_norm_(mine, 1.0), torch.nn.utils.clip_grad_norm_(theirs, 1.0)
    assert float(a) == float(b) or (a.isnan() and b.isnan())
    for p, q in zip(mine, theirs):
        torch.testing.assert_close(p.grad, q.grad, rtol=0, atol=0, equal_nan=True)


@pytest.mark.gpu
def test_layouts_and_parameters_listed_twice():
    g = torch.Generator().manual_seed(0)
    base = torch.randn(40, 60, generator=g).cuda()
    grads = [base.clone().t(), base.clone()[:, ::2], base.clone()[5:9],
             torch.randn(2, 3, 4, 5, generator=g).cuda().to(memory_format=torch.channels_last)]
    kept = [v.clone() for v in grads]
    params = [torch.nn.Parameter(torch.zeros_like(v)) for v in grads]
    for p, v in zip(params, grads):
        p.grad = v
    norm = ops.clip_grad_norm_(params + params[:2], 1.0)
    check([p.grad for p in params], kept, norm, 1.0)
    assert all(p.grad is v for p, v in zip(params, grads))
    assert torch.equal(norm, ops.grad_norm(kept)) or abs(float(norm) - float(
        ops.grad_norm(kept))) <= 2 * U * float(norm)
    outs, _ = ops.clip_grads(kept, 1.0)
    check(outs, kept, norm, 1.0)
    wide = torch.nn.Parameter(torch.zeros(3, 4, device="cuda"))
    wide.grad = torch.ones(4, device="cuda").expand(3, 4)
    with pytest.raises(ValueError, match="in place"):
        ops.clip_grad_norm_([wide], 1.0)
    assert float(ops.grad_norm([wide.grad])) == pytest.approx(math.sqrt(12), rel=1e-6)
    with pytest.raises(ValueError, match="twice"):
        ops.clip_grads([base, base], 1.0, out=[grads[2].new_empty(40, 60)] * 2)


@pytest.mark.gpu
def test_more_elements_than_32_bits_count():
    n = 2**31 + 70_003
    g = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    g[-70_000:] = 2.0
    g[0] = 2.0
    other = torch.ones(5, device="cuda")
    want = (4 * 70_001 + 5) ** 0.5
    (a, b), norm = ops.clip_grads([g, other], 1.0, out=[torch.empty_like(g), other])
    # the norm and the factor are rounded to 24 bits, the product once more to 8
    assert abs(float(norm) - want) <= want * 2**-24
    factor = 1.0 / (want + 1e-6)
    for got, times, eps in ((a, 2.0, 2**-8), (b, 1.0, 2**-24)):
        size = got[got != 0].double()
        assert (size - times * factor).abs().max() <= times * factor * (eps + 3 * 2**-24)
    assert int((a != 0).sum()) == 70_001 and a[0] != 0 and (a[-70_000:] != 0).all()


@pytest.mark.gpu
def test_shared_gradients_are_refused():
    """Memory that would be scaled twice, or read while it is written."""
    p, q = (torch.nn.Parameter(torch.ones(3, device="cuda")) for _ in range(2))
    p.grad = q.grad = torch.ones(3, device="cuda")
    with pytest.raises(ValueError, match="share"):
        ops.clip_grad_norm_([p, q], 0.5)
    a, b = torch.ones(4, device="cuda"), torch.ones(4, device="cuda")
    with pytest.raises(ValueError, match="another gradient"):
        ops.clip_grads([a, b], 0.5, out=[b, torch.empty_like(a)])
    with pytest.raises(ValueError, match="another gradient"):
        ops.clip_grads([a, b], 0.5, out=[b, a])
    with pytest.raises(ValueError, match="twice"):
        ops.clip_grads([a, a], 0.5, out=[a, a])
    assert p.grad.eq(1).all() and a.eq(1).all() and b.eq(1).all()
    # out of place a gradient may be listed twice: it counts twice
    (c, d), norm = ops.clip_grads([a, a], 10.0)
    assert float(norm) == 8**0.5 or abs(float(norm) - 8**0.5) <= 2**-23
    assert torch.equal(c, a) and torch.equal(d, a)


@pytest.mark.gpu
def test_autograd_sees_the_write():
    """A graph that holds a tensor scaled in place says so, as after any in-place operation."""
    p = torch.nn.Parameter(torch.zeros(8, device="cuda"))
    w = torch.ones(8, device="cuda", requires_grad=True)
    p.grad = torch.full((8,), 3.0, device="cuda")
    loss = (w * p.grad).sum()
    ops.clip_grad_norm_([p], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.gpu
def test_captured_and_on_two_streams():
    grads = tensors([(768, 300), (77,)], (F32,))
    src = [g.clone() for g in grads]
    outs = [torch.empty_like(g) for g in grads]
    ops.clip_grads(grads, 1.0, out=outs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, norm = ops.clip_grads(grads, 1.0, out=outs)
    for k in (2.0, 0.001):
        for g, s in zip(grads, src):
            g.copy_(s * k)
        graph.replay()
        check(outs, grads, norm, 1.0)
    other = tensors([(768, 300), (77,)], (BF16,), seed=3)
    want = [ops.clip_grads(v, 1.0) for v in (grads, other)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(6):
        s = streams[i % 2]
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(ops.clip_grads((grads, other)[i % 2], 1.0))
    torch.cuda.synchronize()
    for i, (o, n) in enumerate(got):
        assert torch.equal(n, want[i % 2][1])
        assert all(torch.equal(a, b) for a, b in zip(o, want[i % 2][0]))
