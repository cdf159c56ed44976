"""Gradients and outputs of the clipping calls that have memory in common: scaled twice, or
read while they are written.  All are refused before anything is written; memory that is only
next to other memory is not."""

import pytest
import torch

from llm_training_b200 import ops

pytestmark = pytest.mark.gpu


def params(*grads):
    got = []
    for g in grads:
        p = torch.nn.Parameter(torch.zeros(g.shape, device="cuda", dtype=g.dtype))
        p.grad = g
        got.append(p)
    return got


def buffer(n=120):
    return torch.arange(1.0, n + 1, device="cuda")


@pytest.mark.parametrize("views", [
    lambda b: (b[:60], b[59:]),
    lambda b: (b[:60], b[100:], b[10:20]),  # inside
    lambda b: (b[40:60], b[:100], b[100:]),
    lambda b: (b[:100].view(10, 10).t(), b[99:]),
    lambda b: (b[:60], b.view(torch.bfloat16)[119:]),  # its last two bytes
    lambda b: (b[:40], b[60:80].view(4, 5)[:, ::2], b[39:50]),  # next to one with gaps
])
def test_gradients_in_place(views):
    b = buffer()
    with pytest.raises(ValueError, match="overlap"):
        ops.clip_grad_norm_(params(*views(b)), 0.5)
    assert torch.equal(b, buffer())


def test_neighbours_in_place():
    b = buffer()
    rest = b[80:].view(10, 4)
    grads = (b[60:80], b[:60].view(6, 10).t(), b[20:20], rest[:, ::2], rest[:, 1::2])
    norm = ops.clip_grad_norm_(params(*grads), 0.5)
    want = buffer().double() * (0.5 / (float(norm) + 1e-6))
    assert ((b.double() - want).abs() <= want * 6 * 2.0**-24).all()
    # only next to one another in bytes, in two types
    c = torch.ones(8, device="cuda")
    halves = c.view(torch.bfloat16)
    assert ops.clip_grad_norm_(params(c[:4], halves[8:]), 100.0).isfinite()


def call(grads, out):
    kept = [(t, t.clone()) for t in (*grads, *out)]
    with pytest.raises(ValueError, match="overlap|twice|another"):
        ops.clip_grads(grads, 0.5, out=out)
    assert all(torch.equal(t, k) for t, k in kept)


def test_outputs():
    n = 40
    a, b, big = buffer(n), buffer(n), buffer(3 * n)
    fresh = torch.zeros(n, device="cuda")
    one = big[:n]
    call([a, b], [big[:n], big[n - 1:2 * n - 1]])  # two outputs
    call([one, b], [big[1:n + 1], fresh])  # its own gradient, from another start
    call([one, b], [fresh, big[n - 1:2 * n - 1]])  # another gradient
    call([big, b], [torch.zeros_like(big), big[n:2 * n]])  # inside another gradient
    call([one, big[n // 2:n // 2 + 4]], [one, fresh[:4]])  # in place, but read by another
    call([a, a], [a, fresh])  # the same, the gradient listed twice
    call([a, a], [fresh, a])
    call([one, one[:4]], [fresh, one[:4]])
    half = torch.ones(2 * n, device="cuda", dtype=torch.bfloat16)
    call([half[:n]], [half.view(torch.float32)])  # its memory in the other type
    call([b, half[:n]], [half.view(torch.float32), torch.zeros(n, device="cuda")])


def test_outputs_next_to_gradients():
    n = 40
    big, kept = buffer(4 * n), buffer(4 * n)
    grads = [big[:n], big[n:2 * n], big[2 * n:2 * n]]
    out = [big[:n], big[2 * n:3 * n], big[n:n]]  # in place; the next piece; nothing
    (a, b, c), norm = ops.clip_grads(grads, 0.5, out=out)
    want = kept.double()[:2 * n] * (0.5 / (float(norm) + 1e-6))
    got = torch.cat([a, b]).double()
    assert ((got - want).abs() <= want * 6 * 2.0**-24).all() and c.numel() == 0
    assert torch.equal(big[n:2 * n], kept[n:2 * n]) and torch.equal(big[3 * n:], kept[3 * n:])
    # one gradient into two places
    x, y = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    g = buffer(n)
    ops.clip_grads([g, g], 0.5, out=[x, y])
    assert torch.equal(x, y) and torch.equal(g, buffer(n))
