"""The residual step's C entry points as host programs call them: from several threads at
once, and with the scratch that they ask for."""

import ctypes
import threading

import pytest
import torch

from llm_training_b200 import _lib, ops


class Backward:
    """sqb_residual_norm_bwd of N fp32 rows of C on a stream of its own."""

    def __init__(self, N, C):
        g = torch.Generator("cuda").manual_seed(C)
        self.lib = _lib.lib()
        self.N, self.C = N, C
        self.x, self.h, self.dy = (torch.randn(N, C, device="cuda", generator=g) for _ in range(3))
        self.w = torch.ones(C, device="cuda")
        nbytes = self.lib.sqb_residual_norm_workspace_bytes(N, C, 0)
        self.ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
        self.stats = torch.empty(4 * N, device="cuda")
        self.out = [torch.empty_like(v) for v in (self.x, self.x, self.w)]  # dx, dh, dw
        self.stream = torch.cuda.Stream()
        xo, y = torch.empty_like(self.x), torch.empty_like(self.x)
        p = self.pointer
        rc = self.lib.sqb_residual_norm_fwd(p(self.x), 0, p(self.h), 0, p(self.w), *(None,) * 4, 0,
                                            1.0, 1e-5, 0, p(xo), p(y), 0, p(self.stats), N, C, None)
        assert rc == 0

    @staticmethod
    def pointer(t):
        return ctypes.c_void_p(t.data_ptr())

    def __call__(self):
        p = self.pointer
        return self.lib.sqb_residual_norm_bwd(
            p(self.dy), 0, None, p(self.x), 0, p(self.h), 0, p(self.w), *(None,) * 4, 0, 1.0, 1e-5,
            0, p(self.stats), p(self.out[0]), p(self.out[1]), p(self.out[2]), *(None,) * 4,
            p(self.ws), self.ws.numel(), self.N, self.C, ctypes.c_void_p(self.stream.cuda_stream))

    def expected(self):
        x, h, w = (v.clone().requires_grad_(True) for v in (self.x, self.h, self.w))
        return torch.autograd.grad(ops.residual_norm(x, h, w)[1], (x, h, w), self.dy)


@pytest.mark.gpu
def test_two_threads_with_rows_of_different_widths():
    """Two widths share a kernel and ask it for different amounts of shared memory: neither may
    take the other's away between its limit and its launch."""
    jobs = [Backward(64, 4096), Backward(64, 260)]
    torch.cuda.synchronize()
    codes = [[], []]
    start = threading.Barrier(2)

    def run(i):
        start.wait()
        codes[i] = [jobs[i]() for _ in range(500)]

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    assert set(codes[0]) == set(codes[1]) == {0}
    for job in jobs:
        assert all(torch.equal(a, b) for a, b in zip(job.out, job.expected()))


@pytest.mark.parametrize("gates", [0, 1, 8])
@pytest.mark.parametrize("C", [1, 32, 100, 128, 129, 768, 1999, 4095, 4096])
@pytest.mark.parametrize("N", [1, 7, 1184, 16384, 2**31 - 8])
def test_scratch_is_what_the_rows_need(N, C, gates):
    """A partial row of each of five parameters for every CTA - at most 16 warps of them on each
    of 148 SMs, a warp holding 256 columns of a row - and one row for each run and gate that meet."""
    warps = -(-C // 256)
    ctas = min(N, 148 * (16 // warps))
    runs = min(N, 148 * 16)
    pitch = -(-C // 4) * 4
    most = (5 * ctas + (runs + gates if gates > 1 else 0)) * pitch * 4
    nbytes = _lib.lib().sqb_residual_norm_workspace_bytes(N, C, gates)
    assert 0 < nbytes <= most and nbytes % 16 == 0


def test_no_scratch_for_what_is_refused():
    nbytes = _lib.lib().sqb_residual_norm_workspace_bytes
    assert nbytes(0, 8, 0) == nbytes(8, 0, 0) == nbytes(8, 8, -1) == nbytes(8, 4097, 0) == 0
