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
