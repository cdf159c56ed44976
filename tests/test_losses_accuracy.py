"""How far sums of log-probabilities are from 64 bits.

The losses are made of sums over hundreds of tokens, so an error that all rows share grows with
the length of an answer, where errors without a shared sign do not.  With the reference sums set
to the exact ones, rounded to fp32, a reward of beta = 1 is a sequence's sum less a number that is
known exactly, and small: the sum's own error shows to 2^-24 of about 1e-4.

Bounds.  A row's log-sum is off by the mean of its exponentials' errors, weighted by the
exponentials:
* ex2.approx is off by 2^-22 at most; its mean shortfall, 5.06e-8, is made up for, and over
  arguments that are spread out the rest has no shared sign: below 1e-7 in the root mean square
  where one exponential is all of a row;
* an argument is exact, or rounded where the logit's product is smaller than the reference
  that is taken from it: by 2^-24 of a difference d, weighted by 2^-d, 2^-25 at most;
* partial sums of 32 exponentials in fp32: a few 2^-24, without a shared sign; above that, 64
  bits.
1.2e-7 a row in the root mean square in all: 2.7e-6 for 512 rows, and four times that is 512 *
2e-8.  The mean over all rows is held to the same 2e-8 a row, where 1.2e-7 / sqrt(8192) = 1.3e-9
would come from errors without a shared sign; a rounding of 2^-24 shared by the rows is 6e-8,
the uncorrected shortfall 5e-8.

bf16 logits from 16 on are not spread out: they are multiples of 1/8 (from 512 on of 4), so the
few exponentials that are most of a row's sum take the same few arguments in all rows, and what
ex2.approx is off there is shared.  Nothing but its bound is left: 2^-22, the 2^-24.2 that is
made up for, and 2^-25 of an argument, 0.4 * 2^-20 in all."""

import pytest
import torch

from llm_training_b200 import ops

pytestmark = pytest.mark.gpu

SEQUENCES, T = 16, 512
A_ROW, A_COARSE_ROW = 2e-8, 0.4 * 2.0**-20


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,std,peak,shift", [
    (97, 2.0, 6.0, 0.0), (1003, 4.0, 0.0, 7.0), (50257, 3.0, 9.0, 0.0), (5003, 2.0, 20.0, -40.0),
    (1003, 3.0, 12.0, 600.0)])
def test_sums_of_log_probabilities(V, std, peak, shift, dtype):
    g = torch.Generator("cuda").manual_seed(V)
    rows = SEQUENCES * T
    x = torch.randn(rows, V, device="cuda", generator=g) * std + shift
    x += torch.rand(rows, 1, device="cuda", generator=g)  # no shared place between whole numbers
    t = torch.randint(0, V, (rows,), device="cuda", generator=g)
    x.scatter_add_(1, t[:, None], peak * torch.rand(rows, 1, device="cuda", generator=g))
    x = x.to(dtype)
    exact = torch.cat([torch.log_softmax(c.double(), 1).gather(1, k[:, None])[:, 0]
                       for c, k in zip(x.split(1024), t.split(1024))])
    sums = exact.view(SEQUENCES, T).sum(1)
    ref = sums.float()
    _, chosen, rejected = ops.preference_loss(x.view(SEQUENCES, T, V), t.view(SEQUENCES, T), ref,
                                              beta=1.0)
    coarse = dtype == torch.bfloat16 and float(x.amax(1).abs().max()) >= 16
    a_row = A_COARSE_ROW if coarse else A_ROW
    known = sums - ref.double()
    off = torch.cat([chosen, rejected]).double() - known
    room = known.abs() * 2.0**-23
    assert (off.abs() <= T * a_row + room).all()
    assert abs(float(off.sum())) <= rows * a_row + float(room.sum())
