"""Ratios next to the border of their clipping, with rows of ordinary logits: farther from it than log-probabilities are exact, they fall on the side that they
belong to; nearer, on one of the two."""
import math

import pytest
import torch

from superscaler_amd import layer
from tests.test_layer_loss import BF16, E24, F16, F32, case, cuda_or_skip, logp_bound, logprobs

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("vocab", [700, 20000, 51200, 140001])
def test_the_side_of_the_border(vocab, dtype):
    device = cuda_or_skip()
    low, high, rows = 0.2, 0.28, 64
    z, t = case(vocab, rows, vocab, dtype, none=False)
    logp, bound = logprobs(z, t)[0], logp_bound(z)
    A = torch.where(torch.arange(rows) % 2 == 0, 1.0, -1.0)
    border = torch.where(A > 0, math.log(1 + high), math.log(1 - low)).double()
    # from a few bounds before to a few behind, most of them near
    off = torch.linspace(-4, 4, rows, dtype=torch.float64) * bound
    old = (logp - border - off).float()
    margin = logp - old.double() - border
    r, grad = layer.policy_loss_gradient(*(x.to(device) for x in (z, t, old, A)), clip=(low, high))
    alone = layer.policy_loss(*(x.to(device) for x in (z, t, old, A)), clip=(low, high))
    free, clear = torch.where(A > 0, margin <= 0, margin >= 0), margin.abs() > bound + 2 * E24
    assert int(clear.sum()) > rows // 2
    for got in (r, alone):
        d = got.d_logp.cpu().double()
        assert torch.equal((d != 0)[clear], free[clear])
        # whichever side, the derivative is that side's: nothing, or all of it
        want = -(margin + border).exp() * A / rows
        assert ((d == 0) | ((d - want).abs() <= want.abs() * (2 * bound + 4 * E24))).all()
    assert torch.equal(r.d_logp, alone.d_logp) and torch.equal((grad != 0).any(-1), r.d_logp != 0)
