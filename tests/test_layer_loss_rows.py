"""Where the gradient of logits may go: rows between the logits' rows, and what meets them."""
import random as pyrandom

import pytest
import torch

from superscaler_amd import layer
from tests.test_layer_loss import BF16, F16, F32, cuda_or_skip, policy_case, random

gpu = pytest.mark.gpu


def test_rows_that_meet():
    """Against all of their bytes, one by one.  Rows at different distances that overlap as a whole are refused, whether they meet or not."""
    rng = pyrandom.Random(3)
    met = [0, 0]
    for _ in range(20000):
        rows, size = rng.randint(1, 5), rng.randint(1, 6)
        a_step = rng.randint(size, 15)
        b_step = a_step if rng.random() < 0.8 else rng.randint(size, 15)
        a, b = rng.randint(0, 40), rng.randint(0, 40)
        mine, other = ({at + r * step + i for r in range(rows) for i in range(size)} for at, step in ((a, a_step), (b, b_step)))
        got = layer._meet(a, a_step, b, b_step, rows, size)
        met[got] += 1
        if a == b and (rows == 1 or a_step == b_step):
            assert not got
        elif rows == 1 or a_step == b_step:
            assert got == bool(mine & other), (a, a_step, b, b_step, rows, size)
        else:
            assert got or not mine & other
    assert min(met) > 1000


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("vocab,pad", [(64, 0), (1001, 0), (1001, 7), (20003, 1)])
def test_gradients_between_the_logits_rows(dtype, vocab, pad):
    """Logits and their gradient are the halves of wider rows, in either order."""
    device = cuda_or_skip()
    z, t, c = policy_case(vocab, 9, vocab, dtype)
    given = (t.to(device), c["old_logp"].to(device), c["advantages"].to(device))
    d = random(5, 9).to(device)
    for swapped in (False, True):
        wide = torch.full((9, 2 * vocab + 2 * pad), 3.0, dtype=dtype, device=device)
        halves = wide[:, :vocab], wide[:, vocab + pad:2 * vocab + pad]
        view, out = halves[::-1] if swapped else halves
        view.copy_(z)
        own = torch.empty(9, vocab + 2 * pad + vocab, dtype=dtype, device=device)[:, view.storage_offset():view.storage_offset() + vocab]
        own.copy_(z)
        r, g = layer.policy_loss_gradient(view, *given, out=out)
        want, grad = layer.policy_loss_gradient(own, *given)
        assert torch.equal(g, grad) and torch.equal(r.loss, want.loss) and torch.equal(view.cpu(), z) and (wide[:, vocab:vocab + pad] == 3).all() and (wide[:, 2 * vocab + pad:] == 3).all()
        back = layer.token_logprobs_backward(d, view, t.to(device), r.stats, out=out)
        assert torch.equal(back, layer.token_logprobs_backward(d, own, t.to(device), r.stats)) and torch.equal(view.cpu(), z)
        at = view.storage_offset() - 1 if swapped else 1      # one element beside the logits
        with pytest.raises(ValueError):
            layer.policy_loss_gradient(view, *given, out=wide[:, at:at + vocab])
