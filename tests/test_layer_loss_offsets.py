"""Gradients of logits whose rows lie far from zero: what all logits of a row share does not reach its gradient.  Bounds as in test_layer_loss."""
import pytest
import torch

from superscaler_amd import layer
from tests.layer_reference import SMALLEST, close
from tests.test_layer_loss import BF16, E24, F16, F32, check_policy, cuda_or_skip, logp_bound, logprobs, random

gpu = pytest.mark.gpu


def given(z, targets, seed):
    """A policy's numbers for these logits."""
    rows, logp = z.shape[0], logprobs(z, targets)[0]
    return z, targets, dict(old_logp=(logp + random(seed + 2, rows, by=0.3)).float(), advantages=random(seed + 4, rows), ref_logp=(logp + random(seed + 3, rows, by=0.4)).float(),
                            weights=(0.1 + torch.rand(rows, generator=torch.Generator().manual_seed(seed + 5))) / rows)


def two_calls_agree(device, z, targets, c):
    """The gradient that comes along is the one of the two calls: both are rounded, and their log-probabilities are a bound apart each."""
    zd, td, old, A = (t.to(device) for t in (z, targets, c["old_logp"], c["advantages"]))
    how = dict(ref_logp=c["ref_logp"].to(device), weights=c["weights"].to(device), kl_weight=0.1)
    r, grad = layer.policy_loss_gradient(zd, td, old, A, **how)
    two = layer.token_logprobs_backward(r.d_logp, zd, td, r.stats)
    slack = two.double().abs() * (torch.finfo(z.dtype).eps / 2 + 4 * logp_bound(z)) + r.d_logp.double().abs()[:, None] * 4 * E24 + 2 * SMALLEST[z.dtype]
    close(grad, two.double(), slack)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("vocab", [1000, 20000])
def test_rows_of_one_value(dtype, vocab):
    """A mask that leaves nothing, with any of the values that masks are made of; and very large logits."""
    device = cuda_or_skip()
    info = torch.finfo(dtype)
    values = [v for v in (-1e4, -1e9, -1e30, 1e4, 1e5, -1e6, 1e7, 65504.0, 30.0, -0.125, info.min, info.max) if info.min <= v <= info.max]
    z = torch.tensor(values, dtype=torch.float64).to(dtype)[:, None].repeat(1, vocab)
    targets = torch.arange(len(values)) * 7 % vocab
    args = given(z, targets, vocab)
    check_policy(device, *args)
    two_calls_agree(device, *args)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("offset", [30.0, 100.0, -1000.0, 1e4, -6e4, 1e6, -1e7])
def test_rows_far_from_zero(dtype, offset):
    """Logits a few steps of their type apart, but no more than some 8 from each other where the type has such steps."""
    device = cuda_or_skip()
    if abs(offset) > torch.finfo(dtype).max:
        pytest.skip("not a number of this type")
    gen = torch.Generator().manual_seed(int(abs(offset)))
    base = torch.tensor(offset, dtype=torch.float64).to(dtype).double()
    step = float(base.abs()) * torch.finfo(dtype).eps
    apart = max(1, min(1000, int(8 / step)))
    z = (base + torch.randint(0, apart + 1, (9, 5001), generator=gen).double() * step).to(dtype)
    targets = torch.randint(0, 5001, (9,), generator=gen)
    args = given(z, targets, 3)
    check_policy(device, *args)
    two_calls_agree(device, *args)
