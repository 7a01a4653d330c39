"""Rows of many millions of logits: a lane's sum over its part of a row loses nothing."""
import pytest
import torch

from superscaler_amd import layer
from tests.layer_reference import SMALLEST, close
from tests.test_layer_loss import BF16, E24, F16, F32, cuda_or_skip

gpu = pytest.mark.gpu


def exact(z):
    """log sum exp of a row around its largest, in 64 bits."""
    top = float(z.max())
    return torch.stack([(part.double() - top).exp().sum() for part in z.split(1 << 24)]).sum().log().cpu() + top


@gpu
@pytest.mark.parametrize("vocab,dtype", [(5_000_001, F32), (20_000_003, F32), (40_000_007, BF16), (1 << 28, F16)])
@pytest.mark.parametrize("spread", [0.0, 1.5])
def test_sums_of_a_very_large_row(vocab, dtype, spread):
    """A term is off by its exponential: two roundings of an argument of up to 2 and one of 2^-23.  32 of them are added in 32 bits; where a lane's largest
    grows, and where lanes are joined, an exponential more each.  Beside that there is what the result itself is rounded by."""
    device = cuda_or_skip()
    gen = torch.Generator(device=device).manual_seed(vocab)
    z = torch.empty(1, vocab, dtype=dtype, device=device)
    z.fill_(-0.3)
    if spread:
        z[0, ::7], z[0, 3::11] = -spread, -0.7
        z[0, :1000] = -spread * torch.rand(1000, device=device, generator=gen).to(dtype)
    z[0, vocab // 3] = 0.0
    t = torch.tensor([vocab // 5], device=device)
    logp, stats = layer.token_logprobs(z, t)
    bound = E24 * (32 + 2 * 2 + 2 + 4 * 4)
    want = (z[0, t[0]].double().cpu() - exact(z[0])).view(1)
    close(logp, want, torch.full((1,), bound, dtype=torch.float64))
    d = torch.full((1,), float(2.0 ** 20), device=device)      # (a scale that keeps what is shared by millions within the type)
    at = torch.randint(0, vocab, (5000,), device=device, generator=gen)
    at = at[at != t[0]]
    g = layer.token_logprobs_backward(d, z, t, stats, logp=logp)[0, at]
    p = (z[0, at].double().cpu() - exact(z[0])).exp() * 2.0 ** 20
    close(g, -p, p * (2 * bound + 8 * E24) + SMALLEST[dtype])
