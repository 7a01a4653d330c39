"""Tokens whose probability is next to 1: the target's own gradient is what all others have together, by every way to it."""
import pytest
import torch

from superscaler_amd import layer
from tests.layer_reference import SMALLEST, UNIT
from tests.test_layer_loss import BF16, F16, F32, cuda_or_skip

gpu = pytest.mark.gpu


def rows(vocab, rest, dtype):
    """Logits of five rows whose targets lack about `rest` of probability, all other tokens together; and what they lack, in 64 bits."""
    targets = torch.tensor([0, 1, vocab // 2, vocab - 2, vocab - 1])
    low = torch.tensor(rest / (vocab - 1), dtype=torch.float64).log()
    z = low.expand(5, vocab).to(dtype).clone()
    z.scatter_(1, targets[:, None], 0.0)
    others = (vocab - 1) * z[0, 5].double().exp()
    return z, targets, float(others / (1 + others))


def test_refusals_of_the_c_entry():
    lib = layer.load_library()
    a = layer._TOKEN_LOSS.pack(4, 16, 16, 1, 64, 64, 64, 0, 0, 0, 0, 0.0, 1.0, 0.0, 0.25)
    for logp in (None, 64):
        assert lib.ace_token_logprobs_gradient(a, None, logp, 64, 128, 16, None) == -1 and lib.ace_token_logprobs_gradient(a, 64, logp, None, 128, 16, None) == -1
        assert lib.ace_token_logprobs_gradient(a, 64, logp, 64, None, 16, None) == -1 and lib.ace_token_logprobs_gradient(a, 64, logp, 64, 128, 15, None) == -1
    assert lib.ace_token_logprobs_gradient(None, 64, 64, 64, 128, 16, None) == -1


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("vocab", [600, 4099, 51200, 100003, 140001])
@pytest.mark.parametrize("rest", [1e-9, 1e-7, 1e-3])
def test_the_target_s_gradient(vocab, rest, dtype):
    """A lane that has the target adds its other terms to 1 in 32 bits and loses them.  Of 600 elements and more it has a 32nd at most and an element: 64 lanes or more
    with so many pieces each as half of them would not hold, so that the row has 32 times a lane's pieces (600 elements of 16 bits: two pieces of 8 and one element, 17 of
    600, a 35th).  Exponentials of arguments of up to 40 are off by 40 x 2^-23; the result is rounded to its type.  In half precision a loss scale keeps the gradients
    within its range."""
    device = cuda_or_skip()
    z, t, want = rows(vocab, rest, dtype)
    scale = 2.0 ** 15 if dtype is F16 else 1.0
    bound = want * scale * (1 / 32 + 1 / vocab + 40 * 2.0 ** -23 + UNIT[dtype] * 1.01) + SMALLEST[dtype]
    zd, td = z.to(device), t.to(device)
    logp, stats = layer.token_logprobs(zd, td)
    d = torch.full((5,), scale, device=device)
    # (an advantage of -5, five rows: a derivative of 1 by each log-probability; ratios of 1)
    old, A, g = logp.clone(), torch.full((5,), -5.0, device=device), torch.full((1,), scale, device=device)
    for name, got in (("two calls", layer.token_logprobs_backward(d, zd, td, stats, logp=logp)), ("one", layer.policy_loss_gradient(zd, td, old, A, d_loss=g)[1])):
        mine = got.gather(1, td[:, None]).double().cpu()
        assert float((mine - want * scale).abs().max()) <= bound, (name, mine, want * scale)
    without = layer.token_logprobs_backward(d, zd, td, stats)
    mine = without.gather(1, td[:, None]).double().cpu()
    assert float((mine - want * scale).abs().max()) <= bound + scale * 2.0 ** -22
    others = torch.ones_like(z, dtype=torch.bool).scatter_(1, t[:, None], False)
    assert torch.equal(without.cpu()[others], layer.token_logprobs_backward(d, zd, td, stats, logp=logp).cpu()[others])


@gpu
def test_log_probabilities_that_are_no_numbers_and_refusals():
    device = cuda_or_skip()
    z, t = torch.randn(6, 700, device=device, generator=torch.Generator(device=device).manual_seed(1)), torch.arange(6, device=device) * 100
    z[1, 100], z[2], z[3, 5], z[4, 3], t[5] = -torch.inf, -torch.inf, torch.nan, torch.inf, -1
    r, d = layer.token_logprobs(z, t), torch.full((6,), 2.0, device=device)
    with_, without = (layer.token_logprobs_backward(d, z, t, r.stats, logp=x) for x in (r.logp, None))
    assert torch.equal(with_.isnan(), without.isnan()) and float(with_[1, 100]) == 2.0 and (with_[5] == 0).all() and with_[2:5].isnan().any(1).all()
    strided = torch.stack([r.logp, d], 1)[:, 0]
    assert torch.equal(layer.token_logprobs_backward(d, z, t, r.stats, logp=strided)[:2], with_[:2])
    for bad, kind in ((r.logp.double(), TypeError), (r.logp[:5], ValueError), (r.logp.cpu(), ValueError), (1.0, TypeError)):
        with pytest.raises(kind):
            layer.token_logprobs_backward(d, z, t, r.stats, logp=bad)


@gpu
def test_a_policy_s_numbers_are_not_taken_for_log_probabilities():
    """By the C entries: one structure for the policy's loss and for the gradients after it, with the earlier policy's log-probabilities in it."""
    device = cuda_or_skip()
    z, t = torch.randn(5, 900, device=device, generator=torch.Generator(device=device).manual_seed(1)), torch.arange(5, device=device)
    r, old = layer.token_logprobs(z, t), torch.full((5,), -1.0, device=device)
    d, out = torch.ones(5, device=device), torch.empty_like(z)
    a = layer._TOKEN_LOSS.pack(5, 900, 900, 0, 64, z.data_ptr(), t.data_ptr(), old.data_ptr(), d.data_ptr(), 0, 0, 0.8, 1.2, 0.0, 0.2)
    layer._call(device, "ace_token_logprobs_backward", a, d.data_ptr(), r.stats.data_ptr(), out.data_ptr(), 900)
    assert torch.equal(out, layer.token_logprobs_backward(d, z, t, r.stats))
