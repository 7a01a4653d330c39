"""Gradients of windowed attention in half precision, whose type has five bits of exponent: whatever the answer's gradient is multiplied
with, they keep their digits, and long sequences' small weights theirs."""
import pytest
import torch

from superscaler_amd import layer
from tests import layer_reference as ref

F16 = torch.float16
UNIT = ref.UNIT[F16]


def normal(seed, *shape, by=1.0):
    return (by * torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)).to(F16)


def off(got, want):
    """The norm of the difference over that of the value."""
    return float((got.double().cpu() - want).norm() / want.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("by", [1e-5, 1e-4, 1e-3, 1.0, 64.0])
@pytest.mark.parametrize("queries,dim,window,sinks,heads", [(300, 64, 40, 3, 8), (600, 128, None, 0, 2), (300, 96, 290, 2, 4), (20, 80, None, 0, 2)])
def test_gradients_of_any_size(by, queries, dim, window, sinks, heads):
    """dS is rounded once, delta comes from a rounded answer, the result is rounded: three roundings of 2^-11 at most, independent of each other; 4
    are allowed.  Small queries and keys under a large scale give gradients that are themselves far from the type's least."""
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    shape = (2, queries, heads, dim)
    q, k, v, do = normal(1, *shape, by=2.0 ** -6), normal(2, *shape, by=2.0 ** -6), normal(3, *shape), normal(4, *shape, by=by)
    how = dict(window=window, sinks=sinks, scale=4096 * dim ** -0.5)
    out, lse = layer.window_attention(*(t.cuda() for t in (q, k, v)), **how)
    got = layer.window_attention_backward(*(t.cuda() for t in (do, q, k, v)), out, lse, **how)
    want = ref.attention(q, k, v, d_out=do, **how)
    for name, g in zip(("dq", "dk", "dv"), got):
        value = want[name][0]
        # (half a step of the type's least numbers, for every element)
        assert float((g.double().cpu() - value).norm()) <= 4 * UNIT * float(value.norm()) + 2.0 ** -25 * value.numel() ** 0.5, name


@pytest.mark.gpu
def test_gradients_of_scores_past_the_types_range():
    """Values of 64 under gradients of 256: products of up to a million meet queries and keys whose own gradients are in range."""
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    q, k, v, do = normal(1, 1, 200, 2, 128, by=64.0), normal(2, 1, 200, 2, 128, by=64.0), normal(3, 1, 200, 2, 128, by=64.0), normal(4, 1, 200, 2, 128, by=256.0)
    how = dict(scale=128 ** -0.5 / 4096)
    out, lse = layer.window_attention(*(t.cuda() for t in (q, k, v)), **how)
    got = layer.window_attention_backward(*(t.cuda() for t in (do, q, k, v)), out, lse, **how)
    want = ref.attention(q, k, v, d_out=do, **how)
    for name, g in zip(("dq", "dk", "dv"), got):
        assert off(g, want[name][0]) <= 4 * UNIT, name


@pytest.mark.gpu
def test_weights_of_a_long_sequence():
    """Queries of zeros weigh all that they see alike, the last of 262,144 with 2^-18: dV is a running sum."""
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    n = 1 << 18
    q, k, v = (torch.zeros(1, n, 1, 64, dtype=F16, device="cuda") for _ in range(3))
    do = (256 * torch.randn(1, n, 1, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))).half()
    out, lse = layer.window_attention(q, k, v)
    dv = layer.window_attention_backward(do, q, k, v, out, lse)[2]
    terms = do[0, :, 0].double() / torch.arange(1, n + 1, device="cuda", dtype=torch.float64)[:, None]
    want = terms.flip(0).cumsum(0).flip(0)
    late = slice(n // 2, n - 1024)
    # one rounding of a weight, one of the result, independent; and sums of 2^17 terms in 32 bits, of which those of a block are added first
    assert float((dv[0, late, 0].double() - want[late]).norm() / want[late].norm()) <= 2 * UNIT
