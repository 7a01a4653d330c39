"""Automatic differentiation knows nothing of the training-layer operators, and says so where a gradient would be lost."""
import pytest
import torch

from superscaler_amd import layer
from superscaler_amd.evaluator import AceError


def cuda_or_skip():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")


def test_results_that_cannot_be_gone_through():
    a, b = torch.ones(3, requires_grad=True), torch.ones(3)
    out, lse = torch.ones(2), torch.ones(2)
    assert layer._lost(None, b, a) and not layer._lost(b, None)
    with torch.no_grad():
        assert not layer._lost(a)
    got = layer._untracked("window_attention", (out, None, lse), (a, b, None))
    assert got[1] is None and got[0].requires_grad and got[2].requires_grad and got[0].data_ptr() == out.data_ptr()
    with pytest.raises(AceError, match="window_attention_backward"):
        (got[0] * 2).sum().backward()


@pytest.mark.gpu
def test_a_lost_gradient_is_an_error():
    cuda_or_skip()
    x, block, w = (torch.ones(*s, device="cuda") for s in ((2, 8), (2, 8), (8,)))
    plain = layer.block_norm(x, block, entry_weight=w)
    assert not plain.normed.requires_grad
    for which in range(3):
        args = [t.clone().requires_grad_(i == which) for i, t in enumerate((x, block, w))]
        r = layer.block_norm(args[0], args[1], entry_weight=args[2])
        assert torch.equal(r.normed, plain.normed) and torch.equal(r.residual, plain.residual) and torch.equal(r.stats, plain.stats)
        with pytest.raises(AceError, match="block_norm_backward"):
            r.normed.sum().backward()
        with torch.no_grad():
            assert not layer.block_norm(args[0], args[1], entry_weight=args[2]).normed.requires_grad
        g = layer.block_norm_backward(x, x, args[0], args[1], r.stats, entry_weight=args[2])      # gradients by hand
        assert not g.x.requires_grad
    p = x.clone().requires_grad_()
    r = layer.block_norm(p, entry_weight=w)
    assert r.residual is p
    with pytest.raises(AceError):
        r.normed.sum().backward()
    q = torch.ones(1, 4, 2, 64, dtype=torch.bfloat16, device="cuda")
    leaf = q.clone().requires_grad_()
    for a in ((leaf, q, q), (q, leaf, q), (q, q, leaf * 1)):
        out, lse = layer.window_attention(*a)
        assert torch.equal(out, layer.window_attention(q, q, q)[0])
        with pytest.raises(AceError, match="window_attention_backward"):
            out.float().sum().backward()


@pytest.mark.gpu
def test_a_step_counts_as_a_change_in_place():
    """A graph that has kept a parameter or its copy refuses to go backward with other values."""
    cuda_or_skip()
    p = torch.nn.Parameter(torch.ones(4, device="cuda"))
    copy = p.detach().bfloat16().requires_grad_()
    for t in (p, copy):
        opt = layer.AdamW([p], copies=[copy])
        loss = (t * t).sum()
        opt.step([torch.ones(4, device="cuda")], lr=0.1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
