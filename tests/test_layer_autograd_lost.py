"""Where automatic differentiation would lose a gradient of the packed step's operators, it is told, and what to call instead."""
import pytest
import torch
from torch.autograd import forward_ad

from superscaler_amd import layer
from superscaler_amd.evaluator import AceError

gpu = pytest.mark.gpu


def cuda_or_skip():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


@pytest.mark.parametrize("name", ["block_norm", "window_attention", "packed_attention", "token_logprobs", "policy_loss", "gradient_norm"])
def test_the_message_names_calls_that_are_there(name):
    a = torch.ones(3, requires_grad=True)
    made, = layer._untracked(name, (torch.ones(2),), (a,))
    with pytest.raises(AceError) as e:
        made.sum().backward()
    words = [w.strip("():") for w in str(e.value).split() if "_" in w and "." not in w]
    assert name in words and all(hasattr(layer, w) for w in words)


def test_what_is_changed_in_place_is_told():
    """Without a GPU: tensors with a graph and those that depend on them; leaves and views of what has none stay as they are."""
    a = torch.ones(3, requires_grad=True)
    g, plain, whole = a * 2, torch.ones(3), torch.ones(4)
    with torch.no_grad():
        part = whole[:3]
    layer._untracked_in_place("clip_gradients", [g, plain, part, a], [g, a])
    for t in (g, plain):
        with pytest.raises(AceError, match="clip_gradients"):
            t.sum().backward()
    assert not part.requires_grad and a.is_leaf
    with pytest.raises(AceError, match="no_grad"):
        layer._untracked_in_place("clip_gradients", [(a * 2).split(1)[0]], [a])


@gpu
def test_clipped_gradients_that_carry_a_graph():
    """As with gradient_norm, going backward through what comes back, or through what was clipped, is an error; the values are as without a graph."""
    device = cuda_or_skip()
    x = torch.arange(1.0, 11.0, device=device, requires_grad=True)

    def fresh():
        y = torch.ones(5, device=device)
        return [torch.autograd.grad((x ** 3).sum(), x, create_graph=True)[0], y]
    with torch.no_grad():
        want = [t.detach() for t in [3 * x ** 2, torch.ones(5, device=device)]]
        r0 = layer.clip_gradients(want, 0.5)
        assert not any(t.requires_grad for t in r0)
    for through in (lambda g, r: r.norm.sum(), lambda g, r: r.scale.sum(), lambda g, r: r.norms.sum(), lambda g, r: g[0].sum(), lambda g, r: g[1].sum()):
        grads = fresh()
        r = layer.clip_gradients(grads, 0.5)
        assert all(torch.equal(a, b) for a, b in zip(grads, want)) and all(torch.equal(a, b) for a, b in zip(r, r0))
        with pytest.raises(AceError, match="clip_gradients"):
            through(grads, r).backward()
    scale = torch.ones(1, device=device, requires_grad=True)
    with pytest.raises(AceError, match="clip_gradients"):
        layer.clip_gradients([torch.ones(5, device=device)], 0.5, grad_scale=scale).norm.backward()
    p = torch.ones(5, device=device, requires_grad=True)      # a leaf has no graph to lose
    layer.clip_gradients([p], 0.5)
    assert p.is_leaf and float(p.detach().norm()) < 0.51


@gpu
def test_a_policy_s_gradient_is_not_gone_through():
    """Second derivatives are lost, whichever input they are by; the logits' own graph still takes the gradient, also where they hold it."""
    device = cuda_or_skip()
    gen = torch.Generator(device=device).manual_seed(1)
    w = torch.randn(8, 64, device=device, generator=gen)
    h, t, old, A = torch.randn(6, 8, device=device, generator=gen), torch.arange(6, device=device), torch.full((6,), -4.0, device=device), torch.ones(6, device=device)
    want = layer.policy_loss_gradient(h @ w, t, old, A)[1]
    for in_place in (False, True):
        p = w.clone().requires_grad_()
        logits = h @ p
        r, g = layer.policy_loss_gradient(logits, t, old, A, out=logits if in_place else None)
        assert torch.equal(g, want) and (not in_place or g.data_ptr() == logits.data_ptr())
        with pytest.raises(AceError, match="policy_loss_gradient"):
            g.sum().backward(retain_graph=True)
        g.mul_(2.0)             # a program's own work on it
        logits.backward(g)
        assert torch.equal(p.grad, h.t() @ (2 * want))
    given = dict(logits=h @ w, targets=t, old_logp=old, advantages=A, ref_logp=old + 0.1, weights=A / 6, d_loss=torch.ones(1, device=device))
    for name in ("logits", "old_logp", "advantages", "ref_logp", "weights", "d_loss"):
        how = dict(given, **{name: given[name].clone().requires_grad_()})
        for each in layer.policy_loss_gradient(**how, kl_weight=0.1)[1], layer.policy_loss_gradient(**how, kl_weight=0.1)[0].loss:
            with pytest.raises(AceError):
                each.sum().backward()
        with torch.no_grad():
            assert not layer.policy_loss_gradient(**how, kl_weight=0.1)[1].requires_grad


@gpu
def test_a_factor_that_has_a_gradient():
    device = cuda_or_skip()
    scale = torch.ones(1, device=device, requires_grad=True)
    for result in layer.gradient_norm([torch.ones(5, device=device)], max_norm=0.5, grad_scale=scale):
        with pytest.raises(AceError, match="gradient_norm"):
            result.sum().backward()


def test_tangents():
    """Without a GPU: what carries one is refused before anything else is looked at."""
    x, d = torch.ones(2, 4), torch.ones(2, 4)
    layer._no_tangents(x, None)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, d)
        layer._no_tangents(x, None)
        with pytest.raises(AceError, match="forward-mode"):
            layer._no_tangents(None, x, dual)
        t, f, other = torch.zeros(2, dtype=torch.int64), torch.zeros(2), forward_ad.make_dual(torch.zeros(2), torch.ones(2))
        packing = object.__new__(layer.Packing)
        for call in (lambda: layer.block_norm(dual, entry_weight=x[0]), lambda: layer.block_norm(x, dual, entry_weight=x[0]), lambda: layer.window_attention(x, dual, x),
                     lambda: layer.packed_attention(x, x, dual, packing), lambda: layer.token_logprobs(dual, t), lambda: layer.policy_loss(x, t, other, f),
                     lambda: layer.policy_loss_gradient(x, t, f, f, weights=other), lambda: layer.gradient_norm([x, dual]), lambda: layer.clip_gradients([dual], 1.0),
                     lambda: layer.token_logprobs_backward(f, dual, t, x)):
            with pytest.raises(AceError, match="forward-mode"):
                call()
        layer._no_tangents(forward_ad.unpack_dual(dual).primal)
    layer._no_tangents(x)


@gpu
def test_tangents_on_the_gpu():
    """Of the tensors that come in beside the first ones; a call without any is as it is outside."""
    device = cuda_or_skip()
    z, t, f = torch.randn(4, 30, device=device), torch.arange(4, device=device), torch.full((4,), -3.0, device=device)
    one, q = torch.ones(1, device=device), torch.ones(6, 2, 64, dtype=torch.bfloat16, device=device)
    packing = layer.Packing([6])
    out, lse = layer.packed_attention(q, q, q, packing)
    stats, want = layer.token_logprobs(z, t).stats, layer.policy_loss_gradient(z, t, f, f, d_loss=one)[1]
    with forward_ad.dual_level():
        def dual(x):
            return forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: layer.packed_attention_backward(dual(q), q, q, q, out, lse, packing), lambda: layer.token_logprobs_backward(dual(f), z, t, stats),
                     lambda: layer.policy_loss_gradient(z, t, f, f, d_loss=dual(one)), lambda: layer.gradient_norm([z], grad_scale=dual(one)),
                     lambda: layer.clip_gradients([z], 1.0, grad_scale=dual(one)), lambda: layer.window_attention_backward(*[dual(q[None])] + [q[None]] * 4, lse[None])):
            with pytest.raises(AceError, match="forward-mode"):
                call()
        assert torch.equal(layer.policy_loss_gradient(z, t, f, f, d_loss=one)[1], want)
