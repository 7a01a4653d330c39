"""How large a call of the training-layer operators may be: the gradients take what the forward pass takes, a larger call is refused before
anything is launched, and as what it is.  Without a GPU: the library's host part over a stand-in for HIP."""
import types

import pytest
import torch

from superscaler_amd import layer
from tests import layer_host as host


@pytest.mark.parametrize("how", [dict(batch=70000, queries=1, keys=40, heads=2, kv_heads=1, window=8, sinks=3), dict(batch=4, queries=2, keys=40000, heads=64, kv_heads=64, window=8, sinks=36000),
                                 dict(batch=1 << 20, queries=1, keys=128, heads=2, kv_heads=2, window=4, sinks=128)])
def test_attention_with_first_keys(tmp_path, how):
    forward, backward = host.run(tmp_path, [host.call(*host.attend_forward(**how)), host.call(*host.attend_backward(**how))])
    assert forward["rc"] == 0 and backward["rc"] == 0 and backward["launches"] == 3


@pytest.mark.parametrize("how", [dict(batch=1 << 21), dict(batch=1, queries=1 << 28, keys=64, heads=2, kv_heads=1), dict(batch=1, queries=64, keys=1 << 28, heads=2, kv_heads=2)])
def test_attention_that_is_too_large(tmp_path, how):
    how = dict(how, window=8, sinks=3)
    for r in host.run(tmp_path, [host.call(*host.attend_forward(**how)), host.call(*host.attend_backward(**how))]):
        assert r["rc"] == -2 and r["launches"] == 0


def test_too_large_is_a_value_error(monkeypatch):
    lib = layer.load_library()
    monkeypatch.setattr(layer.torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(layer, "_raw_stream", lambda index: None)
    device = types.SimpleNamespace(index=0)
    assert lib.ace_layer_strerror(-2) == b"larger than the kernels hold"
    with pytest.raises(ValueError, match="larger than the kernels hold"):
        layer._call(device, "ace_attend_forward", host.attend(batch=1 << 21), None, 0)
    with pytest.raises(layer.AceError, match="invalid argument"):
        layer._call(device, "ace_attend_forward", host.attend(dim=12), None, 0)


@pytest.mark.gpu
def test_gradients_of_very_many_sequences():
    """More sequences than a grid's second and third dimension hold, against the same in halves: the same kernels, so the same bits."""
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    batch, gen = 70000, torch.Generator(device="cuda").manual_seed(1)
    q, k, v, do = (torch.randn(batch, n, h, 8, device="cuda", generator=gen).bfloat16() for n, h in ((3, 2), (40, 1), (40, 1), (3, 2)))

    def both(part):
        out, lse = layer.window_attention(q[part], k[part], v[part], window=8, sinks=3)
        return layer.window_attention_backward(do[part], q[part], k[part], v[part], out, lse, window=8, sinks=3)
    whole, halves = both(slice(None)), [both(slice(0, batch // 2)), both(slice(batch // 2, batch))]
    for i, g in enumerate(whole):
        assert torch.equal(g, torch.cat([h[i] for h in halves])) and g.any()


@pytest.mark.parametrize("gates", [65533, 65534, 70000, 1 << 24])
def test_norm_with_very_many_gates(tmp_path, gates):
    how = dict(rows=2 * gates, width=8, per_gate=2, gate=host.AT)
    forward, backward = host.run(tmp_path, [host.call(*host.norm_forward(**how)), host.call(*host.norm_backward(**how))])
    assert forward["rc"] == 0 and backward["rc"] == 0 and backward["launches"] == 2


@pytest.mark.gpu
@pytest.mark.parametrize("gates", [65532, 65533, 65534, 140001])
def test_gradients_of_very_many_gates(gates):
    """A gate for every two rows: its gradient is the sum of their two, the same as with a gate for every row."""
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, block, d = (torch.randn(gates, 2, 8, device="cuda", generator=gen) for _ in range(3))
    gate, weight = torch.randn(gates, 8, device="cuda", generator=gen), torch.randn(8, device="cuda", generator=gen)
    stats = layer.block_norm(x, block, gate=gate, exit_weight=weight).stats
    got = layer.block_norm_backward(d, None, x, block, stats, gate=gate, exit_weight=weight)
    rows = layer.block_norm_backward(d, None, x, block, stats, gate=gate[:, None].expand_as(x), exit_weight=weight)
    assert torch.equal(got.x, rows.x) and torch.equal(got.block, rows.block)
    # a product and a sum of two terms in another order: a few units of the larger term; the weight's sum of 2 x gates likewise, of their root
    assert float((got.gate - rows.gate.sum(1)).abs().max()) <= 2.0 ** -21 * float(rows.gate.abs().max())
    assert torch.allclose(got.exit_weight, rows.exit_weight, rtol=1e-4, atol=2.0 ** -20 * (2 * gates) ** 0.5 * float(gate.abs().max()))
