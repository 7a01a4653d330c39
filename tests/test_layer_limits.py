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
