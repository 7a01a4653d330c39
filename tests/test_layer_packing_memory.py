"""A packing's table and those who use it: other streams, and a packing that goes away while they are at work."""
import contextlib
import copy
import gc
import pickle
import types

import pytest
import torch

from superscaler_amd import layer
from tests.test_layer_packed import case, cuda_or_skip

gpu = pytest.mark.gpu


def busy(ms=60):
    """Work for the current stream that takes some `ms` at least."""
    x = torch.empty(1 << 28, device="cuda")
    for _ in range(ms * 8):     # (1 GiB takes more than an eighth of a millisecond to fill)
        x.fill_(1.0)


def test_a_table_is_kept_for_every_stream_that_uses_it(monkeypatch):
    """Without a GPU: a call on a stream that is not the table's tells the allocator so and goes behind its copy, once, before anything is launched."""
    asked = []
    current = types.SimpleNamespace(cuda_stream=7, wait_event=lambda e: asked.append(("wait", e)))
    p = object.__new__(layer.Packing)
    p.device, p._args, p._streams, p._made = torch.device("cuda:0"), b"args", {3}, "made"
    p._table = types.SimpleNamespace(record_stream=lambda s: asked.append(("record", s.cuda_stream)))
    monkeypatch.setattr(layer.torch.cuda, "current_stream", lambda index: current)
    monkeypatch.setattr(layer.torch.cuda, "device", lambda index: contextlib.nullcontext())
    monkeypatch.setattr(layer.torch.cuda, "is_current_stream_capturing", lambda: True)
    monkeypatch.setattr(layer, "_raw_stream", lambda index: 3)
    assert p._used() == b"args" and asked == []
    monkeypatch.setattr(layer, "_raw_stream", lambda index: current.cuda_stream)
    assert p._used() == b"args" and asked == [("record", 7)]       # a captured call cannot wait: its caller orders it
    monkeypatch.setattr(layer.torch.cuda, "is_current_stream_capturing", lambda: False)
    assert p._used() == b"args" and p._used() == b"args" and asked == [("record", 7), ("record", 7), ("wait", "made")]


def test_a_copied_packing_has_a_table_of_its_own(monkeypatch):
    """Without a GPU: copies and pickles are made from the lengths, not from the address that the first one's arguments hold."""
    made = []
    monkeypatch.setattr(layer.Packing, "__init__", lambda self, lengths, **how: made.append((lengths, how)))
    p = object.__new__(layer.Packing)
    p.lengths, p.tokens, p.device, p._args = (3, 0, 4), 9, torch.device("cuda:0"), b"an address"
    for other in (copy.copy(p), copy.deepcopy(p), pickle.loads(pickle.dumps(p))):
        assert not hasattr(other, "_args")
    assert made == [((3, 0, 4), dict(tokens=9, device="cuda:0"))] * 3


@gpu
def test_a_copied_packing_is_as_good():
    device = cuda_or_skip()
    q, k, v, _ = (t.to(device) for t in case(4, 300, 2, 1, 64))
    packing = layer.Packing([100, 0, 150], tokens=300)
    want, others = layer.packed_attention(q, k, v, packing), [copy.deepcopy(packing), pickle.loads(pickle.dumps(packing))]
    del packing
    gc.collect()
    for other in others:
        assert other.lengths == (100, 0, 150) and all(torch.equal(a, b) for a, b in zip(layer.packed_attention(q, k, v, other), want))


@gpu
def test_a_packing_that_goes_away_under_another_stream_s_work():
    """Its table's memory is not handed out before that work is done."""
    device = cuda_or_skip()
    q, k, v, do = (t.to(device) for t in case(3, 640, 4, 2, 64))
    lengths = [300, 5, 64, 260]

    def both(packing):
        out, lse = layer.packed_attention(q, k, v, packing, window=50, sinks=3)
        return (out, lse) + layer.packed_attention_backward(do, q, k, v, out, lse, packing, window=50, sinks=3)
    want = both(layer.Packing(lengths, tokens=640))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    packing = layer.Packing(lengths, tokens=640)
    place, size = packing._table.data_ptr(), packing._table.numel()
    with torch.cuda.stream(side):
        busy()
        got = both(packing)
        done = torch.cuda.Event()
        done.record()
    del packing
    others = [torch.full((size,), 1 << 20, dtype=torch.int32, device=device) for _ in range(64)]
    early = not done.query()
    assert early and all(t.data_ptr() != place for t in others)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
