"""Making a packing waits for nothing, and calls on any stream find its table."""
import pytest
import torch

from superscaler_amd import layer
from superscaler_amd.evaluator import AceError
from tests.test_layer_packed import case, cuda_or_skip
from tests.test_layer_packing_memory import busy

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("lengths", [[300, 5, 64, 260], [7] * 3000])
def test_a_packing_is_made_while_the_card_is_at_work(lengths):
    """Its queues are as full afterwards, and the packing is there for any stream at once."""
    device = cuda_or_skip()
    q, k, v, _ = (t.to(device) for t in case(3, sum(lengths), 2, 1, 64))
    want = layer.packed_attention(q, k, v, layer.Packing(lengths))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    others = [torch.cuda.Stream() for _ in range(6)]      # (more than there are hardware queues)
    fills = [torch.empty(1 << 26, device=device) for _ in others]
    busy()
    done = [torch.cuda.Event()]
    done[0].record()
    for s, x in zip(others, fills):
        with torch.cuda.stream(s):
            for _ in range(200):
                x.fill_(1.0)
            done.append(s.record_event())
    packing = layer.Packing(lengths)
    assert not done[0].query() and not done[-1].query()
    with torch.cuda.stream(side):
        got = layer.packed_attention(q, k, v, packing)
    here = layer.packed_attention(q, k, v, packing)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in (got, here) for a, b in zip(r, want))


@gpu
def test_tables_of_many_packings_do_not_meet():
    """Made one after the other under queued work, each dropped once it was used: every call reads its own."""
    device = cuda_or_skip()
    q, k, v, _ = (t.to(device) for t in case(5, 700, 2, 1, 64))
    cuts = [[i, 700 - i] for i in range(1, 700, 23)]
    want = [layer.packed_attention(q, k, v, layer.Packing(c)) for c in cuts]
    torch.cuda.synchronize()
    busy(20)
    got = [layer.packed_attention(q, k, v, layer.Packing(c)) for c in cuts]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


def test_not_while_a_graph_is_captured(monkeypatch):
    monkeypatch.setattr(layer.torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(AceError, match="before the graph"):
        layer.Packing([3], device="cuda:0")
