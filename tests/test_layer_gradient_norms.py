"""Attention's answers and gradients by the norm of their error, head by head: element by element the bounds on bfloat16 gradients are about as large
as the gradients, as they add up what rounding may do at worst."""
import pytest
import torch

from superscaler_amd import layer
from tests import layer_reference as ref

BF16, F16 = torch.bfloat16, torch.float16
# (batch, queries, keys, heads, kv_heads, dim, type, window, sinks, ragged)
CASES = [(2, 270, 270, 8, 2, 128, BF16, None, 0, False), (2, 270, 270, 8, 2, 128, BF16, 100, 3, False), (2, 300, 300, 4, 4, 64, BF16, 64, 0, False),
         (3, 200, 333, 6, 3, 96, BF16, None, 0, False), (1, 900, 900, 2, 1, 128, BF16, None, 0, False), (1, 900, 900, 40, 40, 64, BF16, 256, 40, False),
         (4, 260, 260, 4, 1, 80, BF16, 120, 1, True), (2, 270, 270, 8, 2, 128, F16, 100, 3, False), (4, 260, 260, 4, 1, 64, F16, None, 0, True), (64, 130, 130, 8, 8, 64, BF16, None, 0, False)]


def inputs(case, seed=7):
    batch, queries, keys, heads, kv_heads, dim, dtype, window, sinks, ragged = case
    gen = torch.Generator().manual_seed(seed)
    q, k, v, do = (torch.randn(batch, n, h, dim, generator=gen, dtype=torch.float64).to(dtype) for n, h in ((queries, heads), (keys, kv_heads), (keys, kv_heads), (queries, heads)))
    how = dict(window=window, sinks=sinks)
    if ragged:
        how.update(lengths=torch.tensor([keys, keys // 2, 1, 77][:batch], dtype=torch.int32), start=torch.zeros(batch, dtype=torch.int32))
    return q, k, v, do, how


def beyond(got, want, unit):
    """Heads' error over what is allowed, at most: weights (or their gradients), the answer that delta goes by and the result are rounded once
    each, by `unit` at most and half of it in the mean square, independently: the root of three halves, below one unit.  Two are allowed, and
    what 32-bit arithmetic leaves where terms cancel, as with one key, whose weight cannot change.  `want`: a value and that bound."""
    got, (want, slack) = got.double().cpu(), want
    error, size, slack = ((t * t).sum((1, 3)).sqrt() for t in (got - want, want, slack))      # [batch, heads]
    return float((error / (2 * unit * size + slack).clamp(min=2.0 ** -60)).amax())


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_errors_by_norm(case):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    q, k, v, do, how = inputs(case)
    dev = {n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in how.items()}
    out, lse = layer.window_attention(*(t.cuda() for t in (q, k, v)), **dev)
    got = dict(zip(("dq", "dk", "dv"), layer.window_attention_backward(*(t.cuda() for t in (do, q, k, v)), out, lse, **dev)), out=out)
    want = ref.attention(q, k, v, d_out=do, **how)
    assert {n: b for n, g in got.items() if not (b := beyond(g, want[n], ref.UNIT[q.dtype])) <= 1} == {}


@pytest.mark.parametrize("case", [c for c in CASES if c[6] is BF16 and c[0] < 64 and c[3] < 40], ids=str)
def test_what_the_norm_shows(case):
    """Planted in the reference: gradients 2% too large, and a reference whose queries do not see their own key or whose window is one too short."""
    q, k, v, do, how = inputs(case)
    want = ref.attention(q, k, v, d_out=do, **how)
    unit = ref.UNIT[q.dtype]
    less = dict(how, window=how["window"] - 1) if how["window"] else dict(how, start=torch.full((case[0],), case[2] - case[1] - 1, dtype=torch.int32))
    short = ref.attention(q, k, v, d_out=do, **less)
    for n in ("out", "dq", "dk", "dv"):
        value = want[n][0]
        assert beyond(value.to(q.dtype), want[n], unit) <= 1
        assert beyond(value * 1.02, want[n], unit) > 1, n
        assert beyond(short[n][0], want[n], unit) > 1, n
