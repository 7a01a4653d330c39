"""Attention among values that are no finite numbers: what a query does not see does not reach it, what it sees does.  The reference takes every
product by itself and leaves those of hidden pairs out, in 64 bits."""
import math

import pytest
import torch

from superscaler_amd import layer
from tests import layer_reference as ref

BF16, F16 = torch.bfloat16, torch.float16
NAN, INF = math.nan, math.inf


def over(weights, values, seen):
    """sum over j of weights[i, j] values[j], of the pairs that are seen, for every batch and head."""
    out = torch.empty(*weights.shape[:3], values.shape[-1], dtype=torch.float64)
    for b in range(weights.shape[0]):
        for h in range(weights.shape[1]):
            out[b, h] = torch.where(seen[b, :, :, None], weights[b, h, :, :, None] * values[b, h, None], 0.0).sum(1)
    return out


def reference(q, k, v, do, window=None, sinks=0, start=None, lengths=None):
    shared, scale = q.shape[2] // k.shape[2], 1 / math.sqrt(q.shape[3])
    seen = ref.visible(q.shape[0], q.shape[1], k.shape[1], window, sinks, start, lengths)
    q, k, v, do = (t.double().transpose(1, 2) for t in (q, k, v, do))
    kx, vx = k.repeat_interleave(shared, 1), v.repeat_interleave(shared, 1)
    mask = seen[:, None]
    s = torch.where(mask, q @ kx.transpose(2, 3) * scale, -INF)      # (a row of the product goes by its own key only)
    top = s.amax(-1, keepdim=True)
    lse = torch.where(top == -INF, top, top + (s - torch.where(top == -INF, 0.0, top)).exp().sum(-1, keepdim=True).log())
    p = torch.where(mask, (s - torch.where(lse == -INF, 0.0, lse)).exp(), 0.0)
    out = over(p, vx, seen)
    dp = do @ vx.transpose(2, 3)
    ds = torch.where(mask, p * (dp - (do * out).sum(-1, keepdim=True)), 0.0)
    flip = seen.transpose(1, 2)

    def kv(t):
        return t.unflatten(1, (-1, shared)).sum(2).transpose(1, 2)
    return {"out": out.transpose(1, 2), "lse": lse[..., 0], "dq": scale * over(ds, kx, seen).transpose(1, 2), "dk": scale * kv(over(ds.transpose(2, 3), q, flip)),
            "dv": kv(over(p.transpose(2, 3), do, flip))}


def check(q, k, v, do, exact=("out", "lse"), **how):
    """`exact`: results whose infinities are the reference's; of the others, gradients that infinities went into, what is not finite there is not finite here."""
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    dev = {n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in how.items()}
    gpu = [t.cuda() for t in (q, k, v)]
    out, lse = layer.window_attention(*gpu, **dev)
    got = {"out": out, "lse": lse}
    if do is not None:
        got.update(zip(("dq", "dk", "dv"), layer.window_attention_backward(do.cuda(), *gpu, out, lse, **dev)))
        again = layer.window_attention_backward(do.cuda(), *gpu, out, lse, **dev)
        assert all(torch.equal(got[n].nan_to_num(), a.nan_to_num()) for n, a in zip(("dq", "dk", "dv"), again))
    if q.shape[0] > 2 and "start" not in how:      # (of many sequences the first and the last)
        pick = [0, -1]
        q, k, v, do = (None if t is None else t[pick] for t in (q, k, v, do))
        got = {n: t[pick] for n, t in got.items()}
    want = reference(q, k, v, torch.zeros_like(q) if do is None else do, **how)
    tame = [None if t is None else torch.where(t.isfinite(), t, 0.0) for t in (q, k, v, do)]
    bound = ref.attention(*tame[:3], d_out=tame[3], unit=ref.UNIT[q.dtype], **how)
    counts = {}
    for n, g in got.items():
        value, slack = want[n], bound[n][1] + 64 * ref.SMALLEST[q.dtype]
        counts[n] = int((~value.isfinite()).sum()), value.numel()
        if n not in exact:
            g = g.cpu()
            assert torch.equal(g.isfinite(), value.isfinite()), n
            g, value, slack = (t[value.isfinite()] for t in (g, value, slack))
        ref.close(g, value, slack)
    return counts


def tensors(seed, batch, queries, keys, heads, kv_heads, dim, dtype):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(batch, n, h, dim, generator=gen, dtype=torch.float64).to(dtype) for n, h in ((queries, heads), (keys, kv_heads), (keys, kv_heads), (queries, heads))]


@pytest.mark.gpu
@pytest.mark.parametrize("dim,dtype", [(64, BF16), (64, F16), (88, BF16), (128, BF16), (128, F16)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (70, 0), (70, 3), (40, 40)])
def test_values_of_a_prompt(dim, dtype, window, sinks):
    """Values of whole keys, of single elements, both infinities in one channel, and in a first key."""
    q, k, v, _ = tensors(1, 2, 300, 300, 4, 2, dim, dtype)
    v[0, 150] = NAN
    v[0, 230, 1, 5], v[0, 244, 1, 5], v[0, 237, 1, 6] = INF, -INF, -INF
    v[1, 1, 0, 3], v[1, 299, :, 7], v[1, 64, 1, 0] = INF, NAN, -INF
    counts = check(q, k, v, None, window=window, sinks=sinks)
    assert 0 < counts["out"][0] < counts["out"][1]


@pytest.mark.gpu
@pytest.mark.parametrize("queries,keys,heads,kv_heads", [(1, 700, 8, 2), (5, 900, 8, 2), (16, 1000, 4, 1), (1, 40, 2, 2), (3, 9000, 2, 2), (33, 200, 40, 40)])
@pytest.mark.parametrize("dim,dtype", [(64, F16), (96, BF16), (128, BF16)])
def test_values_of_a_cache(queries, keys, heads, kv_heads, dim, dtype):
    """A sliding window over a cache whose places outside hold what is no number."""
    q, k, v, _ = tensors(2, 2, queries, keys, heads, kv_heads, dim, dtype)
    window = 33
    v[:, 4:keys - queries - window + 1], k[:, 4:keys - queries - window + 1] = NAN, INF
    assert check(q, k, v, None, window=window, sinks=4)["out"][0] == 0
    v[0, keys - window, :, 1], v[1, 2, :, 2] = INF, NAN
    counts = check(q, k, v, None, window=window, sinks=4)
    assert 0 < counts["out"][0] < counts["out"][1]


@pytest.mark.gpu
def test_values_past_the_length_and_of_sequences_without_keys():
    q, k, v, do = tensors(3, 4, 150, 200, 4, 2, 64, BF16)
    lengths = torch.tensor([0, 1, 130, 200], dtype=torch.int32)
    for b, n in enumerate(lengths.tolist()):
        k[b, n:], v[b, n:] = NAN, INF
    v[2, 129, 0], v[3, 60, 1, 9] = NAN, INF
    do[3, 100] = NAN
    check(q, k, v, do, start=torch.tensor([0, 0, -20, 50], dtype=torch.int32), lengths=lengths, window=90, sinks=2, exact=("out", "lse"))


@pytest.mark.gpu
@pytest.mark.parametrize("batch,heads,kv_heads,dim,dtype", [(1, 4, 2, 128, BF16), (1, 4, 2, 64, F16), (6, 8, 8, 96, BF16), (19, 8, 8, 64, BF16), (19, 8, 8, 128, F16)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 3)])
def test_gradients(batch, heads, kv_heads, dim, dtype, window, sinks):
    """A query, a key, a value and an answer's gradient each: with key blocks of 32, 64 and 128 keys per workgroup."""
    for which, at, what in ((0, 180, NAN), (1, 100, NAN), (2, 100, NAN), (3, 180, NAN), (3, 170, INF)):
        t = tensors(4 + which, batch, 260, 260, heads, kv_heads, dim, dtype)
        if what is INF:
            t[which][:, at, 0, 3] = INF
        else:
            t[which][-1, at, -1] = NAN
        counts = check(*t, window=window, sinks=sinks, exact=("out", "lse", "dv") if which == 3 else ("out", "lse"))
        touched = {n: c for n, c in counts.items() if c[0]}
        assert touched and all(c[0] < c[1] for c in touched.values()), (which, counts)


@pytest.mark.gpu
def test_gradients_of_first_keys():
    """Queries beyond the window of the first keys, whose gradients are split over workgroups; one that begins behind every key."""
    q, k, v, do = tensors(9, 2, 300, 300, 4, 2, 64, BF16)
    q[0, 20, 1], q[0, 222], do[1, 260, 0, 3] = NAN, NAN, -INF
    check(q, k, v, do, window=16, sinks=40, exact=("out", "lse", "dv"))


@pytest.mark.gpu
def test_all_values_are_no_numbers():
    q, k, v, do = tensors(11, 1, 500, 500, 2, 1, 128, BF16)
    counts = check(q, k, v * NAN, do, exact=("out", "lse"))
    assert counts["out"][0] == counts["out"][1] and counts["lse"][0] == 0
