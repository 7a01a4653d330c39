"""Attention over sequences that lie one after the other against each sequence by itself in 64 bits (layer_reference.attention); without a GPU: the
table of blocks, the launches, what is refused."""
import ctypes
import math
import random as pyrandom

import numpy as np
import pytest
import torch

from superscaler_amd import layer
from superscaler_amd.evaluator import AceError
from tests import layer_host as host
from tests import layer_reference as ref

gpu = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
NAN, INF = math.nan, math.inf


def cuda_or_skip():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


def normal(seed, *shape, dtype=BF16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64).to(dtype)


# ---- without a GPU -------------------------------------------------------------------------------------------------------------
def table(lengths, tokens):
    """(tokens, sequences, blocks, longest) and the table's parts"""
    lib, sizes, head = layer.load_library(), np.array(lengths, dtype=np.int64), ctypes.create_string_buffer(layer._PACKING.size)
    assert lib.ace_packing_table(sizes.ctypes.data, len(sizes), tokens, head, None, 0) == 0
    t, sequences, blocks, longest, _ = layer._PACKING.unpack(head.raw)
    out = np.full(blocks * 16 + sequences * 2 + 4, -7, dtype=np.int32)
    size = blocks * 64 + sequences * 8
    if size:
        assert lib.ace_packing_table(sizes.ctypes.data, len(sizes), tokens, head, out.ctypes.data, size - 1) == -1
    assert lib.ace_packing_table(sizes.ctypes.data, len(sizes), tokens, head, out.ctypes.data, size) == 0
    assert (out[size // 4:] == -7).all()
    return (t, sequences, blocks, longest), *out[:blocks * 16].reshape(4, -1, 4), out[blocks * 16:size // 4].reshape(-1, 2)


@pytest.mark.parametrize("lengths,tail", [([], 0), ([], 5), ([0, 0], 0), ([1], 0), ([128], 1), ([129, 0, 127, 1, 1000], 300), ([5] * 300, 128),
                                          ([pyrandom.Random(i).randint(0, 900) for i in range(50)], 77)])
def test_the_table_has_every_token_once_and_long_walks_first(lengths, tail):
    tokens = sum(lengths) + tail
    head, queries, keys, queries2, keys2, sequences = table(lengths, tokens)
    some = [n for n in lengths if n]
    assert head[0] == tokens and head[1] == len(some) and head[3] == max(some, default=0)
    begins = np.cumsum([0] + some)[:-1].tolist()
    assert sequences.tolist() == [[a, n] for a, n in zip(begins, some)]
    for blocks in (queries, keys, queries2, keys2):
        seen = np.zeros(tokens, dtype=int)
        for first, n, b, s in blocks.tolist():
            assert (first, n) == ((sum(lengths), tail) if s < 0 else (begins[s], some[s])) and 0 <= b * 128 < n
            seen[first + b * 128:first + min(n, b * 128 + 128)] += 1
        assert (seen == 1).all()
    # long walks first, in runs of blocks of one sequence or all of them together; tokens of no sequence last
    for blocks, run, walk in ((queries, 3, lambda n, b: b), (keys, 2, lambda n, b: (n - 1) // 128 - b), (queries2, 1 << 30, lambda n, b: b), (keys2, 1 << 30, lambda n, b: (n - 1) // 128 - b)):
        order = [(s < 0, -(walk(n, b) // run), -n, first, -walk(n, b)) for first, n, b, s in blocks.tolist()]
        assert order == sorted(order)


def pack(tokens=300, sequences=2, blocks=4, longest=200, at=host.AT):
    return layer._PACKING.pack(tokens, sequences, blocks, longest, at)


def attend(tokens=300, heads=4, kv_heads=2, dim=128, window=0, sinks=0, dtype=1, batch=1, start=0):
    strides = [0, heads * dim, dim] * 4
    return layer._ATTEND.pack(batch, tokens, tokens, heads, kv_heads, dim, dtype, window, sinks, 0.125, start, 0, *strides, *[host.AT] * 5)


def forward(p=None, **how):
    return ("ace_packed_attend_forward", attend(**how), pack() if p is None else p, None)


def backward(p=None, **how):
    return ("ace_packed_attend_backward", attend(**how), pack() if p is None else p, host.AT, [0, 512, 128], host.AT, host.AT, host.AT, host.AT, 1 << 62, None)


def test_refusals_of_the_c_entries(tmp_path):
    lib = layer.load_library()
    lengths, head = (ctypes.c_int64 * 2)(3, 4), ctypes.create_string_buffer(layer._PACKING.size)
    assert lib.ace_packing_table(lengths, 2, 6, head, None, 0) == -1 and lib.ace_packing_table(None, 2, 9, head, None, 0) == -1
    assert lib.ace_packing_table(lengths, -1, 9, head, None, 0) == -1 and lib.ace_packing_table(lengths, 2, -1, head, None, 0) == -1
    assert lib.ace_packing_table(lengths, 2, 9, None, None, 0) == -1 and lib.ace_packing_table(lengths, 2, layer.MAX_TOKENS + 1, head, None, 0) == -2
    lengths[0] = -1
    assert lib.ace_packing_table(lengths, 2, 9, head, None, 0) == -1
    lengths[0] = (1 << 63) - 1
    assert lib.ace_packing_table(lengths, 2, 9, head, None, 0) == -1
    bad = [dict(batch=2), dict(tokens=299), dict(start=host.AT), dict(heads=3), dict(dim=12), dict(dtype=0), dict(window=-1), dict(p=pack(at=0)), dict(p=pack(at=host.AT + 8)),
           dict(p=pack(blocks=0)), dict(p=pack(longest=301)), dict(p=pack(sequences=-1))]
    for make in (forward, backward):
        for how, r in zip(bad, host.run(tmp_path, [host.call(*make(**how)) for how in bad])):
            assert r["rc"] == -1 and r["launches"] == 0, how
        big = [dict(dim=136), dict(heads=64, kv_heads=64, p=pack(blocks=1 << 16))]
        assert [r["rc"] for r in host.run(tmp_path, [host.call(*make(**how)) for how in big])] == [-2, -2]
    lib.ace_packed_attend_backward_workspace_bytes.restype = ctypes.c_size_t
    assert lib.ace_packed_attend_backward_workspace_bytes(attend(dim=12), pack()) == 0
    size = lib.ace_packed_attend_backward_workspace_bytes(attend(), pack())
    assert size == 4 * 4 * 300
    many = [dict(window=4, sinks=1 << 20, tokens=1 << 20, heads=2, kv_heads=1, p=pack(1 << 20, n, 9000, longest)) for n, longest in ((130, 1 << 20), (120, 1 << 20), (130, 4))]
    assert [(r["rc"], r["launches"]) for r in host.run(tmp_path, [host.call(*backward(**how)) for how in many])] == [(-2, 0), (0, 3), (0, 2)]
    few = list(backward())
    few[-2] = size - 1
    assert host.run(tmp_path, [host.call(*few)])[0]["rc"] == -1


def test_launches_and_their_lds(tmp_path):
    """Every kernel that needs it asks for its LDS on every device; nothing is launched for no tokens; first keys take a launch more where a sequence
    is longer than the window."""
    calls = [forward(), forward(dim=64, dtype=2), backward(), backward(window=64, sinks=3), backward(window=200, sinks=3), backward(window=64, sinks=3, dim=96),
             forward(tokens=0, p=pack(0, 0, 0, 0, 0)), backward(tokens=0, p=pack(0, 0, 0, 0, 0)), backward(tokens=70000, heads=32, kv_heads=32, p=pack(70000, 300, 700, 800))]
    done = host.run(tmp_path, [host.call(*c, device=d) for d in (0, 3) for c in calls])
    assert [r["launches"] for r in done] == [1, 1, 2, 3, 2, 3, 0, 0, 2] * 2
    assert all(r["rc"] == 0 and r["unprepared"] == 0 for r in done)


def test_refusals():
    for bad in ([1.5], ["a"], [[1, 2]]):
        with pytest.raises(TypeError):
            layer.Packing(bad)
    for bad, tokens in (([-1], None), ([5], 4), ([1], layer.MAX_TOKENS + 1)):
        with pytest.raises(ValueError):
            layer.Packing(bad, tokens=tokens)
    with pytest.raises(ValueError):
        layer.Packing([1], device="cpu")
    with pytest.raises(TypeError):
        layer.packed_attention(*[torch.ones(4, 2, 64, dtype=BF16)] * 3, [4])


# ---- on the GPU ----------------------------------------------------------------------------------------------------------------
def case(seed, tokens, heads, kv_heads, dim, dtype=BF16):
    return tuple(normal(seed + i, tokens, h, dim, dtype=dtype) for i, h in enumerate((heads, kv_heads, kv_heads, heads)))


def run(q, k, v, do, lengths, **how):
    packing = layer.Packing(lengths, tokens=q.shape[0])
    gpu_ = [t.cuda() for t in (q, k, v)]
    out, lse = layer.packed_attention(*gpu_, packing, **how)
    got = {"out": out, "lse": lse}
    if do is not None:
        got.update(zip(("dq", "dk", "dv"), layer.packed_attention_backward(do.cuda(), *gpu_, out, lse, packing, **how)))
        again = layer.packed_attention_backward(do.cuda(), *gpu_, out, lse, packing, **how)
        assert all(torch.equal(got[n].nan_to_num(), a.nan_to_num()) for n, a in zip(("dq", "dk", "dv"), again))
    return got


def check(q, k, v, do, lengths, only=None, **how):
    """`only`: which sequences are looked at (all of them by default)."""
    cuda_or_skip()
    got = {n: t.cpu() for n, t in run(q, k, v, do, lengths, **how).items()}
    small, at = ref.SMALLEST[q.dtype], 0
    for i, n in enumerate(lengths):
        rows = slice(at, at + n)
        at += n
        if n == 0 or (only is not None and i not in only):
            continue
        want = ref.attention(*(t[None, rows] for t in (q, k, v)), d_out=None if do is None else do[None, rows], unit=ref.UNIT[q.dtype], **how)
        ref.close(got["out"][rows], want["out"][0][0], want["out"][1][0] + small)
        ref.close(got["lse"][:, rows], want["lse"][0][0], want["lse"][1][0])
        for name in ("dq", "dk", "dv"):
            if do is not None:
                ref.close(got[name][rows], want[name][0][0], want[name][1][0] + 64 * small)
    assert (got["out"][at:] == 0).all() and (got["lse"][:, at:] == -INF).all()
    for name in ("dq", "dk", "dv"):
        if do is not None:
            assert (got[name][at:] == 0).all()


@gpu
@pytest.mark.parametrize("lengths,tail", [([1], 0), ([128], 0), ([129], 0), ([1, 1, 1], 0), ([0, 5, 0, 300, 64, 1, 0], 3), ([31, 33, 127, 129, 255, 257], 0), ([], 40), ([400], 200),
                                          ([0], 0), ([2] * 150, 129)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (60, 3)])
def test_lengths(lengths, tail, window, sinks):
    cuda_or_skip()
    check(*case(len(lengths), sum(lengths) + tail, 4, 2, 64), lengths, window=window, sinks=sinks)


@gpu
@pytest.mark.parametrize("dim", [8, 40, 64, 80, 96, 104, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_head_sizes(dim, dtype):
    cuda_or_skip()
    check(*case(dim, 405, 4, 2, dim, dtype), [150, 33, 0, 200], window=70, sinks=3)


@gpu
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (2, 1), (3, 3), (6, 2), (8, 1), (8, 8), (12, 4), (20, 20), (40, 40)])
def test_heads(heads, kv_heads):
    """Numbers of heads that are dealt out to the dies in one, two, four and eight classes."""
    cuda_or_skip()
    check(*case(heads, 700, heads, kv_heads, 64), [290, 3, 150, 130, 127])


@gpu
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (64, 4), (65, 70), (100, 200), (300, 5), (10 ** 9, 10 ** 9)])
def test_windows(window, sinks):
    cuda_or_skip()
    check(*case(7, 640, 2, 1, 128), [300, 5, 64, 260], window=window, sinks=sinks)


@gpu
@pytest.mark.parametrize("kv_heads,shared", [(2, 2), (16, 1), (32, 1)])
@pytest.mark.parametrize("dim,dtype", [(128, BF16), (56, F16)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (100, 40)])
def test_gradients_with_every_size_of_key_block(kv_heads, shared, dim, dtype, window, sinks):
    """Key blocks of 32, 64 and 128 keys per workgroup."""
    cuda_or_skip()
    lengths = [pyrandom.Random(i).randint(0, 270) for i in range(8)] + [131, 1, 260]
    check(*case(47, sum(lengths) + 20, kv_heads * shared, kv_heads, dim, dtype), lengths, window=window, sinks=sinks)


@gpu
def test_very_many_sequences():
    cuda_or_skip()
    rng = pyrandom.Random(5)
    lengths = [rng.choice([0, 1, 2, 7, 40, 64, 130]) for _ in range(3000)]
    check(*case(9, sum(lengths) + 9, 2, 1, 32), lengths, only=set(range(0, 3000, 37)) | set(range(2990, 3000)), window=50, sinks=2)


@gpu
def test_long_sequences():
    cuda_or_skip()
    check(*case(11, 5000, 2, 1, 64), [3001, 17, 1900], window=None)
    check(*case(12, 5000, 2, 1, 64), [3001, 17, 1900], window=700, sinks=33)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_what_stands_in_other_sequences_does_not_matter(dtype):
    """Values that are no numbers in one sequence, and behind the last: every other one's results have the same bits."""
    cuda_or_skip()
    lengths = [100, 200, 5, 300, 64]
    for window, sinks in ((None, 0), (40, 3)):
        args = case(21, 700, 4, 2, 64, dtype)
        want = run(*args, lengths, window=window, sinks=sinks)
        for t in args:
            t[100:300], t[669:] = NAN, INF
        got = run(*args, lengths, window=window, sinks=sinks)
        for name, t in got.items():
            w = want[name]
            if name == "lse":
                t, w = t.t(), w.t()
            assert torch.equal(t[:100], w[:100]) and torch.equal(t[300:669], w[300:669]) and torch.equal(t[669:], w[669:]), name
            assert t[100:300].isnan().any()


@gpu
def test_a_value_that_is_no_number_reaches_those_that_see_it():
    cuda_or_skip()
    q, k, v, do = case(23, 400, 2, 2, 64)
    v[250, 0, 5] = NAN
    got = run(q, k, v, do, [200, 200])
    out = got["out"].cpu()
    assert out[250:400, 0, 5].isnan().all() and out[:250].isfinite().all() and out[:, 1].isfinite().all() and out[250:, 0, :5].isfinite().all()


@gpu
def test_strides_and_places():
    """A slice of the product for queries, keys and values, heads before tokens, rows that have to be copied."""
    device = cuda_or_skip()
    packing, lengths = layer.Packing([70, 130], tokens=210), [70, 130]
    qkv, do = normal(1, 210, 8, 64).to(device), normal(2, 210, 4, 64).to(device)
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]

    def both(q, k, v, do):
        out, lse = layer.packed_attention(q, k, v, packing)
        return (out, lse) + layer.packed_attention_backward(do, q, k, v, out, lse, packing)
    want = both(*(t.contiguous() for t in (q, k, v, do)))
    odd = torch.zeros(210 * 4 * 64 + 1, dtype=BF16, device=device)[1:].view(210, 4, 64)
    odd.copy_(do)
    swap = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v, do)]
    flip = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v, do)]
    for other in ((q, k, v, odd), swap, flip):
        assert all(torch.equal(a, b) for a, b in zip(both(*other), want))
    assert len(lengths) == 2 and packing.lengths == (70, 130) and packing.tokens == 210 and packing.longest == 130


@gpu
def test_as_each_sequence_alone():
    """A sequence of several blocks by window_attention takes the same steps: the same bits."""
    device = cuda_or_skip()
    lengths = [700, 520, 300]
    q, k, v, do = (t.to(device) for t in case(31, 1520, 16, 16, 128))
    packing = layer.Packing(lengths)
    for how in (dict(), dict(window=200, sinks=4)):
        out, lse = layer.packed_attention(q, k, v, packing, **how)
        at = 0
        for n in lengths:
            rows = slice(at, at + n)
            at += n
            alone, alone_lse = layer.window_attention(*(t[None, rows] for t in (q, k, v)), **how)
            assert torch.equal(out[rows], alone[0]) and torch.equal(lse[:, rows], alone_lse[0])


@gpu
def test_refused_on_the_gpu():
    device = cuda_or_skip()
    q = torch.ones(10, 4, 64, dtype=BF16, device=device)
    p = layer.Packing([4, 6])
    out, lse = layer.packed_attention(q, q, q, p)
    for call, kind in ((lambda: layer.packed_attention(q[:9], q[:9], q[:9], p), ValueError), (lambda: layer.packed_attention(q[None], q[None], q[None], p), ValueError),
                       (lambda: layer.packed_attention(q.float(), q.float(), q.float(), p), TypeError), (lambda: layer.packed_attention(q, q[:, :3], q[:, :3], p), ValueError),
                       (lambda: layer.packed_attention(q, q, q[:, :2], p), ValueError), (lambda: layer.packed_attention(q, q, q, p, window=0), ValueError),
                       (lambda: layer.packed_attention(q, q.half(), q, p), TypeError), (lambda: layer.packed_attention(q, q, q, p, scale=-1.0), ValueError),
                       (lambda: layer.packed_attention_backward(q[:5], q, q, q, out, lse, p), ValueError), (lambda: layer.packed_attention_backward(q, q, q, q, out, lse[:2], p), ValueError),
                       (lambda: layer.packed_attention_backward(q, q, q, q, out[:, :2], lse, p), ValueError), (lambda: layer.Packing(torch.tensor([4], device=device)), ValueError)):
        with pytest.raises(kind):
            call()


@gpu
def test_graphs_streams_and_two_packings():
    """Forward and backward captured, replayed with other values and eager calls of another packing between; on two streams at once."""
    device = cuda_or_skip()
    q, k, v, do = (t.to(device) for t in case(41, 900, 8, 4, 64))
    p, other = layer.Packing([300, 1, 500], tokens=900), layer.Packing([900])

    def both(packing):
        out, lse = layer.packed_attention(q, k, v, packing, window=100, sinks=2)
        return (out, lse) + layer.packed_attention_backward(do, q, k, v, out, lse, packing, window=100, sinks=2)
    both(p), both(other)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both(p)
    for i in range(4):
        for t in (q, k, v, do):
            t.copy_(torch.randn(t.shape, device=device, generator=torch.Generator(device=device).manual_seed(i)))
        graph.replay()
        both(other)
        want = both(p)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(both(p))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


@gpu
def test_automatic_differentiation_is_told():
    device = cuda_or_skip()
    q = torch.ones(10, 4, 64, dtype=BF16, device=device, requires_grad=True)
    with pytest.raises(AceError):
        layer.packed_attention(q, q, q, layer.Packing([10]))[0].sum().backward()
