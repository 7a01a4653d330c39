"""The training-layer operators on the GPU against plain implementations in 64 bits (layer_reference.py), at the sizes, masks and
values where they can go wrong; and without a GPU: the formulas of the gradients against differences, the exported
functions, what is refused."""
import ctypes
import itertools
import os
import re

import pytest
import torch

from superscaler_amd import layer
from superscaler_amd.evaluator import AceError
from tests import layer_reference as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
gpu = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def cuda_or_skip():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


def normal(seed, *shape, at=0.0, by=1.0, dtype=F32):
    return (at + by * torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)).to(dtype)


# ---- without a GPU ----------------------------------------------------------------------------------------------------------------
def test_every_declared_function_is_exported():
    lib = layer.load_library()
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "ace_layer.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(ace_[a-z_0-9]+)\s*\(", text)))
    assert names == sorted(layer.EXPORTS)
    assert all(hasattr(lib, n) for n in names)
    assert lib.ace_layer_abi_version() == layer.ABI_VERSION
    for name, value in (("ACE_NORM_MAX_WIDTH", layer.MAX_WIDTH), ("ACE_ADAMW_BLOCK", layer.ADAMW_BLOCK), ("ACE_ADAMW_CHUNK", layer.ADAMW_CHUNK)):
        assert int(re.search(rf"#define {name} (\d+)", text).group(1)) == value


def test_missing_library_fails_loudly(monkeypatch):
    monkeypatch.setattr(layer, "_lib", None)
    monkeypatch.setattr(layer, "_LIB_PATH", "/nonexistent/libace_layer.so")
    with pytest.raises(AceError):
        layer.load_library()


def test_refusals_of_the_c_entries():
    """Everything here is refused before a kernel would be launched."""
    lib = layer.load_library()
    assert lib.ace_layer_strerror(-1) == b"invalid argument" and lib.ace_layer_strerror(-99) == b"unknown error"

    def norm(rows=4, width=8, dtype=1):
        return layer._BLOCK_NORM.pack(rows, 1, width, dtype, 1, 1.0, 1e-5, 64, 64, 0, 0, 0, 0, 0)      # x and a block
    assert lib.ace_block_norm_forward(None, 64, 64, 64, None) == -1
    assert lib.ace_block_norm_forward(norm(), None, None, 64, None) == -1          # nowhere to write the residual
    assert lib.ace_block_norm_forward(norm(width=layer.MAX_WIDTH + 1), 64, None, 64, None) == -2
    assert lib.ace_block_norm_forward(norm(dtype=3), 64, None, 64, None) == -1
    assert lib.ace_block_norm_forward(norm(rows=0), 64, None, 64, None) == 0       # no rows
    assert lib.ace_block_norm_backward(norm(), 64, None, 64, 64, 64, None, None, None, None, None, None, 0, None) == -1   # no workspace
    assert lib.ace_block_norm_workspace_bytes(norm()) == 2 * 4 * 8 * 4
    one_gate = layer._BLOCK_NORM.pack(4, (1 << 63) - 1, 8, 1, 1, 1.0, 1e-5, 64, 64, 64, 0, 0, 0, 0)
    assert lib.ace_block_norm_workspace_bytes(one_gate) == 2 * 4 * 8 * 4      # (as many rows per gate as there can be)

    def attend(**change):
        a = dict(batch=2, queries=32, keys=32, heads=4, kv_heads=2, dim=64, dtype=1, window=0, sinks=0, scale=0.125, d_start=0, d_length=0)
        a.update({f"{t}_stride{i}": s for t in ("q", "k", "v", "out") for i, s in enumerate((8192, 256, 64))}, d_q=64, d_k=64, d_v=64, d_out=64, d_lse=64)
        return lib.ace_attend_forward(layer._ATTEND.pack(*{**a, **change}.values()), None, 0, None)
    assert attend(batch=0) == 0 and attend(queries=0) == 0
    for bad in ({"heads": 3}, {"dim": 12}, {"dim": 0}, {"dtype": 0}, {"scale": 0.0}, {"scale": float("nan")}, {"window": -1}, {"d_q": 0}, {"d_k": 72}, {"keys": -1},
                {"kv_heads": 0}, {"k_stride1": 252}):
        assert attend(**bad) == -1, bad
    assert attend(dim=136) == -2 and attend(batch=1 << 21) == -2 and attend(keys=(1 << 28) + 1) == -2 and attend(v_stride1=1 << 23) == -2
    a = layer._AdamW(64, 64, 1, 1, 16, 1, 1, 64, 64)
    first = (ctypes.c_int64 * 2)(0, 1)
    grads = (ctypes.c_void_p * 1)(64)
    assert lib.ace_adamw_step(ctypes.byref(a), grads, first, None, *[0.5] * 8, None) == -1        # 16 bits
    a.state_bits = 8
    assert lib.ace_adamw_step(ctypes.byref(a), grads, first, None, *[0.5] * 8, None) == -1        # no scales
    a.state_bits, first[1] = 32, 2
    assert lib.ace_adamw_step(ctypes.byref(a), grads, first, None, *[0.5] * 8, None) == -1        # chunks that disagree
    first[1], grads[0] = 1, None
    assert lib.ace_adamw_step(ctypes.byref(a), grads, first, None, *[0.5] * 8, None) == -1        # no gradient
    assert lib.ace_adamw_moments(None, None, None, None, 1, None, None, None) == -1
    assert lib.ace_adamw_moments(None, None, None, None, 0, None, None, None) == 0


def test_tensors_of_the_host_are_refused():
    x, w = torch.ones(2, 8), torch.ones(8)
    with pytest.raises(ValueError):
        layer.block_norm(x, entry_weight=w)
    q = torch.ones(1, 4, 2, 64, dtype=BF16)
    with pytest.raises(ValueError):
        layer.window_attention(q, q, q)
    with pytest.raises(ValueError):
        layer.AdamW([w])
    with pytest.raises(TypeError):
        layer.block_norm([1.0], entry_weight=w)


def norm_case(seed, shape, kind, parts, gate, bias, dtype=torch.float64, at=0.0):
    width = shape[-1]
    c = dict(x=normal(seed, *shape, at=at, dtype=dtype), block=None, residual_scale=1.0, gate=None, exit_weight=None, exit_bias=None, entry_weight=None, entry_bias=None, kind=kind,
             eps=1e-5)
    if "b" in parts:
        c.update(block=normal(seed + 1, *shape, by=0.7, at=at, dtype=dtype), residual_scale=0.5)
        if gate is not None:
            c["gate"] = normal(seed + 2, *gate, at=0.5, dtype=dtype)
    if "x" in parts:
        c["exit_weight"] = normal(seed + 3, width, at=1.0, by=0.3, dtype=dtype)
        c["exit_bias"] = normal(seed + 4, width, dtype=dtype) if bias else None
    if "n" in parts:
        c["entry_weight"] = normal(seed + 5, width, at=1.0, by=0.3, dtype=dtype)
        c["entry_bias"] = normal(seed + 6, width, dtype=dtype) if bias else None
    return c


def wide_gate(gate, x):
    """The gate in a shape that broadcasts over x."""
    if gate is None or gate.dim() in (1, x.dim()):
        return gate
    return gate.view(gate.shape[:-1] + (1,) * (x.dim() - gate.dim()) + gate.shape[-1:])


@pytest.mark.parametrize("kind,parts,gate", [("layer", "bxn", (5,)), ("rms", "bxn", (2, 1, 5)), ("layer", "bx", (2, 3, 5)), ("rms", "bn", (5,)), ("layer", "n", None)])
def test_norm_gradients_against_differences(kind, parts, gate):
    c = norm_case(1, (2, 3, 5), kind, parts, gate, True)
    dr, dy = normal(50, 2, 3, 5, dtype=torch.float64), normal(51, 2, 3, 5, dtype=torch.float64)
    grads = ref.block_norm_grads(dr, dy if "n" in parts else None, **c)

    def loss(**change):
        r, y = ref.block_norm(**{**c, **change})
        return float((r * dr).sum() + (0 if y is None else (y * dy).sum()))
    h = 1e-5
    for name, (g, _) in grads.items():
        for at in range(0, c[name].numel(), 3):
            step = torch.zeros_like(c[name])
            step.view(-1)[at] = h
            assert abs((loss(**{name: c[name] + step}) - loss(**{name: c[name] - step})) / (2 * h) - float(g.reshape(-1)[at])) < 1e-6


def test_attention_gradients_against_differences():
    q, k, v, do = (normal(i, 2, 5, h, 8, dtype=torch.float64) for i, h in ((1, 4), (2, 2), (3, 2), (4, 4)))
    how = dict(window=2, sinks=1, start=torch.tensor([0, -1]), lengths=torch.tensor([5, 3]))
    r = ref.attention(q, k, v, d_out=do, **how)
    h = 1e-5
    for name, t in (("dq", q), ("dk", k), ("dv", v)):
        for at in range(0, t.numel(), 7):
            def loss(by):
                moved = t.clone()
                moved.view(-1)[at] += by
                a = {"dq": (moved, k, v), "dk": (q, moved, v), "dv": (q, k, moved)}[name]
                return float((ref.attention(*a, **how)["out"][0] * do).sum())
            assert abs((loss(h) - loss(-h)) / (2 * h) - float(r[name][0].reshape(-1)[at])) < 1e-6


# ---- norms around a block -----------------------------------------------------------------------------------------------------------
def slack(t):
    """What 32-bit arithmetic may be off by: 128 units of the largest value of a row."""
    return 2.0 ** -17 * t.double().abs().amax(-1, keepdim=True).expand_as(t)


def check_norm(c, dr, dy, device):
    d = {k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    eps = d.pop("eps")
    got = layer.block_norm(d["x"], d["block"], **{k: v for k, v in d.items() if k not in ("x", "block")}, eps=eps)
    wide = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    wide["gate"] = wide_gate(wide["gate"], wide["x"])
    r, y = ref.block_norm(**wide)
    terms = wide["residual_scale"] * wide["x"].abs() + (0 if wide["block"] is None else ((r - wide["residual_scale"] * wide["x"]).abs() + wide["block"].abs()))
    if c["block"] is None:
        assert got.residual is d["x"]
    else:
        ref.close(got.residual, r, 4 * slack(terms) + ref.SMALLEST[c["x"].dtype])
    if y is not None:
        spread = ref.norm_parts(r, c["kind"], eps)[1]
        # a residual is off by its terms' rounding, and the norm divides that by its spread
        ref.close(got.normed, y, 8 * slack(y) + 2.0 ** -18 * spread * terms.amax(-1, keepdim=True) * wide["entry_weight"].abs().amax() + ref.SMALLEST[c["x"].dtype])
    dd = [None if t is None else t.to(device) for t in (dr, dy)]
    grads = layer.block_norm_backward(*dd, d["x"], d["block"], got.stats, **{k: v for k, v in d.items() if k not in ("x", "block")})
    again = layer.block_norm_backward(*dd, d["x"], d["block"], got.stats, **{k: v for k, v in d.items() if k not in ("x", "block")})
    want = ref.block_norm_grads(*(None if t is None else t.double() for t in (dr, dy)), **wide)
    for name, g in grads._asdict().items():
        if c[name] is None:
            assert g is None
            continue
        value, size = want[name]
        assert torch.equal(g, getattr(again, name))
        ref.close(g, value.reshape(g.shape), 2.0 ** -16 * size.reshape(g.shape) * 8 + ref.SMALLEST[g.dtype])


@gpu
@pytest.mark.parametrize("width", [1, 7, 8, 63, 64, 513, 1000, 1024, 2048, 2056, 4097, 6144, 8192, 12288, 16384, 20001, 24576, 32768])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_norm_widths(width, dtype):
    device = cuda_or_skip()
    kind = "layer" if width % 2 else "rms"
    c = norm_case(width, (3, 2, width), kind, "bxn", (3, width), True, dtype)
    check_norm(c, normal(8, 3, 2, width, dtype=dtype), normal(9, 3, 2, width, dtype=dtype), device)


@gpu
@pytest.mark.parametrize("kind,parts,gate,bias", [(k, p, g, b) for (k, b), p in itertools.product([("layer", True), ("rms", False)], ["bxn", "bx", "bn", "b", "n"])
                                                  for g in (["none", "channel", "sequence", "wide", "token"] if "b" in p else ["none"])])
def test_norm_parts_and_gates(kind, parts, gate, bias):
    device = cuda_or_skip()
    shape = (3, 37, 264)
    size = {"none": None, "channel": (264,), "sequence": (3, 264), "wide": (3, 1, 264), "token": shape}[gate]
    c = norm_case(3, shape, kind, parts, size, bias)
    c = {k: v.float() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    check_norm(c, normal(8, *shape), normal(9, *shape) if "n" in parts else None, device)


@gpu
@pytest.mark.parametrize("shape,gate", [((1, 40), (40,)), ((40,), None), ((1, 1, 40), (1, 40)), ((2500, 40), (40,)), ((5, 700, 40), (5, 40)), ((900, 3, 40), (900, 40)),
                                        ((1537, 1, 40), (1537, 1, 40))])
def test_norm_rows_and_runs(shape, gate):
    """Rows that fill many runs, gates that end inside a run and runs that end inside a gate."""
    device = cuda_or_skip()
    c = norm_case(4, shape, "layer", "bxn", gate, True, F32)
    check_norm(c, normal(8, *shape), normal(9, *shape), device)


@gpu
def test_norm_of_no_rows_and_of_missing_gradients():
    device = cuda_or_skip()
    c = norm_case(4, (0, 16), "layer", "bxn", (16,), True, F32)
    d = {k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    r = layer.block_norm(d.pop("x"), d.pop("block"), **d)
    assert r.residual.shape == r.normed.shape == (0, 16)
    d.pop("eps")
    g = layer.block_norm_backward(None, None, c["x"].to(device), c["block"].to(device), r.stats, **d)
    assert g.x.shape == (0, 16) and all(int(t.count_nonzero()) == 0 for t in g)
    c = norm_case(4, (5, 16), "rms", "bxn", (16,), False, F32)
    check_norm(c, None, normal(9, 5, 16), device)
    check_norm(c, normal(9, 5, 16), None, device)


@gpu
def test_norm_far_from_zero_and_with_one_large_channel():
    """A mean of hundreds of deviations, and a channel of a thousand others: the variance keeps its digits."""
    device = cuda_or_skip()
    c = norm_case(5, (4, 3000), "layer", "n", None, True, F32, at=300.0)
    c["x"][:, 0] = 1000.0
    x = c["x"].double()
    n, rstd = ref.norm_parts(x, "layer", 1e-5)
    got = layer.block_norm(c["x"].to(device), entry_weight=c["entry_weight"].to(device), entry_bias=c["entry_bias"].to(device))
    # (x - mean in 32 bits: half a unit of the mean, divided by the spread)
    ref.close(got.normed, n * c["entry_weight"] + c["entry_bias"], (2.0 ** -22 * 1000 * rstd + 2.0 ** -20) * c["entry_weight"].abs().amax() + 2.0 ** -20 * (n.abs() + 1))
    assert torch.allclose(got.stats[:, 3].double().cpu(), rstd[:, 0], rtol=2.0 ** -18)


@gpu
def test_norm_rows_that_are_no_numbers_stay_among_themselves():
    device = cuda_or_skip()
    c = norm_case(6, (6, 320), "rms", "bxn", None, False, F32)
    c["block"][2, 5] = float("nan")
    c["x"][4, 0] = float("inf")
    d = {k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    got = layer.block_norm(d.pop("x"), d.pop("block"), **d)
    r, y = ref.block_norm(**{k: v.double() if isinstance(v, torch.Tensor) else v for k, v in c.items()})
    for row in (0, 1, 3, 5):
        ref.close(got.normed[row], y[row], 16 * slack(y[row]))
    assert got.normed[2].isnan().all() and got.residual[2].isnan().all() and got.normed[4, 0].isnan()


@gpu
def test_norm_strides_streams_and_other_orders():
    """Rows of a wider tensor, a transposed tensor and a broadcast one give what their contiguous copies give; so does a call on
    another stream."""
    device = cuda_or_skip()
    wide = normal(1, 6, 5, 128).to(device)
    w = normal(2, 96, at=1.0).to(device)
    for x in (wide[:, :, 16:112], wide[:, :, 16:112].transpose(0, 1), wide[:1, :, 16:112].expand(4, -1, -1), wide[:, :, 17:113]):
        a, b = layer.block_norm(x, x, entry_weight=w), layer.block_norm(x.contiguous(), x.contiguous(), entry_weight=w)
        assert torch.equal(a.normed, b.normed) and torch.equal(a.residual, b.residual)
    side = torch.cuda.Stream()
    x = wide[:, :, :96].contiguous()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = layer.block_norm(x * 2, entry_weight=w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(c.normed, layer.block_norm(x * 2, entry_weight=w).normed)
    flat = torch.zeros(1 + 7 * 96, device=device)      # an odd start
    flat[1:] = normal(3, 7 * 96).to(device)
    v = flat[1:].view(7, 96)
    assert torch.equal(layer.block_norm(v, entry_weight=w).normed, layer.block_norm(v.clone(), entry_weight=w).normed)


@gpu
def test_norm_refusals():
    device = cuda_or_skip()
    x, w = torch.ones(2, 3, 8, device=device), torch.ones(8, device=device)
    for error, a, k in ((ValueError, (x,), {}), (ValueError, (x,), {"gate": w}), (ValueError, (x,), {"entry_weight": w, "residual_scale": 0.5}), (ValueError, (x, x[:1]), {}),
                        (ValueError, (x, x), {"gate": torch.ones(3, 8, device=device)}), (ValueError, (x, x), {"exit_bias": w}), (ValueError, (x, x), {"entry_weight": w[:4]}),
                        (ValueError, (x, x), {"kind": "group"}), (TypeError, (x, x.half()), {}), (TypeError, (x.double(), x.double()), {}), (ValueError, (x, x), {"entry_weight": w.cpu()}),
                        (ValueError, (torch.ones(1, layer.MAX_WIDTH + 1, device=device),), {"entry_weight": torch.ones(layer.MAX_WIDTH + 1, device=device)})):
        with pytest.raises(error):
            layer.block_norm(*a, **k)
    stats = layer.block_norm(x, x, entry_weight=w).stats
    for error, a, k in ((ValueError, (x, x, x, x, stats), {}), (ValueError, (x[:1], None, x, x, stats), {}), (TypeError, (x.half(), None, x, x, stats), {}),
                        (ValueError, (x, x, x, x, stats[:1]), {"entry_weight": w})):
        with pytest.raises(error):
            layer.block_norm_backward(*a, **k)


# ---- attention --------------------------------------------------------------------------------------------------------------------------
def attention_case(seed, batch, queries, keys, heads, kv_heads, dim, dtype):
    return (normal(seed, batch, queries, heads, dim, dtype=dtype), normal(seed + 1, batch, keys, kv_heads, dim, dtype=dtype), normal(seed + 2, batch, keys, kv_heads, dim, dtype=dtype),
            normal(seed + 3, batch, queries, heads, dim, dtype=dtype))


def check_attention(q, k, v, do, device, backward=True, **how):
    dev = {n: t.to(device) if isinstance(t, torch.Tensor) else t for n, t in how.items()}
    dq, dk, dv, ddo = (t.to(device) for t in (q, k, v, do))
    out, lse = layer.window_attention(dq, dk, dv, **dev)
    want = ref.attention(q, k, v, d_out=do if backward else None, unit=ref.UNIT[q.dtype], **how)
    small = ref.SMALLEST[q.dtype]
    ref.close(out, want["out"][0], want["out"][1] + small)
    assert out.dtype == q.dtype
    ref.close(lse, want["lse"][0], want["lse"][1])
    if backward:
        got = layer.window_attention_backward(ddo, dq, dk, dv, out, lse, **dev)
        again = layer.window_attention_backward(ddo, dq, dk, dv, out, lse, **dev)
        for name, g, a in zip(("dq", "dk", "dv"), got, again):
            assert torch.equal(g, a)
            ref.close(g, want[name][0], want[name][1] + 64 * small)


@gpu
@pytest.mark.parametrize("dim", [8, 40, 64, 80, 96, 104, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("queries,keys", [(150, 150), (33, 170)])
def test_attention_head_sizes(dim, dtype, queries, keys):
    device = cuda_or_skip()
    check_attention(*attention_case(dim, 2, queries, keys, 4, 2, dim, dtype), device, window=70, sinks=3)


@gpu
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (6, 2), (8, 1), (40, 40)])
@pytest.mark.parametrize("length", [1, 2, 31, 64, 65, 128, 129, 257])
def test_attention_lengths_and_shared_heads(heads, kv_heads, length):
    device = cuda_or_skip()
    check_attention(*attention_case(length, 2, length, length, heads, kv_heads, 64, BF16), device)


@gpu
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (1, 1), (16, 0), (64, 4), (65, 70), (100, 0), (100, 200), (300, 5), (10 ** 9, 10 ** 9)])
def test_attention_windows(window, sinks):
    device = cuda_or_skip()
    check_attention(*attention_case(7, 1, 300, 300, 2, 1, 128, BF16), device, window=window, sinks=sinks)


@gpu
@pytest.mark.parametrize("queries,keys", [(1, 1), (1, 31), (1, 33), (1, 500), (2, 700), (5, 300), (16, 1000), (17, 1000), (64, 900), (3, 2), (200, 40)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (100, 3)])
def test_attention_of_new_tokens(queries, keys, window, sinks):
    device = cuda_or_skip()
    check_attention(*attention_case(queries, 3, queries, keys, 8, 2, 128, BF16), device, window=window, sinks=sinks)


@gpu
@pytest.mark.parametrize("batch,heads,kv_heads", [(1, 4, 2), (6, 8, 8), (19, 8, 8)])
@pytest.mark.parametrize("dim,dtype", [(128, BF16), (56, F16)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (100, 40)])
def test_attention_gradients_of_few_and_many_heads(batch, heads, kv_heads, dim, dtype, window, sinks):
    """Key blocks of 32, 64 and 128 keys per workgroup."""
    device = cuda_or_skip()
    check_attention(*attention_case(47, batch, 270, 270, heads, kv_heads, dim, dtype), device, window=window, sinks=sinks)


@gpu
@pytest.mark.parametrize("batch", [1, 6, 19])
@pytest.mark.parametrize("window,sinks", [(None, 0), (90, 5), (33, 70)])
def test_attention_gradients_of_ragged_sequences(batch, window, sinks):
    """Key blocks of 32, 64 and 128 keys per workgroup, sequences of any length that begin anywhere."""
    device = cuda_or_skip()
    lengths = (torch.arange(batch, dtype=torch.int32) * 53 + 201) % 271
    start = (torch.arange(batch, dtype=torch.int32) * 61 + 17) % 300 - 120
    check_attention(*attention_case(53, batch, 265, 270, 8, 8, 64, BF16), device, window=window, sinks=sinks, start=start, lengths=lengths)


@gpu
@pytest.mark.parametrize("window,sinks", [(None, 0), (150, 3), (1, 0)])
@pytest.mark.parametrize("batch,queries,keys,heads,kv_heads", [(1, 1, 700, 2, 2), (3, 7, 1200, 6, 2), (1, 16, 1000, 40, 4), (2, 100, 1500, 2, 1), (20, 1, 256, 20, 20), (3, 128, 600, 2, 2),
                                                               (40, 9, 200, 8, 1)])
def test_attention_of_few_queries_over_long_caches(batch, queries, keys, heads, kv_heads, window, sinks):
    """Keys split over wavefronts and workgroups, whose answers are joined, and caches too short for that."""
    device = cuda_or_skip()
    q, k, v, do = attention_case(31, batch, queries, keys, heads, kv_heads, 64, BF16)
    check_attention(q, k, v, do, device, backward=False, window=window, sinks=sinks)
    lengths = torch.arange(batch, dtype=torch.int32) * 37 % (keys + 1)
    check_attention(q, k, v, do, device, backward=False, window=window, sinks=sinks, start=lengths - queries, lengths=lengths)


@gpu
@pytest.mark.parametrize("queries,heads,kv_heads", [(1, 8, 2), (5, 16, 1), (130, 4, 2)])
def test_attention_of_ragged_sequences(queries, heads, kv_heads):
    """Lengths from none to all, queries before the first key and behind the last, and what is past a length is not read."""
    device = cuda_or_skip()
    lengths = torch.tensor([0, 1, 150, 400, 77, 400], dtype=torch.int32)
    start = torch.tensor([0, 0, 149, 399, -40, 1000], dtype=torch.int32)
    q, k, v, do = attention_case(3, 6, queries, 400, heads, kv_heads, 64, F16)
    for b, n in enumerate(lengths.tolist()):
        k[b, n:], v[b, n:] = float("nan"), float("inf")
    check_attention(q, k, v, do, device, window=120, sinks=2, start=start, lengths=lengths)


@gpu
def test_attention_of_padded_sequences():
    device = cuda_or_skip()
    lengths = torch.tensor([0, 1, 64, 199, 130], dtype=torch.int32)
    check_attention(*attention_case(4, 5, 199, 199, 4, 4, 80, BF16), device, window=33, sinks=1, start=torch.zeros(5, dtype=torch.int32), lengths=lengths)


@gpu
def test_attention_of_large_and_equal_scores():
    """Scores of hundreds (weights of one and zero), scores that are all the same, and a growing sequence of maxima."""
    device = cuda_or_skip()
    q, k, v, do = attention_case(9, 1, 140, 140, 2, 2, 64, BF16)
    check_attention(q * 16, k * 16, v, do, device)
    check_attention(q * 0, k, v, do, device, window=50)
    ramp = k.clone()
    ramp[:] = torch.linspace(-20, 20, 140)[None, :, None, None].to(BF16)
    check_attention(torch.ones_like(q), ramp, v, do, device, scale=0.5)
    check_attention(torch.ones_like(q), -ramp, v, do, device, scale=0.5, window=30, sinks=1)


@gpu
def test_attention_lets_values_that_are_no_numbers_through():
    device = cuda_or_skip()
    q, k, v, _ = (t.to(device) for t in attention_case(9, 1, 200, 200, 1, 1, 64, BF16))
    q[0, 150, 0, 3] = float("nan")
    out, lse = layer.window_attention(q, k, v)
    assert out[0, 150].isnan().all() and lse[0, 0, 150].isnan()
    assert out[0, :150].isfinite().all() and out[0, 151:].isfinite().all()


@gpu
def test_attention_strides():
    """One tensor of queries, keys and values, other orders of batch and length, a shared batch, and views that have to be copied."""
    device = cuda_or_skip()
    qkv = normal(1, 2, 70, 8, 64, dtype=BF16).to(device)
    do = normal(2, 2, 70, 4, 64, dtype=BF16).to(device)
    time_first = qkv.transpose(0, 1).contiguous().transpose(0, 1)
    for t in (qkv, time_first, qkv[:1].expand(2, -1, -1, -1), normal(1, 2, 70, 8, 68, dtype=BF16).to(device)[..., 2:66], normal(1, 2, 70, 64, 8, dtype=BF16).to(device).transpose(2, 3)):
        q, k, v = t[:, :, :4], t[:, :, 4:6], t[:, :, 6:]
        plain = [x.clone(memory_format=torch.contiguous_format) for x in (q, k, v)]
        a, b = layer.window_attention(q, k, v, window=20, sinks=1), layer.window_attention(*plain, window=20, sinks=1)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        ga = layer.window_attention_backward(do, q, k, v, *a, window=20, sinks=1)
        gb = layer.window_attention_backward(do, *plain, *b, window=20, sinks=1)
        assert all(torch.equal(x, y) for x, y in zip(ga, gb))
        token = layer.window_attention(q[:, -1:], k, v, window=20)[0], layer.window_attention(plain[0][:, -1:], *plain[1:], window=20)[0]
        assert torch.equal(*token)


@gpu
def test_attention_at_offsets_past_32_bits():
    """A cache of more than 2^32 bytes, of which the last keys are seen."""
    device = cuda_or_skip()
    keys = (1 << 32) // (8 * 128 * 2) + 1000
    k = torch.zeros(1, keys, 8, 128, dtype=BF16, device=device)
    v = torch.zeros(1, keys, 8, 128, dtype=BF16, device=device)
    for queries in (1, 130):
        q, k1, v1, _ = attention_case(3, 1, queries, 500, 8, 8, 128, BF16)
        k[:, -500:], v[:, -500:] = k1.to(device), v1.to(device)
        out, lse = layer.window_attention(q.to(device), k, v, window=300)
        want = ref.attention(q, k1, v1, window=300, unit=ref.UNIT[BF16])
        ref.close(out, *want["out"])
        ref.close(lse, *want["lse"])


@gpu
@pytest.mark.parametrize("queries", [3, 40])
def test_attention_at_positions_and_windows_at_the_ends_of_32_bits(queries):
    """A window that holds every key is none, a sequence before the first key sees none, one far behind the last sees the first keys:
    the same kernels on the same keys, so the same bits."""
    device, least, most = cuda_or_skip(), -(1 << 31), (1 << 31) - 1
    q, k, v, do = (t.to(device) for t in attention_case(23, 1, queries, 90, 2, 1, 64, BF16))

    def both(start, **how):
        at = torch.tensor([start], dtype=torch.int32, device=device)
        out, lse = layer.window_attention(q, k, v, start=at, **how)
        return (out, lse) + layer.window_attention_backward(do, q, k, v, out, lse, start=at, **how)
    for start, window in ((50, most), (0, 1 << 30), (1 << 30, most), (most, most), (1000, (1 << 30) + 5)):
        for got, want in zip(both(start, window=window), both(start)):
            assert torch.equal(got, want), (start, window)
    for start in (least, -(1 << 30), -(1 << 28) - 7, -queries):
        for window in (None, 5, most):
            out, lse, dq, dk, dv = both(start, window=window, sinks=3)
            assert (out == 0).all() and (lse == -float("inf")).all() and not any(g.any() for g in (dq, dk, dv)), (start, window)
    for start in (most, 1 << 30, 100_000):
        out, lse, dq, dk, dv = both(start, window=5, sinks=3)
        few, few_lse = layer.window_attention(q, k[:, :3], v[:, :3], start=torch.tensor([9], dtype=torch.int32, device=device))
        assert torch.equal(out, few) and torch.equal(lse, few_lse), start
        assert not dk[:, 3:].any() and not dv[:, 3:].any() and dv[:, :3].any()


@gpu
def test_attention_without_keys_or_queries():
    device = cuda_or_skip()
    q, k = torch.ones(2, 3, 4, 64, dtype=BF16, device=device), torch.ones(2, 0, 2, 64, dtype=BF16, device=device)
    out, lse = layer.window_attention(q, k, k)
    assert int(out.count_nonzero()) == 0 and (lse == -float("inf")).all()
    dq, dk, dv = layer.window_attention_backward(q, q, k, k, out, lse)
    assert int(dq.count_nonzero()) == 0 and dk.shape == k.shape
    out, lse = layer.window_attention(q[:, :0], q[:, :, :2], q[:, :, :2])
    assert out.shape == (2, 0, 4, 64) and lse.shape == (2, 4, 0)
    dq, dk, dv = layer.window_attention_backward(q[:, :0], q[:, :0], q[:, :, :2], q[:, :, :2], out, lse)
    assert int(dk.count_nonzero()) == 0 and int(dv.count_nonzero()) == 0


@gpu
def test_attention_refusals():
    device = cuda_or_skip()
    q = torch.ones(2, 4, 4, 64, dtype=BF16, device=device)
    n = torch.ones(2, dtype=torch.int32, device=device)
    for error, a, k in ((ValueError, (q[0], q, q), {}), (TypeError, (q.float(),) * 3, {}), (TypeError, (q, q.half(), q), {}), (ValueError, (q, q, q[:, :2]), {}),
                        (ValueError, (q, q[:, :, :3], q[:, :, :3]), {}), (ValueError, (q[..., :12],) * 3, {}), (ValueError, (torch.cat([q, q, q], 3),) * 3, {}),
                        (ValueError, (q, q, q), {"window": 0}), (ValueError, (q, q, q), {"sinks": -1}), (ValueError, (q, q, q), {"scale": 0.0}),
                        (ValueError, (q, q, q), {"scale": float("nan")}), (TypeError, (q, q, q), {"lengths": n.long()}), (ValueError, (q, q, q), {"start": n[:1]}),
                        (ValueError, (q, q, q.cpu()), {})):
        with pytest.raises(error):
            layer.window_attention(*a, **k)
    out, lse = layer.window_attention(q, q, q)
    for error, a in ((ValueError, (q[:, :1], q, q, q, out, lse)), (ValueError, (q, q, q, q, out, lse[:1])), (TypeError, (q.half(), q, q, q, out, lse))):
        with pytest.raises(error):
            layer.window_attention_backward(*a)


# ---- AdamW ----------------------------------------------------------------------------------------------------------------------------------
HOW = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
SIZES = [1, 255, 256, 257, 8191, 8192, 8193, 0, 3, 70001]


def adamw_tensors(device, sizes, grad, copy, shift=0):
    """Parameters, copies and gradients; with `shift` at odd places of one buffer."""
    at, starts = shift, []
    for n in sizes:
        starts.append(at)
        at += n + shift
    flat, g, c = (torch.empty(at + 1, dtype=t, device=device) for t in (F32, grad, copy or BF16))
    flat.copy_(normal(1, at + 1, by=0.1))
    g.copy_(normal(2, at + 1, by=0.01).to(grad))
    views = [slice(s, s + n) for s, n in zip(starts, sizes)]
    return [flat[v] for v in views], [g[v] for v in views], [c[v] for v in views] if copy else None


@gpu
@pytest.mark.parametrize("grad,copy", [(F32, None), (BF16, BF16), (F16, F16), (F32, BF16), (BF16, None)])
@pytest.mark.parametrize("shift", [0, 1])
def test_adamw_in_32_bits(grad, copy, shift):
    device = cuda_or_skip()
    params, grads, copies = adamw_tensors(device, SIZES, grad, copy, shift)
    opt = layer.AdamW(params, copies=copies)
    want = [(p.double().cpu(), torch.zeros(p.shape, dtype=torch.float64), torch.zeros(p.shape, dtype=torch.float64)) for p in params]
    scale = torch.tensor([0.5], device=device)
    for t in (1, 2, 3):
        opt.step(grads, step=t, grad_scale=scale, **HOW)
        want = [ref.adamw(*(w[0], g.double().cpu(), *w[1:]), step=t, grad_scale=0.5, **HOW) for w, g in zip(want, grads)]
    m, v = opt.moments()
    for i, (p, at) in enumerate(zip(params, opt.offsets)):
        n = p.numel()
        # nine roundings in three steps, of the parameter and of updates of at most a few lr
        ref.close(p, want[i][0], 9 * 2.0 ** -24 * want[i][0].abs() + 2.0 ** -20 * 4 * HOW["lr"])
        ref.close(m[at:at + n], want[i][1], 2.0 ** -20 * torch.full((n,), 0.01, dtype=torch.float64))
        ref.close(v[at:at + n], want[i][2], 2.0 ** -20 * want[i][2])
        if copy:
            assert torch.equal(copies[i], p.to(copy))


@gpu
@pytest.mark.parametrize("shift", [0, 1])
def test_adamw_in_8_bits(shift):
    device = cuda_or_skip()
    params, grads, copies = adamw_tensors(device, SIZES, BF16, BF16, shift)
    grads[5][:512] = 0.0          # two blocks without any gradient
    grads[6][:100] = 0.0          # and a part of one
    opt = layer.AdamW(params, copies=copies, state_bits=8)
    for t in (1, 2, 3):
        before = [p.double().cpu() for p in params]
        m0, v0 = (x.double().cpu() for x in opt.moments())
        opt.step(grads, step=t, **HOW)
        m1, v1 = (x.cpu() for x in opt.moments())
        for i, (p, at) in enumerate(zip(params, opt.offsets)):
            n = p.numel()
            if n == 0:
                continue
            want = ref.adamw(before[i], grads[i].double().cpu(), m0[at:at + n], v0[at:at + n], step=t, **HOW)
            ref.close(p, want[0], 3 * 2.0 ** -24 * want[0].abs() + 2.0 ** -20 * 12 * HOW["lr"])
            assert torch.equal(copies[i], p.to(BF16))
            blocks = -(-n // 256)
            full = lambda x: torch.nn.functional.pad(x, (0, blocks * 256 - n)).view(blocks, 256)  # noqa: E731
            # half a step of the block's scale, and the 32-bit arithmetic before it
            m, root = full(want[1]), full(want[2]).sqrt()
            off = (full(m1[at:at + n].double()) - m).abs() - (0.5 * (1 + 2.0 ** -12) + 127 * 2.0 ** -21) * m.abs().amax(1, keepdim=True) / 127
            assert float(off.max()) <= 0
            got = full(v1[at:at + n].double()).sqrt()
            step = root.amax(1, keepdim=True) / 255
            allowed = torch.where(root < step, step - root, (0.5 * (1 + 2.0 ** -12) + 255 * 2.0 ** -21) * step).maximum((0.5 + 255 * 2.0 ** -21) * step)
            assert float(((got - root).abs() - allowed).max()) <= 2.0 ** -20 * float(step.max())
            assert torch.equal(got == 0, root == 0)
    assert int(opt.state["m"][opt.offsets[5]:opt.offsets[5] + 512].count_nonzero()) == 0


@gpu
def test_adamw_codes_are_those_of_32_bit_arithmetic():
    """Unfused sums and correctly rounded roots and quotients: the same codes and scales as elementary tensor operations give."""
    device = cuda_or_skip()
    params, grads, _ = adamw_tensors(device, [70000], F32, None)
    opt = layer.AdamW(params, state_bits=8)
    opt.state["m"].copy_(normal(5, opt.size, by=40).clamp(-127, 127))
    opt.state["v"].copy_(normal(6, opt.size, by=80).abs().clamp(1, 255))
    opt.state["m_scale"].copy_(normal(7, opt.size // 256, at=2e-4, by=2e-5))
    opt.state["v_scale"].copy_(normal(8, opt.size // 256, at=2e-4, by=2e-5))
    opt.state["m"][70000:], opt.state["v"][70000:] = 0, 0
    m, v = opt.moments()
    g = torch.nn.functional.pad(grads[0], (0, opt.size - 70000))
    m = m * 0.9 + g * (1 - 0.9)
    v = v * 0.99 + (g * g) * (1 - 0.99)
    m, u = m.view(-1, 256), v.sqrt().view(-1, 256)
    opt.step(grads, **HOW)
    top = m.abs().amax(1)
    assert torch.equal(opt.state["m_scale"], top * (1 / 127))
    assert torch.equal(opt.state["m"].view(-1, 256), (m * (127 / top)[:, None]).round().to(torch.int8))
    top = u.amax(1)
    assert torch.equal(opt.state["v_scale"], top * (1 / 255))
    code = (u * (255 / top)[:, None]).round()
    assert torch.equal(opt.state["v"].view(-1, 256), torch.where(u > 0, code.clamp(min=1), code).to(torch.uint8))


@gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_gradients_that_are_no_numbers(bits):
    """An infinite or undefined gradient spoils its element, and with 8 bits its block of 256, and nothing else."""
    device = cuda_or_skip()
    params, grads, _ = adamw_tensors(device, [1024, 300], F32, None)
    grads[0][300], grads[1][299] = float("nan"), float("inf")
    opt = layer.AdamW(params, state_bits=bits)
    opt.step(grads, **HOW)
    m, _ = opt.moments()
    bad = torch.zeros(opt.size, dtype=torch.bool)
    if bits == 8:
        bad[256:512] = True
        bad[1024 + 256:1024 + 300] = True
        assert torch.equal(~m.isfinite().cpu()[:1324], bad[:1324])
    else:
        bad[300] = bad[1024 + 299] = True
        assert torch.equal(~m.isfinite().cpu(), bad)
    assert int((~params[0].isfinite()).sum()) == 1 and int((~params[1].isfinite()).sum()) == 1


@gpu
def test_adamw_many_tensors_and_replaced_gradients():
    """More tensors than a launch names, and gradients that lie elsewhere at every step."""
    device = cuda_or_skip()
    sizes = [(37 * i) % 700 + 1 for i in range(901)]
    params, grads, _ = adamw_tensors(device, sizes, F32, None)
    whole = [torch.cat([p.clone() for p in params])]
    opt, one = layer.AdamW(params), layer.AdamW(whole)
    for t in (1, 2):
        fresh = [g.clone() for g in grads]
        opt.step(fresh, step=t, **HOW)
        one.step([torch.cat(fresh)], step=t, **HOW)
    assert torch.equal(torch.cat(params), whole[0])


@gpu
def test_adamw_state_is_saved_and_restored():
    device = cuda_or_skip()
    params, grads, _ = adamw_tensors(device, SIZES, BF16, None)
    start = [p.clone() for p in params]
    opt = layer.AdamW(params, state_bits=8)
    opt.step(grads, step=1, **HOW)
    middle, saved = [p.clone() for p in params], {n: t.clone() for n, t in opt.state.items()}
    opt.step(grads, step=2, **HOW)
    other = layer.AdamW(middle, state_bits=8)
    for n, t in saved.items():
        other.state[n].copy_(t)
    other.step(grads, step=2, **HOW)
    assert all(torch.equal(a, b) for a, b in zip(params, middle)) and not torch.equal(params[-1], start[-1])


@gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_calls_replayed_in_a_graph(bits):
    """A layer's calls, captured, give on every replay the bits that they give by themselves on the same inputs."""
    device = cuda_or_skip()
    x, f, w = normal(1, 64, 256, dtype=BF16).to(device), normal(2, 64, 256, dtype=BF16).to(device), normal(3, 256, dtype=BF16).to(device)
    q, k, v, do = (t.to(device) for t in attention_case(5, 2, 200, 200, 4, 2, 64, BF16))
    cache = normal(9, 2, 600, 2, 64, dtype=BF16).to(device)
    params, grads = [normal(11, n).to(device) for n in (300, 5000)], [normal(12, n).to(device) for n in (300, 5000)]
    start = [p.clone() for p in params]
    opt = layer.AdamW(params, state_bits=bits)

    def calls():
        r = layer.block_norm(x, f, entry_weight=w, exit_weight=w)
        g = layer.block_norm_backward(r.residual, r.normed, x, f, r.stats, entry_weight=w, exit_weight=w)
        out, lse = layer.window_attention(q, k, v, window=50, sinks=3)
        back = layer.window_attention_backward(do, q, k, v, out, lse, window=50, sinks=3)
        one = layer.window_attention(q[:, :1], cache, cache)
        opt.step(grads, lr=1e-2)
        return [t for t in (*r, *g, out, lse, *back, *one, *params, *opt.state.values()) if t is not None]

    def reset(seed):
        for t, s in ((x, 0), (f, 1), (q, 2), (cache, 3)):
            t.copy_(normal(seed + s, *t.shape, dtype=BF16))
        for p, s in zip(params, start):
            p.copy_(s)
        for t in opt.state.values():
            t.copy_(torch.zeros_like(t))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = calls()
    for seed in (100, 200, 300, 400):
        reset(seed)
        want = [t.clone() for t in calls()]
        torch.cuda.synchronize()
        reset(seed)
        graph.replay()
        torch.cuda.synchronize()
        for i, (got, w0) in enumerate(zip(held, want)):
            assert torch.equal(got, w0), (seed, i)


@gpu
def test_adamw_refusals():
    device = cuda_or_skip()
    p = torch.ones(8, 4, device=device)
    for error, a, k in ((ValueError, ([],), {}), (TypeError, ([p.half()],), {}), (ValueError, ([p.t()],), {}), (ValueError, ([p],), {"state_bits": 16}), (TypeError, ([p],), {"copies": [p]}),
                        (ValueError, ([p, p],), {"copies": [p.half()]}), (ValueError, ([p],), {"copies": [p.half()[:4]]}), (ValueError, ([p, p],), {"copies": [p.half(), None]})):
        with pytest.raises(error):
            layer.AdamW(*a, **k)
    opt = layer.AdamW([p])
    for error, g, k in ((ValueError, [], {}), (ValueError, [p[:4]], {}), (TypeError, [p.double()], {}), (ValueError, [p], {"step": 0}), (ValueError, [p], {"betas": (1.0, 0.9)}),
                        (ValueError, [p], {"grad_scale": torch.ones(2, device=device)}), (ValueError, [p.t().contiguous().t()], {}), (ValueError, [p.cpu()], {})):
        with pytest.raises(error):
            opt.step(g, lr=0.1, **k)
    opt.state["m"] = opt.state["m"][1:]
    with pytest.raises(ValueError):
        opt.step([p], lr=0.1)
