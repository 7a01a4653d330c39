"""The norm of many gradients and clipping against 64 bits; without a GPU: what is refused."""
import ctypes
import math

import pytest
import torch

from superscaler_amd import layer
from superscaler_amd.evaluator import AceError

gpu = pytest.mark.gpu
BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
E24 = 2.0 ** -24


def cuda_or_skip():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


def random(seed, *shape, by=1.0, dtype=F32):
    return (by * torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=F64)).to(dtype)


def near(got, want, units=1.0):
    """One rounding to 32 bits, and the sums' own in 64 (10^5 of them at most: 2^-36).  What is past the largest number of 32 bits by half a
    step is infinite there, and below the normal ones a step is 2^-149."""
    got, want = float(got), float(want)
    if abs(want) > 2.0 ** 128 * (1 - 2.0 ** -25):
        want = math.copysign(math.inf, want)
    return got == want or abs(got - want) <= abs(want) * (units * E24 + 2 ** -36) + 2.0 ** -150


# ---- without a GPU -------------------------------------------------------------------------------------------------------------
def table(*tensors):
    return (ctypes.c_int64 * (3 * len(tensors)))(*(v for t in tensors for v in t))


def test_refusals_of_the_c_entries():
    lib = layer.load_library()
    good = table((64, 10, 1))
    at = ctypes.addressof
    assert lib.ace_gradient_norm_workspace_bytes(at(good), 1) == 8 * (1 + 1 + 1)
    for bad in (table((64, -1, 1)), table((64, 1, 3)), table((0, 1, 1)), table((65, 1, 1)), table((66, 1, 0)), table((64, 1, -1))):
        assert lib.ace_gradient_norm(at(bad), 1, 1.0, None, 64, 64, 64, 1 << 20, None) == -1
        assert lib.ace_gradient_scale(at(bad), 1, 64, None) == -1
        assert lib.ace_gradient_norm_workspace_bytes(at(bad), 1) == 0
    assert lib.ace_gradient_norm(None, 1, 1.0, None, 64, 64, 64, 1 << 20, None) == -1
    assert lib.ace_gradient_norm(at(good), 0, 1.0, None, 64, 64, 64, 1 << 20, None) == -1
    assert lib.ace_gradient_norm(at(good), -1, 1.0, None, 64, 64, 64, 1 << 20, None) == -1
    for limit in (-1.0, math.nan):
        assert lib.ace_gradient_norm(at(good), 1, limit, None, 64, 64, 64, 1 << 20, None) == -1
    assert lib.ace_gradient_norm(at(good), 1, 1.0, None, 64, 64, 64, 23, None) == -1
    assert lib.ace_gradient_norm(at(good), 1, 1.0, None, None, 64, 64, 24, None) == -1
    assert lib.ace_gradient_norm(at(good), 1, 1.0, None, 64, None, 64, 24, None) == -1
    assert lib.ace_gradient_norm(at(good), 1, 1.0, None, 64, 64, 68, 24, None) == -1
    assert lib.ace_gradient_norm(at(table((64, (1 << 37) + 1, 1))), 1, 1.0, None, 64, 64, 64, 1 << 62, None) == -2
    assert lib.ace_gradient_norm(at(good), (1 << 20) + 1, 1.0, None, 64, 64, 64, 1 << 62, None) == -2
    assert lib.ace_gradient_scale(at(good), 1, None, None) == -1 and lib.ace_gradient_scale(None, 0, None, None) == 0


def test_refusals():
    with pytest.raises(ValueError):
        layer.gradient_norm([])
    with pytest.raises(ValueError):
        layer.gradient_norm([torch.ones(3)])
    with pytest.raises(TypeError):
        layer.gradient_norm([1.0])
    with pytest.raises(ValueError):
        layer.clip_gradients([], 1.0)


@pytest.mark.parametrize("shape,strides,want", [((3, 4), (4, 1), True), ((3, 4), (1, 3), True), ((3, 4), (5, 1), False), ((2, 3, 4), (4, 8, 1), True), ((3, 1), (1, 7), True),
                                                ((3, 4), (0, 1), False), ((0, 4), (9, 2), True), ((5,), (2,), False), ((), (), True)])
def test_tensors_without_gaps(shape, strides, want):
    assert layer._dense(torch.empty(100).as_strided(shape, strides)) is want


# ---- on the GPU ----------------------------------------------------------------------------------------------------------------
def check(grads, max_norm=None, gs=None, device="cuda:0"):
    wide = [g.double() for g in grads]
    s = 1.0 if gs is None else float(torch.tensor(gs, dtype=F32))
    norms = [math.sqrt(float(g.square().sum())) * abs(s) for g in wide]
    norm = math.sqrt(math.fsum(n * n for n in norms))
    scale = s * min(1.0, max_norm / (norm + 1e-6)) if max_norm else s
    on = [g.to(device) for g in grads]
    given = None if gs is None else torch.tensor([gs], device=device)
    r = layer.gradient_norm(on, max_norm=max_norm, grad_scale=given)
    assert r.norm.shape == (1,) and r.scale.shape == (1,) and r.norms.shape == (len(grads),)
    assert near(r.norm, norm) and near(r.scale, scale, 2.0), (float(r.norm), norm, float(r.scale), scale)
    assert all(near(a, b) for a, b in zip(r.norms.cpu(), norms))
    for g, before in zip(on, grads):
        assert torch.equal(g.cpu(), before)
    if max_norm is None:
        return r
    clipped = layer.clip_gradients(on, max_norm, grad_scale=given)
    assert all(torch.equal(a, b) for a, b in zip(clipped, r))
    factor = r.scale.cpu()
    for g, before in zip(on, grads):
        assert torch.equal(g.cpu(), before if float(factor) == 1.0 else (before.float() * factor).to(before.dtype))
    return r


@gpu
@pytest.mark.parametrize("n", [1, 2, 7, 8, 255, 2047, 2048, 2049, 16383, 16384, 16385, 100003])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_one_tensor_of_every_size(n, dtype):
    cuda_or_skip()
    check([random(n, n, dtype=dtype)], max_norm=0.5, gs=0.25)


@gpu
@pytest.mark.parametrize("count", [2, 3, 239, 240, 241, 500, 1201])
def test_many_tensors_of_every_type(count):
    """Empty ones among them, at the beginning, the end, and where a launch's list of tensors ends."""
    cuda_or_skip()
    kinds = (BF16, F32, F16)
    grads = [random(i, 0 if i % 5 == 0 or i in (239, 240) else 1 + 977 * i % 5000, by=10.0 ** (i % 7 - 3), dtype=kinds[i % 3]) for i in range(count)]
    check(grads, max_norm=3.0)
    check(grads[::-1], max_norm=1e9, gs=-2.0)


@gpu
def test_shapes_orders_and_places():
    device = cuda_or_skip()
    base = random(1, 40, 33, dtype=BF16)
    flat = torch.zeros(1321, dtype=BF16, device=device)[1:]        # begins at an odd element
    flat.copy_(base.view(-1))
    want = layer.gradient_norm([base.to(device)])
    for other in (flat, flat.view(40, 33).t(), flat.view(40, 33, 1).permute(2, 1, 0)):
        assert near(layer.gradient_norm([other]).norm, want.norm)
    gaps = torch.full((40, 50), 9.0, dtype=BF16, device=device)
    gaps[:, 5:38] = base.to(device)
    assert near(layer.gradient_norm([gaps[:, 5:38]]).norm, want.norm)
    with pytest.raises(ValueError):
        layer.clip_gradients([gaps[:, 5:38]], 1.0)
    r = layer.clip_gradients([flat.view(40, 33).t()], 1.0)
    assert torch.equal(flat.cpu(), (base.view(-1).float() * r.scale.cpu()).to(BF16))
    scalar = torch.tensor(3.0, device=device)
    assert float(layer.gradient_norm([scalar]).norm) == 3.0
    assert float(layer.gradient_norm([scalar, scalar]).norm) == float(torch.tensor(18.0, dtype=F64).sqrt().float())      # counted twice
    empty = layer.gradient_norm([torch.empty(0, device=device)], max_norm=1.0)
    assert float(empty.norm) == 0.0 and float(empty.scale) == 1.0 and float(empty.norms) == 0.0


@gpu
def test_clipping_writes_what_is_there_and_nothing_else():
    device = cuda_or_skip()
    whole = torch.full((70000,), 2.0, device=device)
    a, b = whole[3:20000], whole[20001:69990]
    layer.clip_gradients([b, a], 1e-3)
    left = torch.ones(70000, dtype=torch.bool)
    left[3:20000], left[20001:69990] = False, False
    assert (whole.cpu()[left] == 2.0).all() and (whole.cpu()[~left] < 1e-4).all()


@gpu
@pytest.mark.parametrize("size", [1e20, 3e38, 1e-25, 1e-38, 1e-44])
def test_squares_past_the_range_of_32_bits(size):
    cuda_or_skip()
    check([torch.full((5000,), size, dtype=F32), random(3, 100, by=size / 10)], max_norm=1e30)


@gpu
def test_what_is_no_number():
    device = cuda_or_skip()
    for value in (math.inf, -math.inf, math.nan):
        g = [torch.ones(20000, device=device), torch.ones(70, dtype=BF16, device=device)]
        g[0][17777] = value
        r = layer.gradient_norm(g, max_norm=1.0)
        if math.isnan(value):
            assert r.norm.isnan() and r.scale.isnan() and r.norms[0].isnan()
        else:
            assert r.norm.isinf() and float(r.scale) == 0.0 and r.norms[0].isinf()
        assert near(r.norms[1], math.sqrt(70))
        free = layer.gradient_norm(g)
        assert float(free.scale) == 1.0 and not free.norm.isfinite()
        layer.clip_gradients(g, 1.0)
        assert g[0][17777].isnan() and (g[1].isnan().all() if math.isnan(value) else (g[1] == 0).all())


@gpu
def test_refused_on_the_gpu():
    device = cuda_or_skip()
    a = torch.ones(100, device=device)
    for call, kind in ((lambda: layer.gradient_norm([a.double()]), TypeError), (lambda: layer.gradient_norm([a, a.cpu()]), ValueError),
                       (lambda: layer.gradient_norm([a], max_norm=0.0), ValueError), (lambda: layer.gradient_norm([a], max_norm=math.nan), ValueError),
                       (lambda: layer.gradient_norm([a], grad_scale=a), ValueError), (lambda: layer.clip_gradients([a, a], 1.0), ValueError),
                       (lambda: layer.clip_gradients([a[:60], a[59:]], 1.0), ValueError), (lambda: layer.clip_gradients([a.expand(3, 100)], 1.0), ValueError)):
        with pytest.raises(kind):
            call()
    assert (a == 1).all()


@gpu
def test_a_step_s_gradients_are_clipped_by_the_factor():
    """norm -> AdamW.step, captured and replayed with eager work between; the same bits as one after the other, and those of gradients that
    were clipped in place but for their rounding."""
    device = cuda_or_skip()
    sizes = (5000, 33, 70001)
    grads = [random(i, n, by=0.1).to(device) for i, n in enumerate(sizes)]

    def fresh():
        params = [random(10 + i, n).to(device) for i, n in enumerate(sizes)]
        return params, layer.AdamW(params)
    params, opt = fresh()
    held, opt2 = fresh()

    def step(o, g):
        o.step(g, lr=1e-2, step=3, grad_scale=layer.gradient_norm(g, max_norm=1.0).scale)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(opt2, grads)
    for k in range(4):
        for i, g in enumerate(grads):
            g.copy_(random(20 + 3 * k + i, sizes[i], by=0.05 * (k + 1)))
        graph.replay()
        step(opt, grads)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(params, held))
    inplace = [g.clone() for g in grads]
    layer.clip_gradients(inplace, 1.0)
    scale = layer.gradient_norm(grads, max_norm=1.0).scale
    assert float(scale) < 0.2 and all(torch.equal(a, g * scale) for a, g in zip(inplace, grads))


@gpu
def test_two_streams_at_once():
    device = cuda_or_skip()
    grads = [random(i, 30000 + i).to(device) for i in range(50)]
    want = layer.gradient_norm(grads, max_norm=1.0)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(layer.gradient_norm(grads, max_norm=1.0))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in got for a, b in zip(r, want))


@gpu
def test_automatic_differentiation_is_told():
    device = cuda_or_skip()
    g = torch.ones(10, device=device, requires_grad=True)
    with pytest.raises(AceError):
        layer.gradient_norm([g]).norm.sum().backward()
    x = torch.ones(10, device=device)
    y = x * torch.ones((), device=device, requires_grad=True)
    layer.clip_gradients([x], 0.5)
    with pytest.raises(RuntimeError):      # (x was kept for that product's gradient and has changed)
        y.sum().backward()
