"""Log-probabilities of taken tokens and the policy's clipped loss against the definition in 64 bits, with bounds that follow from the
kernels' arithmetic; without a GPU: the definition's gradients against differences, and what is refused."""
import math

import pytest
import torch

from superscaler_amd import layer
from superscaler_amd.evaluator import AceError
from tests.layer_reference import SMALLEST, UNIT, close

gpu = pytest.mark.gpu
BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
E24 = 2.0 ** -24


def cuda_or_skip():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


def random(seed, *shape, by=1.0, dtype=F32):
    return (by * torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=F64)).to(dtype)


def logprobs(logits, targets):
    """In 64 bits: 0 where there is no target."""
    there = (targets >= 0) & (targets < logits.shape[-1])
    all_ = torch.log_softmax(logits.double(), -1)
    return torch.where(there, all_.gather(-1, targets.long().clamp(0, logits.shape[-1] - 1).unsqueeze(-1)).squeeze(-1), torch.zeros((), dtype=F64)), there


def policy(logits, targets, old_logp, advantages, ref_logp=None, weights=None, clip=(0.2, 0.2), kl_weight=0.0):
    """(loss, logp) in 64 bits, differentiable."""
    logp, there = logprobs(logits, targets)
    w = torch.full_like(logp, 1 / max(1, logp.numel())) if weights is None else weights.double()
    part = there & (w != 0)
    zero = torch.zeros((), dtype=F64)
    logp_, old, A = (torch.where(part, t.double(), zero) for t in (logp, old_logp, advantages))
    ratio = torch.exp(logp_ - old)
    each = -torch.minimum(ratio * A, ratio.clamp(1 - clip[0], 1 + clip[1]) * A)
    if ref_logp is not None:
        away = torch.where(part, ref_logp.double(), zero) - logp_
        each = each + kl_weight * (torch.expm1(away) - away)
    return (torch.where(part, w, zero) * each).sum(), logp


def logp_bound(logits):
    """What logp may be off by: a lane adds up to vocab / 256 + 32 terms, each off by its exponential (two roundings of an argument of up
    to `spread` and one of 2^-23), and the result is rounded."""
    z = logits.double()
    fine = z.masked_fill(~z.isfinite(), 0)
    spread = float((fine.amax() - fine.amin()).clamp(max=100))
    return E24 * (logits.shape[-1] / 256 + 32 + 2 * spread + 8)


# ---- without a GPU -------------------------------------------------------------------------------------------------------------
def test_the_definition_s_gradients_against_differences():
    z = random(1, 4, 7, dtype=F64).requires_grad_()
    targets = torch.tensor([2, -100, 6, 0])
    old, A, ref = random(2, 4, by=0.2) - 2, random(3, 4), random(4, 4, by=0.2) - 2
    w = torch.tensor([0.5, 0.25, 0.0, 0.25])

    def loss(x):
        return policy(x, targets, old, A, ref, w, (0.3, 0.1), 0.4)[0]
    grad, = torch.autograd.grad(loss(z), z)
    assert (grad[1] == 0).all() and (grad[2] == 0).all()
    h = 1e-6
    for r in range(4):
        for c in range(7):
            step = torch.zeros_like(z)
            step[r, c] = h
            assert abs(float(loss(z.detach() + step) - loss(z.detach() - step)) / (2 * h) - float(grad[r, c])) < 1e-8


def test_refusals_of_the_c_entries():
    lib = layer.load_library()

    def pack(rows=4, stride=16, vocab=16, dtype=1, bits=64, logits=64, targets=64, old=64, adv=64, low=0.8, high=1.2, kl=0.0):
        return layer._TOKEN_LOSS.pack(rows, stride, vocab, dtype, bits, logits, targets, old, adv, 0, 0, low, high, kl, 0.25)
    bad = ({"rows": -1}, {"vocab": 0}, {"dtype": 3}, {"dtype": -1}, {"bits": 16}, {"logits": 0}, {"targets": 0}, {"stride": 15}, {"logits": 65}, {"targets": 68})
    for change in bad:
        assert lib.ace_token_logprobs(pack(**change), 64, 64, None) == -1, change
        assert lib.ace_policy_loss_workspace_bytes(pack(**change)) == 0
    assert lib.ace_token_logprobs(None, 64, 64, None) == -1
    assert lib.ace_token_logprobs(pack(), None, 64, None) == -1 and lib.ace_token_logprobs(pack(), 64, None, None) == -1
    assert lib.ace_token_logprobs(pack(vocab=layer.MAX_VOCAB + 1, stride=1 << 30), 64, 64, None) == -2
    assert lib.ace_token_logprobs(pack(rows=0), None, None, None) == 0
    assert lib.ace_token_logprobs_backward(pack(), 64, 64, None, 16, None) == -1
    assert lib.ace_token_logprobs_backward(pack(), 64, 64, 128, 15, None) == -1
    assert lib.ace_token_logprobs_backward(pack(), 64, 64, 64, 32, None) == -1        # the logits themselves, but other rows
    for change in ({"low": -0.1}, {"low": 1.1}, {"high": 0.9}, {"kl": -1.0}, {"kl": math.nan}, {"old": 0}, {"adv": 0}):
        assert lib.ace_policy_loss(pack(**change), 64, 64, 64, 64, 64, 1 << 20, None) == -1, change
    assert lib.ace_policy_loss(pack(), 64, 64, 64, 64, 64, 31, None) == -1             # too little workspace
    assert lib.ace_policy_loss(pack(), None, 64, 64, 64, 64, 32, None) == -1
    assert lib.ace_policy_loss_gradient(pack(), None, 64, 64, 64, 64, None, 16, 64, 32, None) == -1
    assert lib.ace_policy_loss_workspace_bytes(pack()) == 32


def test_refusals():
    z, t, f = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64), torch.zeros(2)
    with pytest.raises(ValueError):
        layer.token_logprobs(z, t)              # on the host
    with pytest.raises(TypeError):
        layer.token_logprobs([1.0], t)
    with pytest.raises(ValueError):
        layer.policy_loss(z, t, f, f, clip=(1.5, 0.2))
    with pytest.raises(ValueError):
        layer.policy_loss(z, t, f, f, kl_weight=-1.0)
    with pytest.raises(TypeError):
        layer.policy_loss(z, t, None, f)
    with pytest.raises(ValueError):
        layer.policy_loss_gradient(z, t, f, f)


@pytest.mark.parametrize("shape,strides,want", [((3, 4, 7), (40, 10, 1), 10), ((3, 4, 7), (50, 10, 1), None), ((1, 7), (7, 1), 7), ((3, 7), (1, 3), None), ((4, 7), (0, 1), None),
                                                ((7,), (1,), 7), ((5, 1), (1, 9), 1), ((2, 1, 7), (9, 3, 1), 9)])
def test_rows_that_lie_evenly(shape, strides, want):
    assert layer._flat_rows(torch.empty(200).as_strided(shape, strides)) == want


# ---- on the GPU ----------------------------------------------------------------------------------------------------------------
def case(seed, rows, vocab, dtype, by=2.0, none=True, int32=False):
    z = random(seed, rows, vocab, by=by, dtype=dtype)
    gen = torch.Generator().manual_seed(seed + 1)
    targets = torch.randint(0, vocab, (rows,), generator=gen, dtype=torch.int32 if int32 else torch.int64)
    if none and rows > 2:
        targets[1], targets[-1] = -100, vocab
    return z, targets


def check_logprobs(device, z, targets, d_logp=None, out=None):
    want, there = logprobs(z, targets)
    zd, td = z.to(device), targets.to(device)
    r = layer.token_logprobs(zd, td)
    bound = logp_bound(z)
    close(r.logp, want, torch.full_like(want, bound))
    assert (r.logp.cpu()[~there] == 0).all()
    d = random(7, *targets.shape) if d_logp is None else d_logp
    got = layer.token_logprobs_backward(d.to(device), zd, td, r.stats, out=out)
    again = layer.token_logprobs_backward(d.to(device), zd, td, r.stats)
    assert torch.equal(got, again)
    p = torch.softmax(z.double(), -1)
    hot = torch.zeros_like(p).scatter_(-1, targets.long().clamp(0, z.shape[-1] - 1).unsqueeze(-1), 1.0)
    part = (there & (d != 0)).unsqueeze(-1)
    want = torch.where(part, d.double().unsqueeze(-1) * (hot - p), torch.zeros((), dtype=F64))
    slack = d.double().abs().unsqueeze(-1) * (p * (2 * bound + 4 * E24) + 2 * E24 * hot) + SMALLEST[z.dtype]
    close(got, want, slack)
    assert (got.cpu()[~part.squeeze(-1)] == 0).all()


@gpu
@pytest.mark.parametrize("vocab", [1, 2, 7, 64, 500, 2047, 2048, 2056, 8191, 8192, 8193, 16385, 32001, 51200, 131072, 150001])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_logprobs_of_every_size(vocab, dtype):
    device = cuda_or_skip()
    check_logprobs(device, *case(vocab, 5, vocab, dtype, int32=vocab % 2 == 0))


@gpu
@pytest.mark.parametrize("rows,vocab", [(1, 51200), (511, 8200), (512, 8200), (513, 1000), (3000, 33)])
def test_logprobs_of_many_rows(rows, vocab):
    device = cuda_or_skip()
    check_logprobs(device, *case(rows, rows, vocab, BF16))


@gpu
def test_no_rows_and_leading_dimensions():
    device = cuda_or_skip()
    z = torch.empty(0, 3, 40, device=device)
    t = torch.empty(0, 3, dtype=torch.int64, device=device)
    r = layer.token_logprobs(z, t)
    assert r.logp.shape == (0, 3) and r.stats.shape == (0, 3, 2)
    assert layer.token_logprobs_backward(r.logp, z, t, r.stats).shape == z.shape
    f = torch.empty(0, 3, device=device)
    p, g = layer.policy_loss_gradient(z, t, f, f)
    assert float(p.loss) == 0.0 and g.shape == z.shape
    z, t = case(1, 6, 70, F32)
    want = layer.token_logprobs(z.to(device), t.to(device)).logp
    assert torch.equal(layer.token_logprobs(z.view(2, 3, 70).to(device), t.view(2, 3).to(device)).logp.view(-1), want)
    one = layer.token_logprobs(z[0].to(device), t[0].to(device))
    assert one.logp.shape == () and torch.equal(one.logp, want[0])


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_of_other_strides_and_places(dtype):
    """Rows that begin at odd elements, rows of a padded vocabulary, rows that do not lie evenly; gradients into rows of their own stride,
    and into the logits, whose padding stays."""
    device = cuda_or_skip()
    z, t = case(3, 6, 1001, dtype)
    want = layer.token_logprobs(z.to(device), t.to(device))
    wide = torch.full((6, 1024), 5.0, dtype=dtype, device=device)
    wide[:, 3:1004] = z.to(device)
    view = wide[:, 3:1004]
    got = layer.token_logprobs(view, t.to(device))
    close(got.logp, want.logp.double(), torch.full_like(want.logp.double().cpu(), 2 * logp_bound(z)))
    d = random(9, 6).to(device)
    ref = layer.token_logprobs_backward(d, z.to(device), t.to(device), got.stats)
    for other in (view.t().contiguous().t(), wide.view(2, 3, 1024)[:, :2, 3:1004]):
        tt = t.to(device) if other.dim() == 2 else t.view(2, 3)[:, :2].to(device)
        assert torch.equal(layer.token_logprobs(other, tt).logp, layer.token_logprobs(other.contiguous(), tt).logp)
    out = torch.full((6, 1010), 7.0, dtype=dtype, device=device)
    assert torch.equal(layer.token_logprobs_backward(d, view, t.to(device), got.stats, out=out[:, 5:1006]), ref)
    assert (out[:, :5] == 7).all() and (out[:, 1006:] == 7).all()
    layer.token_logprobs_backward(d, view, t.to(device), got.stats, out=view)
    assert torch.equal(view, ref) and (wide[:, :3] == 5).all() and (wide[:, 1004:] == 5).all()


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("vocab", [5, 64, 1001, 20003])
def test_the_policy_s_gradient_goes_anywhere(dtype, vocab):
    """Rows of logits and of their gradient that begin at any element, as far from 16 bytes as there are; into the logits; what is beside them stays.  Where a
    row's pieces begin, other lanes add up other elements: results differ by what the sums' order gives."""
    device = cuda_or_skip()
    z, t, c = policy_case(vocab, 9, vocab, dtype)
    given = (t.to(device), c["old_logp"].to(device), c["advantages"].to(device))
    how = dict(ref_logp=c["ref_logp"].to(device), weights=c["weights"].to(device), kl_weight=0.1)
    want, grad = layer.policy_loss_gradient(z.to(device), *given, **how)
    bound = 2 * logp_bound(z)
    for at in range(0, 9):
        wide = torch.full((9, vocab + 19), 5.0, dtype=dtype, device=device)
        view = wide[:, at:at + vocab]
        view.copy_(z)
        out = torch.full((9, vocab + 13), 7.0, dtype=dtype, device=device)
        got, g = layer.policy_loss_gradient(view, *given, **how, out=out[:, 9 - at:9 - at + vocab])
        close(got.logp, want.logp.double(), torch.full((9,), bound))
        # (both are rounded, and their derivatives are as far apart as ratios of these log-probabilities)
        close(g, grad.double(), (grad.double().abs().amax(-1, keepdim=True) * (8 * bound) + grad.double().abs() * UNIT[dtype]).cpu() + 2 * SMALLEST[dtype])
        assert (out[:, :9 - at] == 7).all() and (out[:, 9 - at + vocab:] == 7).all() and (wide[:, :at] == 5).all() and (wide[:, at + vocab:] == 5).all()
        inside, same = layer.policy_loss_gradient(view, *given, **how, out=view)
        assert torch.equal(view, g) and torch.equal(inside.loss, got.loss) and same is view
        assert (wide[:, :at] == 5).all() and (wide[:, at + vocab:] == 5).all()


@gpu
def test_refused_on_the_gpu():
    device = cuda_or_skip()
    z, t = (x.to(device) for x in case(3, 6, 64, F32))
    f = torch.zeros(6, device=device)
    stats = layer.token_logprobs(z, t).stats
    for call, kind in ((lambda: layer.token_logprobs(z.double(), t), TypeError), (lambda: layer.token_logprobs(z, t.float()), TypeError),
                       (lambda: layer.token_logprobs(z, t[:5]), ValueError), (lambda: layer.token_logprobs(z[:, :0], t), ValueError),
                       (lambda: layer.token_logprobs_backward(f.double(), z, t, stats), TypeError), (lambda: layer.token_logprobs_backward(f, z, t, stats[:5]), ValueError),
                       (lambda: layer.token_logprobs_backward(f, z, t, stats, out=z[:5]), ValueError),
                       (lambda: layer.token_logprobs_backward(f, z, t, stats, out=z.bfloat16()), TypeError),
                       (lambda: layer.token_logprobs_backward(f, z[:, :60], t, stats, out=z[:, 1:61]), ValueError),
                       (lambda: layer.token_logprobs_backward(f, z, t, stats, out=torch.empty(64, 6, device=device).t()), ValueError),
                       (lambda: layer.policy_loss(z, t, f, f[:5]), ValueError), (lambda: layer.policy_loss(z, t, f, f, weights=f.double()), TypeError),
                       (lambda: layer.policy_loss(z, t, f, f, ref_logp=f.cpu()), ValueError), (lambda: layer.policy_loss_gradient(z, t, f, f, d_loss=f), ValueError)):
        with pytest.raises(kind):
            call()


def policy_case(seed, rows, vocab, dtype, by=2.0):
    z, t = case(seed, rows, vocab, dtype, by)
    logp = logprobs(z, t)[0]
    A, w = random(seed + 4, rows), torch.rand(rows, generator=torch.Generator().manual_seed(seed + 5)) / rows
    if rows > 5:
        w[2], A[3] = 0.0, 0.0
    return z, t, dict(old_logp=(logp + random(seed + 2, rows, by=0.3)).float(), advantages=A, ref_logp=(logp + random(seed + 3, rows, by=0.4)).float(), weights=w)


def check_policy(device, z, t, c, clip=(0.2, 0.28), kl_weight=0.1, d_loss=None):
    how = dict(clip=clip, kl_weight=kl_weight)
    given = [x.to(device) for x in (z, t)] + [c["old_logp"].to(device), c["advantages"].to(device)]
    opt = {k: c[k].to(device) for k in ("ref_logp", "weights") if c.get(k) is not None}
    r = layer.policy_loss(*given, **opt, **how)
    g = None if d_loss is None else torch.tensor([d_loss], device=device)
    again, grad = layer.policy_loss_gradient(*given, **opt, **how, d_loss=g)
    x = z.double().requires_grad_()
    logp = logprobs(x, t)[0]
    logp.retain_grad()
    # (the loss by each log-probability: the graph is cut there)
    cut = logp.detach().requires_grad_()
    n = max(1, t.numel())
    w = torch.full((t.numel(),), 1 / n, dtype=F64) if c.get("weights") is None else c["weights"].double()
    there = logprobs(z, t)[1]
    part = there & (w != 0)
    zero = torch.zeros((), dtype=F64)
    safe = {k: torch.where(part, c[k].double(), zero) for k in ("old_logp", "advantages", "ref_logp") if c.get(k) is not None}
    ratio = torch.exp(torch.where(part, cut, zero) - safe["old_logp"])
    A = safe["advantages"]
    terms = -torch.minimum(ratio * A, ratio.clamp(1 - clip[0], 1 + clip[1]) * A)
    size = ratio * A.abs()
    if "ref_logp" in safe:
        away = safe["ref_logp"] - torch.where(part, cut, zero)
        terms = terms + kl_weight * (torch.expm1(away) - away)
        size = size + kl_weight * (away.exp() + away.abs() + 1)
    each = torch.where(part, w, zero) * terms
    d = torch.autograd.grad(each.sum(), cut)[0]
    bound = logp_bound(z)
    weighed = (torch.where(part, w, zero) * size).detach() * (2 * bound + 2 ** -40)
    for got in (r, again):
        close(got.logp, logp.detach(), torch.full_like(logp.detach(), bound))
        close(got.loss, each.sum().detach(), weighed.sum())
        close(got.d_logp, d, weighed)
        assert (got.d_logp.cpu()[~part] == 0).all()
    p = torch.softmax(z.double(), -1)
    hot = torch.zeros_like(p).scatter_(-1, t.long().clamp(0, z.shape[-1] - 1).unsqueeze(-1), 1.0)
    s = d_loss or 1.0
    want = torch.where((part & (d != 0)).unsqueeze(-1), s * d.unsqueeze(-1) * (hot - p), zero)
    slack = s * (d.abs().unsqueeze(-1) * (p * (2 * bound + 8 * E24) + 4 * E24 * hot) + weighed.unsqueeze(-1) * (p + hot)) + SMALLEST[z.dtype]
    close(grad, want, slack)
    assert (grad.cpu()[~part] == 0).all()
    assert torch.equal(grad, layer.policy_loss_gradient(*given, **opt, **how, d_loss=g)[1])
    return r, grad


@gpu
@pytest.mark.parametrize("vocab", [1, 3, 63, 64, 1000, 2049, 4096, 8193, 12800, 25601, 32001, 51200, 65537, 131072, 131080])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_policy_of_every_size(vocab, dtype):
    device = cuda_or_skip()
    check_policy(device, *policy_case(vocab + 1, 7, vocab, dtype))


@gpu
@pytest.mark.parametrize("rows,vocab", [(1, 9000), (600, 5000), (2111, 130)])
@pytest.mark.parametrize("plain", [False, True])
def test_policy_of_many_rows(rows, vocab, plain):
    device = cuda_or_skip()
    z, t, c = policy_case(rows, rows, vocab, F16)
    if plain:
        c = dict(c, ref_logp=None, weights=None)
    check_policy(device, z, t, c, clip=(0.0, 0.0) if plain else (1.0, 3.0), d_loss=1024.0)


@gpu
@pytest.mark.parametrize("low,high", [(0.2, 0.2), (0.2, 0.28), (0.1, 0.5)])
def test_ratios_next_to_the_border(low, high):
    """Where logp is -log 4 but for 64 bits' rounding, an old log-probability of 32 bits one step before or behind the border decides."""
    device = cuda_or_skip()
    z = torch.zeros(8, 4)
    t = torch.zeros(8, dtype=torch.int64)
    logp = -math.log(4.0)
    old, A, free = [], [], []
    for sign, border in ((1.0, 1 + high), (-1.0, 1 - low)):
        at = torch.tensor(logp - math.log(border), dtype=F64)
        near = at.float()
        for k in range(-2, 2):
            value = near.clone()
            for _ in range(abs(k)):
                value = torch.nextafter(value, torch.tensor(math.inf if k > 0 else -math.inf))
            old.append(float(value)), A.append(sign)
            ratio = math.exp(logp - float(value))
            free.append(ratio <= border if sign > 0 else ratio >= border)
    r = layer.policy_loss(z.to(device), t.to(device), torch.tensor(old, device=device), torch.tensor(A, device=device), clip=(low, high))
    assert [bool(d != 0) for d in r.d_logp.cpu()] == free


@gpu
def test_what_takes_no_part_may_be_anything():
    """Logits of rows without a target, all numbers of rows of weight 0: the others' results have the same bits, theirs are 0."""
    device = cuda_or_skip()
    for dtype, vocab in ((BF16, 3000), (F32, 70000)):
        z, t, c = policy_case(11, 9, vocab, dtype)
        t[4] = 1 << 40
        c["weights"][5] = 0.0
        want, grad = layer.policy_loss_gradient(*(x.to(device) for x in (z, t, c["old_logp"], c["advantages"])), ref_logp=c["ref_logp"].to(device), weights=c["weights"].to(device),
                                                kl_weight=0.2)
        z[[1, 4, 8]], z[5] = math.nan, math.inf
        for k in ("old_logp", "advantages", "ref_logp"):
            c[k][[1, 2, 4, 5, 8]] = torch.tensor([math.nan, math.inf, -math.inf, math.nan, math.nan])
        c["weights"][1] = math.nan
        got, grad2 = layer.policy_loss_gradient(*(x.to(device) for x in (z, t, c["old_logp"], c["advantages"])), ref_logp=c["ref_logp"].to(device), weights=c["weights"].to(device),
                                                kl_weight=0.2)
        assert torch.equal(want.loss, got.loss) and torch.equal(want.d_logp, got.d_logp) and torch.equal(grad, grad2)
        keep = [i for i in range(9) if i != 5]
        assert torch.equal(want.logp[keep], got.logp[keep]) and (grad2[[1, 2, 4, 5, 8]] == 0).all()
        d = torch.ones(9, device=device)
        d[5] = 0.0
        assert (layer.token_logprobs_backward(d, z.to(device), t.to(device), got.stats)[[1, 4, 5, 8]] == 0).all()


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("vocab", [700, 20000])
def test_tokens_that_cannot_be_taken_and_what_is_no_number(dtype, vocab):
    device = cuda_or_skip()
    z, t = case(21, 6, vocab, dtype, none=False)
    low = torch.finfo(dtype).min
    z[0, 5:], z[1, 1:] = -math.inf, low
    t[0], t[1] = 3, 0
    z[2, 10], z[3, 600] = math.nan, math.inf
    z[4] = -math.inf
    zd, td = z.to(device), t.to(device)
    r = layer.token_logprobs(zd, td)
    want = logprobs(z, t)[0]
    logp = r.logp.cpu().double()
    assert logp[[2, 3, 4]].isnan().all() and (logp[[0, 1, 5]] - want[[0, 1, 5]]).abs().max() < logp_bound(z[[0, 5]]) + 1e-12
    g = layer.token_logprobs_backward(torch.ones(6, device=device), zd, td, r.stats).cpu()
    assert g[[2, 3, 4]].isnan().all() and g[[0, 1, 5]].isfinite().all()
    assert (g[0, 5:] == 0).all() and (g[1, 1:] == 0).all() and float(g[1, 0]) == 0.0


@gpu
def test_results_of_one_call_are_none_of_another_s():
    """Captured, replayed with other inputs and with eager calls between; on two streams at once; the loss is the same bits every time."""
    device = cuda_or_skip()
    z, t, c = policy_case(31, 300, 9000, BF16)
    z, t = z.to(device), t.to(device)
    c = {k: v.to(device) for k, v in c.items()}
    how = dict(ref_logp=c["ref_logp"], weights=c["weights"], kl_weight=0.1)
    eager = layer.policy_loss_gradient(z, t, c["old_logp"], c["advantages"], **how)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = layer.policy_loss_gradient(z, t, c["old_logp"], c["advantages"], **how)
    for k in range(4):
        z.copy_(random(40 + k, 300, 9000, dtype=BF16))
        graph.replay()
        want = layer.policy_loss_gradient(z, t, c["old_logp"], c["advantages"], **how)
        torch.cuda.synchronize()
        for a, b in zip(held[0] + (held[1],), want[0] + (want[1],)):
            assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = layer.policy_loss_gradient(z, t, c["old_logp"], c["advantages"], **how)
    mine = layer.policy_loss_gradient(z, t, c["old_logp"], c["advantages"], **how)
    torch.cuda.synchronize()
    assert torch.equal(other[1], mine[1]) and torch.equal(other[0].loss, mine[0].loss) and not torch.equal(eager[1], mine[1])


@gpu
def test_automatic_differentiation_is_told():
    device = cuda_or_skip()
    z, t = (x.to(device) for x in case(3, 6, 64, F32))
    z.requires_grad_()
    f = torch.zeros(6, device=device)
    with pytest.raises(AceError):
        layer.token_logprobs(z, t).logp.sum().backward()
    with pytest.raises(AceError):
        layer.policy_loss(z, t, f, f).loss.backward()
    with pytest.raises(AceError):
        layer.policy_loss_gradient(z, t, f, f)[0].loss.backward()
    with torch.no_grad():
        assert not layer.policy_loss(z, t, f, f).loss.requires_grad
    x = z.detach().clone()
    y = x * torch.ones((), device=device, requires_grad=True)
    with torch.no_grad():
        layer.token_logprobs_backward(f + 1, x, t, layer.token_logprobs(x, t).stats, out=x)
    with pytest.raises(RuntimeError):      # (x was kept for that product's gradient and has changed)
        y.sum().backward()
