"""The profiled layer over packed documents, its gradients as a policy's, and the command's options for them."""
import json
import math

import pytest
import torch

from superscaler_amd import layer, opgraph, profile_layer

gpu = pytest.mark.gpu


def cuda_or_skip():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")


@pytest.mark.parametrize("rows,seq,documents", [(1, 5, 1), (3, 64, 4), (2, 10, 40)])
def test_documents_fill_the_rows(rows, seq, documents):
    lengths = profile_layer.cut(rows, seq, documents, seed=2)
    assert len(lengths) == rows * documents and all(n >= 0 for n in lengths)
    assert [sum(lengths[i * documents:(i + 1) * documents]) for i in range(rows)] == [seq] * rows
    assert lengths == profile_layer.cut(rows, seq, documents, seed=2)


def test_options_that_make_no_sense_are_refused():
    for bad in (["--documents", "-1"], ["--clip", "0"]):
        with pytest.raises(SystemExit):
            profile_layer.main(["--workload", "gpt3_1_3b"] + bad)


@gpu
def test_packed_documents_are_what_each_is_alone():
    """Rows of a product of the matrix library may be summed in another order where there are more of them, so not the same bits: a
    few roundings to bfloat16 (2^-9 each) of some twenty tensors apart, as in the layer's test of gradients."""
    cuda_or_skip()
    net = profile_layer.GptLayer(256, window=20, sinks=2, seed=5)
    gen = torch.Generator(device="cuda").manual_seed(1)
    lengths = [70, 1, 0, 130, 55]
    x, block, dr, db = (torch.randn(256, 256, device="cuda", generator=gen).bfloat16() for _ in range(4))
    r, b, saved = net.forward(x, block, layer.Packing(lengths))
    d_x, d_block, grads = net.backward(dr, db, saved)
    sums, at = {n: torch.zeros_like(g, dtype=torch.float64) for n, g in grads.items()}, 0
    for n in filter(None, lengths):
        rows = slice(at, at + n)
        at += n
        r1, b1, saved1 = net.forward(x[None, rows], block[None, rows])
        d_x1, d_block1, grads1 = net.backward(dr[None, rows], db[None, rows], saved1)
        for got, want in ((r, r1), (b, b1), (d_x, d_x1), (d_block, d_block1)):
            assert float((got[rows].double() - want[0].double()).norm() / want.double().norm()) < 0.02
        for name, g in grads1.items():
            sums[name] += g.double()
    for name, g in grads.items():
        assert float((g.double() - sums[name]).norm() / sums[name].norm()) < 0.02, name


@gpu
def test_a_policy_s_gradients():
    """Packed attention, the loss and its gradient, the layer backward, the norm: against automatic differentiation of the same in 64 bits, with the bound of
    the layer's test of gradients (rounded tensors on the way, independent: 2^-9 sqrt(20), doubled)."""
    cuda_or_skip()
    lengths, vocab, tokens = [40, 3, 90], 777, 133
    policy = profile_layer.Policy(256, vocab, window=20, sinks=2, seed=5)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, block = (torch.randn(tokens, 256, device="cuda", generator=gen).bfloat16() for _ in range(2))
    targets = torch.randint(0, vocab, (tokens,), device="cuda", generator=gen)
    targets[::5] = -100
    packing = layer.Packing(lengths)
    logits, saved = policy.forward(x, block, packing)
    logp = layer.token_logprobs(logits, targets).logp
    # (away from the clipping's borders, which rounded logits would cross)
    step = torch.randint(0, 3, (tokens,), device="cuda", generator=gen).float() - 1
    old, ref, A = logp + 0.5 * step, logp + 0.3, torch.randn(tokens, device="cuda", generator=gen)
    w = torch.rand(tokens, device="cuda", generator=gen) / tokens
    scale = torch.tensor([64.0], device="cuda")
    loss, d_logits = layer.policy_loss_gradient(logits, targets, old, A, ref_logp=ref, weights=w, kl_weight=0.2, d_loss=scale, out=logits)
    assert d_logits is logits
    grads = policy.backward(d_logits, saved)
    norm = layer.gradient_norm(list(grads.values()), max_norm=0.5, grad_scale=1 / scale)

    p = {n: t.cpu().double().requires_grad_() for n, t in policy.params.items()}
    first = torch.tensor([sum(lengths[:i]) for i, n in enumerate(lengths) for _ in range(n)])
    pos = torch.arange(tokens)
    seen = (first[:, None] == first[None]) & (pos[None] <= pos[:, None]) & ((pos[:, None] - pos[None] < 20) | (pos[None] - first[None] < 2))

    def normed(t, name):
        return torch.nn.functional.layer_norm(t, (256,), p[name], p[name + "_bias"])
    r1 = x.cpu().double() + block.cpu().double()
    q, k, v = (normed(r1, "norm1") @ p["qkv"]).view(tokens, 3, 2, 128).permute(1, 2, 0, 3)
    s = (q @ k.transpose(1, 2) / math.sqrt(128)).masked_fill(~seen, -math.inf).softmax(-1)
    r2 = r1 + (s @ v).transpose(0, 1).reshape(tokens, 256) @ p["dense"]
    z = (r2 + torch.nn.functional.gelu(normed(r2, "norm2") @ p["up"]) @ p["down"]) @ p["head"]
    there = targets.cpu() >= 0
    lp = torch.log_softmax(z, -1).gather(1, targets.cpu().clamp(min=0)[:, None])[:, 0]
    ratio, away = (lp - old.cpu().double()).exp(), ref.cpu().double() - lp
    Ad = A.cpu().double()
    each = w.cpu().double() * (-torch.minimum(ratio * Ad, ratio.clamp(0.8, 1.2) * Ad) + 0.2 * (away.exp() - away - 1))
    total = each[there].sum()
    total.backward()
    assert abs(float(loss.loss) - float(total.detach())) < 0.02 * float(each.detach().abs().sum())
    for name, g in grads.items():
        want = p[name].grad
        off = float((g.cpu().double() / 64 - want).norm() / want.norm())
        assert off < 0.02, (name, off)
    exact = math.sqrt(sum(float(p[n].grad.square().sum()) for n in p))
    assert abs(float(norm.norm) - exact) < 0.02 * exact and abs(float(norm.scale) * 64 - min(1.0, 0.5 / exact)) < 0.02
    assert norm.norms.shape == (len(grads),)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_training_over_packed_documents_runs(bits):
    cuda_or_skip()
    losses = profile_layer.train(256, 64, 2, 4, bits, window=16, sinks=1, documents=3, clip=0.01)
    assert len(losses) == 4 and all(math.isfinite(v) for v in losses)
    losses, norms = profile_layer.train_policy(256, 1000, [40, 0, 13, 75], 3, bits, clip=0.1)
    assert len(losses) == len(norms) == 3 and all(math.isfinite(v) for v in losses + norms) and all(v > 0 for v in norms)


@gpu
def test_the_command(capsys):
    cuda_or_skip()
    profile_layer.main(["--workload", "gpt3_1_3b", "--micro-batches", "1", "--tp", "1", "--window", "256", "--sinks", "4", "--reps", "2", "--plans", "512", "--documents", "5",
                        "--loss", "--clip", "1", "--steps", "2", "--policy-steps", "2"])
    r = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    times = next(iter(r["forward_backward_us"].values()))
    assert set(times) == set(opgraph.GPT_TYPES) and all(f > 0 and b > 0 for n, (f, b) in times.items() if n not in profile_layer.CONTAINED)
    assert r["documents"] == 5 and len(r["policy"]["losses"]) == 2 and all(math.isfinite(v) for v in r["policy"]["losses"] + r["policy"]["gradient_norms"])
