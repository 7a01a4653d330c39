"""The operators of a training step over packed sequences, as cases that can be timed.

A case is a dict of plain values.  `op` says which operator it is:

  packed  layer.packed_attention, and layer.packed_attention_backward where `back`: causal attention over sequences of different
          lengths that lie one after the other
  loss    layer.token_logprobs (`what` "logprobs"), with layer.token_logprobs_backward ("logprobs_train"), layer.policy_loss
          ("policy") or layer.policy_loss_gradient ("policy_train"): log-probabilities of the tokens that were taken, the clipped
          policy loss with its KL term, and the gradients of logits
  norm    layer.gradient_norm, or layer.clip_gradients where `clip`: the norm of each of a stage's gradients and of all,
          and the factor that clips them

Where `own` is false the same is computed from elementary torch operations in 32 bits (sums over a row's vocabulary, and what follows from
them for the row, in 64: a ratio next to the border of its clipping has to fall on the right side).
"""
import math
import random

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
CLIP, KL_WEIGHT = (0.2, 0.28), 0.05
#: rows of logits that are taken at a time where inputs and their 64-bit results are made
ROWS = 1024


def listed():
    return [
        # four short prompts answered at once: latency
        _packed("packed_prompts_509_h8", 509, 4, 8, 2, 128, layout=1),
        # forward of the 40-layer GPT graph: eight rows of 2,048 tokens filled with documents
        _packed("packed_gpt_16384_h40", 16384, 24, 40, 40, 128, layout=2),
        # a few long documents with shared key heads
        _packed("packed_long_32768_h8", 32768, 3, 8, 2, 128, layout=3),
        # training the 24-layer GPT graph on four rows of documents
        _packed("packed_train_8192_h16", 8192, 12, 16, 16, 128, layout=4, back=True),
        # training on many short texts in half precision, small heads, a window with first keys, the last tokens unused
        _packed("packed_train_short_6143_h16", 6143, 40, 16, 4, 64, window=256, sinks=4, dtype="fp16", tail=130, layout=5, back=True),
        # the tokens that eight sequences have just taken: latency
        _loss("logprobs_8x51200", 8, 51200),
        # cross entropy of three short texts over a vocabulary of odd size, full precision
        _loss("logprobs_train_1531x32001", 1531, 32001, "logprobs_train", "fp32"),
        # a policy's loss alone, half precision, on a shard's vocabulary whose rows are padded
        _loss("policy_4096x25600", 4096, 25600, "policy", "fp16", pad=64),
        # the policy's training step on four rows of 2,048 tokens
        _loss("policy_train_8192x51200", 8192, 51200, "policy_train"),
        # one T5 layer's encoder half in full precision: latency
        _norm("norm_t5_1_layer", 1024, 1, grad="fp32"),
        # all layers of the 24-layer GPT graph
        _norm("norm_gpt_24x2048", 2048, 24),
        # a pipeline stage of two layers of the 40-layer GPT graph, scaled gradients brought back and clipped in place
        _norm("clip_gpt_2x5120", 5120, 2, clip=True),
    ]


def _named(name, c):
    return dict(c, name=name) if name else c


def _packed(name, tokens, sequences, heads, kv_heads, dim, window=0, sinks=0, dtype="bf16", tail=0, layout=0, back=False):
    """`sequences` of lengths that follow from `layout`, over all of `tokens` but the last `tail`; `window` 0: all earlier tokens."""
    return _named(name, dict(op="packed", tokens=tokens, sequences=sequences, heads=heads, kv_heads=kv_heads, dim=dim, window=window, sinks=sinks, dtype=dtype, tail=tail,
                             layout=layout, back=back))


def _loss(name, rows, vocab, what="logprobs", dtype="bf16", pad=0, ignored=0.2):
    """`rows` tokens over a vocabulary of `vocab`, whose rows lie `vocab` + `pad` elements apart; a part of them, `ignored`, has no
    target (tokens of the prompt)."""
    return _named(name, dict(op="loss", rows=rows, vocab=vocab, what=what, dtype=dtype, pad=pad, ignored=ignored))


def _norm(name, hidden, layers, vocab=0, grad="bf16", clip=False, most=2.0):
    """Gradients of `layers` layers (and an embedding of `vocab` rows), of type `grad` or "mixed": matrices bf16, vectors fp32.
    `most`: the largest norm, as a multiple of the gradients'."""
    return _named(name, dict(op="norm", hidden=hidden, layers=layers, vocab=vocab, grad=grad, clip=clip, most=most))


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _largest(op):
    each = [work(c) for c in listed() if c["op"] == op]
    return max(w["bytes"] for w in each), max(w["flops"] for w in each)


def draw(rng):
    op = rng.choice(["packed", "packed", "loss", "loss", "norm"])
    most_bytes, most_flops = _largest(op)
    while True:
        c = {"packed": _draw_packed, "loss": _draw_loss, "norm": _draw_norm}[op](rng)
        w = work(c)
        if w["bytes"] <= most_bytes and w["flops"] <= most_flops:
            return c


def _draw_packed(rng):
    kv_heads, dim, dtype = rng.choice([1, 2, 4, 8, 16, 20]), rng.choice([64, 80, 128, 128]), rng.choice(["bf16", "fp16"])
    heads = kv_heads * rng.choice([1, 1, 2, 4, 8] if kv_heads <= 4 else [1, 2])
    tokens = _log_int(rng, 16, 32768)
    tail = rng.choice([0, 0, rng.randint(0, tokens // 4)])
    sequences = _log_int(rng, 1, max(2, min(256, tokens // 8)))
    window = rng.choice([0, 0, _log_int(rng, 16, max(17, tokens))])
    return _packed(None, tokens, sequences, heads, kv_heads, dim, window, rng.choice([0, 1, 4, 37]) if window else 0, dtype, tail, rng.randrange(1 << 30), rng.random() < 0.5)


def _draw_loss(rng):
    vocab = rng.choice([51200, 25600, 12800, _log_int(rng, 500, 150000), 2 * _log_int(rng, 250, 60000) + 1])
    return _loss(None, _log_int(rng, 1, 8192), vocab, rng.choice(["logprobs", "logprobs_train", "policy", "policy_train", "policy_train"]), rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                 rng.choice([0, 0, 64 - vocab % 64, 3]), rng.choice([0.0, 0.2, 0.6]))


def _draw_norm(rng):
    hidden = rng.choice([1024, 2048, 4096, 20 * rng.randint(5, 255) + 4, 2 * rng.randint(50, 2500) + 1])
    return _norm(None, hidden, _log_int(rng, 1, 24), rng.choice([0, rng.randint(1000, 51200)]), rng.choice(["bf16", "bf16", "fp16", "fp32", "mixed"]), rng.random() < 0.4,
                 rng.choice([2.0, 2.0, 0.5]))


# ---- what a user's program has before the call -----------------------------------------------------------------------------
def prepare(case, seed):
    s = {"packed": _packed_inputs, "loss": _loss_inputs, "norm": _norm_inputs}[case["op"]](case, torch.Generator(device=DEVICE).manual_seed(seed))
    if own and case["op"] == "packed":
        from superscaler_amd import layer
        s["packing"] = layer.Packing(s["lengths"], tokens=case["tokens"], device=DEVICE)     # one for all layers of a step
    return s


def _lengths(c):
    """Cuts at random places: a few long sequences and many short ones, some perhaps empty."""
    rng, used = random.Random(c["layout"]), c["tokens"] - c["tail"]
    cuts = [0] + sorted(rng.randint(0, used) for _ in range(c["sequences"] - 1)) + [used]
    return [b - a for a, b in zip(cuts, cuts[1:])]


def _packed_inputs(c, gen):
    T, H, Hk, D = (c[k] for k in ("tokens", "heads", "kv_heads", "dim"))
    # as the product with the weights of queries, keys and values leaves them
    qkv = torch.randn(T, H + 2 * Hk, D, device=DEVICE, generator=gen).to(TYPES[c["dtype"]])
    s = {"case": c, "lengths": _lengths(c), "q": qkv[:, :H], "k": qkv[:, H:H + Hk], "v": qkv[:, H + Hk:], "d_out": None}
    if c["back"]:
        s["d_out"] = torch.randn(T, H, D, device=DEVICE, generator=gen).to(TYPES[c["dtype"]])
    return s


def _loss_inputs(c, gen):
    N, V = c["rows"], c["vocab"]

    def normal(at=0.0, by=1.0):
        return at + by * torch.randn(N, device=DEVICE, generator=gen)
    logits = torch.empty(N, V + c["pad"], dtype=TYPES[c["dtype"]], device=DEVICE)[:, :V]
    targets = torch.randint(0, V, (N,), device=DEVICE, generator=gen)
    # a token that was taken stands out among the others, by more or less
    ahead = 4 + 8 * torch.rand(N, device=DEVICE, generator=gen)
    logp = torch.empty(N, device=DEVICE, dtype=torch.float64)
    for a in range(0, N, ROWS):
        rows = slice(a, min(N, a + ROWS))
        z = 2 * torch.randn(rows.stop - a, V, device=DEVICE, generator=gen)
        z.scatter_add_(1, targets[rows, None], ahead[rows, None])
        logits[rows] = z
        logp[rows] = _wide_logp(logits[rows], targets[rows])[0]
    s = {"case": c, "logits": logits, "targets": targets, "advantages": normal()}
    # the policy that took them, a few steps ago, and the one that it should stay near to
    s["old_logp"], s["ref_logp"] = (logp + normal(by=0.15)).float(), (logp + normal(by=0.3)).float()
    some = torch.rand(N, device=DEVICE, generator=gen) >= c["ignored"]
    s["targets"] = torch.where(some, targets, -100)
    s["weights"] = some.float() / some.sum().clamp(min=1)
    s["d_logp"] = -s["weights"]     # cross entropy, averaged
    return s


def _norm_inputs(c, gen):
    s = {"case": c, "grads": []}
    for n in _sizes(c):
        kind = c["grad"] if c["grad"] != "mixed" else "bf16" if n > 8 * c["hidden"] else "fp32"
        by = 10.0 ** (-4 + len(s["grads"]) % 7 / 3)     # tensors differ
        s["grads"].append((by * torch.randn(n, device=DEVICE, generator=gen)).to(TYPES[kind]))
    # of a loss that was scaled so that the gradients' type holds them
    s["grad_scale"] = 0.95 + 0.04 * torch.rand(1, device=DEVICE, generator=gen)
    squares = torch.stack([g.float().square().sum(dtype=torch.float64) for g in s["grads"]])
    s["max_norm"] = c["most"] * float(squares.sum().sqrt())
    return s


def _sizes(c):
    """Numbers of elements of the stage's tensors, layer by layer: weights and biases of queries, keys, values, the product behind
    them and the two of the MLP, and those of two norms."""
    h = c["hidden"]
    return ([c["vocab"] * h] if c["vocab"] else []) + ([h * h, h] * 4 + [4 * h * h, 4 * h, 4 * h * h, h] + [h] * 4) * c["layers"]


# ---- one pass ---------------------------------------------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if not own:
        return {"packed": _plain_packed, "loss": _plain_loss, "norm": _plain_norm}[c["op"]](s)
    from superscaler_amd import layer
    if c["op"] == "packed":
        how = dict(window=c["window"] or None, sinks=c["sinks"])
        out, lse = layer.packed_attention(s["q"], s["k"], s["v"], s["packing"], **how)
        if not c["back"]:
            return {"out": out, "lse": lse}
        dq, dk, dv = layer.packed_attention_backward(s["d_out"], s["q"], s["k"], s["v"], out, lse, s["packing"], **how)
        return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    if c["op"] == "loss":
        z, t = s["logits"], s["targets"]
        if c["what"].startswith("logprobs"):
            r = layer.token_logprobs(z, t)
            if c["what"] == "logprobs":
                return {"logp": r.logp}
            return {"logp": r.logp, "d_logits": layer.token_logprobs_backward(s["d_logp"], z, t, r.stats)}
        how = dict(ref_logp=s["ref_logp"], weights=s["weights"], clip=CLIP, kl_weight=KL_WEIGHT)
        if c["what"] == "policy":
            r = layer.policy_loss(z, t, s["old_logp"], s["advantages"], **how)
            return {"loss": r.loss, "logp": r.logp, "d_logp": r.d_logp}
        r, d_logits = layer.policy_loss_gradient(z, t, s["old_logp"], s["advantages"], **how)
        return {"loss": r.loss, "logp": r.logp, "d_logp": r.d_logp, "d_logits": d_logits}
    if c["clip"]:
        r = layer.clip_gradients(s["grads"], s["max_norm"], grad_scale=s["grad_scale"])
        return {"norm": r.norm, "scale": r.scale, "norms": r.norms, "grads": s["grads"]}
    r = layer.gradient_norm(s["grads"], max_norm=s["max_norm"], grad_scale=s["grad_scale"])
    return {"norm": r.norm, "scale": r.scale, "norms": r.norms}


def _seen(n, c):
    """Which keys each query of a sequence of n tokens sees: bool [n, n]."""
    i = torch.arange(n, device=DEVICE)
    far = i[:, None] - i[None, :]
    seen = far >= 0
    if c["window"]:
        seen &= (far < c["window"]) | (i[None, :] < c["sinks"])
    return seen


def _plain_packed(s):
    c = s["case"]
    T, H, Hk, D = (c[k] for k in ("tokens", "heads", "kv_heads", "dim"))
    dtype, shared, scale = s["q"].dtype, H // Hk, 1 / math.sqrt(D)

    def zeros(heads):
        return torch.zeros(T, heads, D, dtype=dtype, device=DEVICE)
    out = {"out": zeros(H), "lse": torch.full((H, T), -math.inf, device=DEVICE)}
    if c["back"]:
        out.update(dq=zeros(H), dk=zeros(Hk), dv=zeros(Hk))
    at = 0
    for n in s["lengths"]:
        rows = slice(at, at + n)
        at += n
        if n == 0:
            continue

        def heads(t):       # [n, heads, D] -> [Hk, heads / Hk * n, D]
            return t[rows].float().view(n, Hk, -1, D).permute(1, 2, 0, 3).reshape(Hk, -1, D)

        def tokens(t):      # and back
            return t.view(Hk, -1, n, D).permute(2, 0, 1, 3).reshape(n, -1, D)

        def flip(t):
            return t.transpose(1, 2).contiguous()
        q, k, v = heads(s["q"]), heads(s["k"]), heads(s["v"])
        hidden = ~_seen(n, c)
        scores = torch.bmm(q, flip(k)).mul_(scale).view(Hk, shared, n, n).masked_fill_(hidden, -math.inf).view(Hk, shared * n, n)
        top = scores.amax(-1, keepdim=True)
        p = scores.sub_(top).exp_()
        total = p.sum(-1, keepdim=True)
        out["lse"][:, rows] = (total.log() + top).view(H, n)
        p = p.div_(total)
        o = torch.bmm(p, v)
        out["out"][rows] = tokens(o).to(dtype)
        if c["back"]:
            do = heads(s["d_out"])
            out["dv"][rows] = tokens(torch.bmm(flip(p), do)).to(dtype)
            ds = torch.bmm(do, flip(v)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
            out["dq"][rows] = tokens(torch.bmm(ds, k)).to(dtype)
            out["dk"][rows] = tokens(torch.bmm(flip(ds), q)).to(dtype)
    return out


def _wide_logp(logits, targets):
    """(log-probabilities of the targets in 64 bits, exponentials around each row's largest logit, their sums in 64 bits)"""
    z = logits.float()
    top = z.amax(-1, keepdim=True)
    taken = z.gather(1, targets[:, None]) - top
    e = (z - top).exp_()
    total = e.sum(-1, keepdim=True, dtype=torch.float64)
    return (taken.double() - total.log())[:, 0], e, total


def _policy(s, logp):
    """(loss, its derivative by each logp) in 64 bits."""
    w, A = s["weights"].double(), s["advantages"].double()
    r = (logp - s["old_logp"].double()).exp()
    lo, hi = 1 - CLIP[0], 1 + CLIP[1]
    away = s["ref_logp"].double() - logp
    loss = w * (-torch.minimum(r * A, r.clamp(lo, hi) * A) + KL_WEIGHT * (away.exp() - away - 1))
    free = torch.where(A > 0, r <= hi, r >= lo)
    return loss, w * (torch.where(free, -r * A, torch.zeros_like(r)) + KL_WEIGHT * (1 - away.exp()))


def _plain_loss(s):
    c, z = s["case"], s["logits"]
    there = s["targets"] >= 0
    targets = s["targets"].clamp(min=0)
    logp, e, total = _wide_logp(z, targets)
    none = torch.zeros_like(logp)
    out = {"logp": torch.where(there, logp, none).float()}
    d = s["d_logp"].double()
    if c["what"].startswith("policy"):
        loss, d = _policy(s, logp)
        out["loss"] = torch.where(there, loss, none).sum().float()
    d = torch.where(there, d, none)
    if c["what"].startswith("policy"):
        out["d_logp"] = d.float()
    if c["what"].endswith("train"):
        d = d.float()[:, None]
        p = e.mul_((1 / total).float())
        grad = p.neg_().scatter_add_(1, targets[:, None], torch.ones_like(d)).mul_(d)
        out["d_logits"] = torch.where(there[:, None], grad, torch.zeros_like(grad)).to(z.dtype)
    return out


def _plain_norm(s):
    c = s["case"]
    squares = torch.stack([g.float().square().sum(dtype=torch.float64) for g in s["grads"]])
    norms = squares.sqrt() * s["grad_scale"].double()
    norm = squares.sum().sqrt() * s["grad_scale"].double()
    scale = s["grad_scale"].double() * (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    out = {"norm": norm.float(), "scale": scale.float(), "norms": norms.float()}
    if c["clip"]:
        for g in s["grads"]:
            g.copy_(g.float() * out["scale"])
        out["grads"] = s["grads"]
    return out


# ---- the same in 64 bits ----------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = {"packed": _packed_inputs, "loss": _loss_inputs, "norm": _norm_inputs}[case["op"]](case, torch.Generator(device=DEVICE).manual_seed(seed))
    return {"packed": _exact_packed, "loss": _exact_loss, "norm": _exact_norm}[case["op"]](s)


def _exact_packed(s):
    """Head by head, by automatic differentiation's rules written out."""
    c, H, Hk = s["case"], s["case"]["heads"], s["case"]["kv_heads"]
    f = {n: s[n].double() for n in ("q", "k", "v", "d_out") if s[n] is not None}
    out = {"out": torch.zeros_like(f["q"]), "lse": f["q"].new_full((H, c["tokens"]), -math.inf)}
    if c["back"]:
        out.update(dq=torch.zeros_like(f["q"]), dk=torch.zeros_like(f["k"]), dv=torch.zeros_like(f["v"]))
    begin = 0
    for n in s["lengths"]:
        end = begin + n
        hidden = ~_seen(n, c)
        for h in range(H if n else 0):
            g = h * Hk // H
            q, k, v = f["q"][begin:end, h].contiguous(), f["k"][begin:end, g].contiguous(), f["v"][begin:end, g].contiguous()
            scores = (q @ k.t().contiguous() / c["dim"] ** 0.5).masked_fill_(hidden, -math.inf)
            lse = torch.logsumexp(scores, 1)
            p = torch.exp(scores - lse[:, None])
            out["lse"][h, begin:end] = lse
            out["out"][begin:end, h] = p @ v
            if c["back"]:
                do = f["d_out"][begin:end, h].contiguous()
                dp = do @ v.t().contiguous()
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) / c["dim"] ** 0.5
                out["dv"][begin:end, g] += p.t().contiguous() @ do
                out["dq"][begin:end, h] = ds @ k
                out["dk"][begin:end, g] += ds.t().contiguous() @ q
        begin = end
    return out


def _exact_loss(s):
    c, what = s["case"], s["case"]["what"]
    there = s["targets"] >= 0
    logp = torch.zeros(c["rows"], dtype=torch.float64, device=DEVICE)
    for a in range(0, c["rows"], ROWS):
        z = torch.log_softmax(s["logits"][a:a + ROWS].double(), 1)
        logp[a:a + ROWS] = z[torch.arange(len(z), device=DEVICE), s["targets"][a:a + ROWS].clamp(min=0)]
    logp = torch.where(there, logp, 0.0)
    out = {"logp": logp}
    d = s["d_logp"].double()
    if what.startswith("policy"):
        x = logp.clone().requires_grad_(True)
        ratio = torch.exp(x - s["old_logp"].double())
        A = s["advantages"].double()
        gain = torch.where(A > 0, ratio.clamp(max=1 + CLIP[1]), ratio.clamp(min=1 - CLIP[0])) * A
        away = s["ref_logp"].double() - x
        each = s["weights"].double() * (KL_WEIGHT * (torch.expm1(away) - away) - gain)
        loss = each[there].sum()
        out["loss"], d = loss.detach(), torch.autograd.grad(loss, x)[0]
        out["d_logp"] = d
    if what.endswith("train"):
        grad = torch.empty(c["rows"], c["vocab"], dtype=torch.float64, device=DEVICE)
        for a in range(0, c["rows"], ROWS):
            p = torch.softmax(s["logits"][a:a + ROWS].double(), 1)
            i = torch.arange(len(p), device=DEVICE)
            p[i, s["targets"][a:a + ROWS].clamp(min=0)] -= 1
            grad[a:a + ROWS] = torch.where(there[a:a + ROWS, None], -d[a:a + ROWS, None] * p, 0.0)
        out["d_logits"] = grad
    return out


def _exact_norm(s):
    c, gs = s["case"], s["grad_scale"].double()
    norms = torch.stack([torch.linalg.vector_norm(g.double()) for g in s["grads"]]) * gs
    norm = torch.linalg.vector_norm(norms)[None]
    scale = gs * torch.minimum(s["max_norm"] / (norm + 1e-6), torch.ones_like(norm))
    out = {"norm": norm, "scale": scale, "norms": norms}
    if c["clip"]:
        out["grads"] = [g.double() * scale for g in s["grads"]]
    return out


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------
def work(case):
    return {"packed": _packed_work, "loss": _loss_work, "norm": _norm_work}[case["op"]](case)


def _packed_work(c):
    """Queries, keys and values in, the answer out once, gradients likewise.  Four operations per seen pair and element of a head
    forward, ten backward."""
    pairs = 0
    for n in _lengths(c):
        w = min(n, c["window"] or n)
        near = w * (w + 1) // 2 + (n - w) * w
        m = max(0, min(c["sinks"], n - w))
        pairs += near + m * (n - w) - m * (m - 1) // 2
    moved = 2 * (c["tokens"] - c["tail"]) * (c["heads"] + c["kv_heads"]) * c["dim"] * BYTES[c["dtype"]]
    return {"bytes": moved * (2 if c["back"] else 1) + 4 * c["heads"] * c["tokens"], "flops": c["heads"] * c["dim"] * pairs * (14 if c["back"] else 4)}


def _loss_work(c):
    """Logits in once, their gradient out once; four operations per logit forward, three more for its gradient."""
    n, train = c["rows"] * c["vocab"], c["what"].endswith("train")
    return {"bytes": n * BYTES[c["dtype"]] * (2 if train else 1) + c["rows"] * 24, "flops": n * (7 if train else 4)}


def _norm_work(c):
    """Every gradient in once, clipped ones out once; two operations per element, one more to clip."""
    size = 0
    for n in _sizes(c):
        size += n * BYTES[c["grad"] if c["grad"] != "mixed" else "bf16" if n > 8 * c["hidden"] else "fp32"]
    return {"bytes": size * (2 if c["clip"] else 1) + 8, "flops": sum(_sizes(c)) * (3 if c["clip"] else 2)}
