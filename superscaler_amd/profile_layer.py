"""A profile database taken on this GPU, and plans scored with it.

    python -m superscaler_amd.profile_layer --workload gpt3_13b --window 512 --sinks 4 --plans 65536

Times the operators of a GPT layer's training step on the card, forward and backward, for every micro-batch size and
tensor-parallel degree of the workload: products by the matrix library, norms with their residual, and attention, by superscaler_amd.layer.
The times go into a database of the form that ProfileDB.from_directory loads; seeded plans are scored with it twice, with the
optimizer's moments in 32 bits and in 8.  `--steps` trains the layer for that many steps with both, as a check that what was
timed works together.  Collectives and bandwidths between GPUs cannot be taken on one card: they are those of the synthetic database.
Where only some sizes and degrees are measured, the others are the synthetic database's, too: the line names them and no best plan.
Prints one JSON line; `--out` writes the database as files, and beside them which of them were measured.

A row's times are those of calls that follow each other on the card without waiting for the host, as in a training step whose host is
ahead.  Its reserved memory is what a call has in use at its peak beyond what it leaves: forward its results, backward the gradients
of weights.

Attention is one operator here: its time stands in the row of the scores, which keeps the answer and a log-sum per query, and the rows of
softmax, dropout and context keep and take nothing.  A block's residual addition is part of the norm behind it, whose row has both.  The
layer has no dropout: a database of one that has needs its times from elsewhere.
"""
import argparse
import csv
import dataclasses
import json
import os
import statistics
import time

import numpy as np
import torch

from . import layer, synth
from .profile_db import FIELDS, CostModelSettings, ProfileDB

HEAD = 128
MB = 1.0 / (1 << 20)
#: rows that another row's operator contains
CONTAINED = ("enc-attention-softmax", "enc-attention-dropout", "enc-attention-context", "enc-post-attention-dropout", "enc-post-MLP-dropout")


class GptLayer:
    """One layer's shard of a tensor-parallel group of `tp`, in bfloat16: (residual stream, previous block's output) -> the same
    for the next layer.  A group's sums of partial products are left out: what is here is one GPU's part."""

    def __init__(self, hidden, tp=1, window=None, sinks=0, device="cuda:0", seed=0):
        if hidden % (HEAD * tp):
            raise ValueError(f"{hidden} elements are not {tp} equal parts of heads of {HEAD}")
        gen = torch.Generator(device=device).manual_seed(seed)
        self.heads, self.window, self.sinks = hidden // HEAD // tp, window, sinks

        def weight(*size):
            return torch.randn(*size, device=device, generator=gen).mul_(size[0] ** -0.5).bfloat16()
        part = hidden // tp
        self.params = {"qkv": weight(hidden, 3 * part), "dense": weight(part, hidden), "up": weight(hidden, 4 * part), "down": weight(4 * part, hidden)}
        for name in ("norm1", "norm2"):
            self.params[name] = torch.ones(hidden, dtype=torch.bfloat16, device=device)
            self.params[name + "_bias"] = torch.zeros(hidden, dtype=torch.bfloat16, device=device)

    def _norm(self, name):
        return dict(entry_weight=self.params[name], entry_bias=self.params[name + "_bias"], kind="layer")

    def forward(self, x, block):
        p, s = self.params, {"x": x, "block": block}
        s["r1"], s["y1"], s["st1"] = layer.block_norm(x, block, **self._norm("norm1"))
        qkv = (s["y1"] @ p["qkv"]).unflatten(-1, (3, self.heads, HEAD))
        s["q"], s["k"], s["v"] = qkv.unbind(2)
        s["o"], s["lse"] = layer.window_attention(s["q"], s["k"], s["v"], window=self.window, sinks=self.sinks)
        s["a"] = s["o"].flatten(2) @ p["dense"]
        s["r2"], s["y2"], s["st2"] = layer.block_norm(s["r1"], s["a"], **self._norm("norm2"))
        s["u"] = s["y2"] @ p["up"]
        s["g"] = torch.nn.functional.gelu(s["u"])
        return s["r2"], s["g"] @ p["down"], s

    def backward(self, d_residual, d_block, s):
        """Gradients of (x, block) and of the parameters, by name."""
        p, grads = self.params, {}

        def product(name, a, d):
            grads[name] = a.flatten(0, -2).t() @ d.flatten(0, -2)
            return d @ p[name].t()

        def norm(name, d_r, d_y, x, block, stats):
            g = layer.block_norm_backward(d_r, d_y, x, block, stats, **self._norm(name))
            grads[name], grads[name + "_bias"] = g.entry_weight, g.entry_bias
            return g.x, g.block
        d = torch.ops.aten.gelu_backward(product("down", s["g"], d_block), s["u"])
        d_r1, d_a = norm("norm2", d_residual, product("up", s["y2"], d), s["r1"], s["a"], s["st2"])
        d_o = product("dense", s["o"].flatten(2), d_a).view_as(s["o"])
        dqkv = layer.window_attention_backward(d_o, s["q"], s["k"], s["v"], s["o"], s["lse"], window=self.window, sinks=self.sinks)
        d_x, d_in = norm("norm1", d_r1, product("qkv", s["y1"], torch.stack(dqkv, 2).flatten(2)), s["x"], s["block"], s["st1"])
        return d_x, d_in, grads


def train(hidden, seq, batch, steps, state_bits, window=None, sinks=0, device="cuda:0"):
    """A layer trained to make its output rows what another layer's are: the losses, step by step."""
    net, goal = (GptLayer(hidden, 1, window, sinks, device, seed) for seed in (1, 2))
    names = list(net.params)
    main = [net.params[n].float() for n in names]
    opt = layer.AdamW(main, copies=[net.params[n] for n in names], state_bits=state_bits)
    gen = torch.Generator(device=device).manual_seed(3)
    x, block = (torch.randn(batch, seq, hidden, device=device, generator=gen).bfloat16() for _ in range(2))
    want = sum(goal.forward(x, block)[:2]).float()
    losses = []
    for t in range(1, steps + 1):
        r, b, saved = net.forward(x, block)
        off = r.float() + b.float() - want
        losses.append(off.square().mean())
        d = (off * (2 / off.numel())).bfloat16()
        grads = net.backward(d, d, saved)[2]
        opt.step([grads[n] for n in names], lr=1e-3, betas=(0.9, 0.95), step=t)
    return [float(v) for v in losses]


def _time_us(call, reps, device="cuda:0"):
    """Microseconds of `call` on the card, one of `reps` in a row that are queued while it is still at work on something else."""
    filler = torch.empty(1 << 29, dtype=torch.uint8, device=device)     # some 80 us to fill
    for _ in range(2):
        call()
    torch.cuda.synchronize(device)
    begin = time.perf_counter()
    for _ in range(reps):
        call()
    fills = 4 + int(2 * (time.perf_counter() - begin) / 75e-6)
    times = []
    for _ in range(8):
        torch.cuda.synchronize(device)
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        for _ in range(fills):
            filler.zero_()
        a.record()
        for _ in range(reps):
            call()
        b.record()
        ahead = not a.query()
        b.synchronize()
        if ahead:
            times.append(a.elapsed_time(b) * 1e3 / reps)
        else:
            fills *= 2      # the card caught up with the host
        if len(times) == 3:
            break
    if not times:
        raise RuntimeError("the host does not get ahead of the card")
    return statistics.median(times)


def _reserved_mb(call, device="cuda:0", left=None):
    """MB that `call` has in use at its peak beyond its results, or beyond `left` MB of them."""
    torch.cuda.synchronize(device)
    before = torch.cuda.memory_allocated(device)
    torch.cuda.reset_peak_memory_stats(device)
    results = call()
    peak, after = torch.cuda.max_memory_allocated(device), torch.cuda.memory_allocated(device)
    del results
    return max(0.0, (peak - after) * MB if left is None else (peak - before) * MB - left)


def measure(w, micro_batch, tp, window=None, sinks=0, vocab=51200, reps=10, device="cuda:0"):
    """{operator name: (forward us, backward us, reserved forward MB, backward MB)} of a layer's shard of workload `w`, for the rows of
    opgraph.GPT_TYPES."""
    net, h, s = GptLayer(w.hidden, tp, window, sinks, device), w.hidden, w.seq
    x = torch.randn(micro_batch, s, h, device=device).bfloat16()
    block, d = torch.randn_like(x), torch.randn_like(x)
    r2, m, saved = net.forward(x, block)
    out = {name: (0.0,) * 4 for name in CONTAINED}

    def both(name, forward, backward):
        out[name] = (_time_us(forward, reps, device), _time_us(backward, reps, device), _reserved_mb(forward, device),
                     _reserved_mb(backward, device, sizes(w, name, micro_batch, tp)[2]))

    def product(name, a, weight):
        a = a.flatten(0, -2)
        g = torch.randn(a.shape[0], weight.shape[1], device=device).bfloat16()
        both(name, lambda: a @ weight, lambda: (g @ weight.t(), a.t() @ g))
    p = net.params
    for name, key, a, b, stats in (("enc-1st-layernorm", "norm1", x, block, "st1"), ("enc-2nd-layernorm", "norm2", saved["r1"], saved["a"], "st2"),
                                   ("final-layernorm", "norm1", x, block, "st1")):
        both(name, lambda: layer.block_norm(a, b, **net._norm(key)), lambda: layer.block_norm_backward(d, d, a, b, saved[stats], **net._norm(key)))
    product("enc-attention-qkv", saved["y1"], p["qkv"])
    how = dict(window=window, sinks=sinks)
    q, k, v, o, lse = (saved[n] for n in ("q", "k", "v", "o", "lse"))
    both("enc-attention-score", lambda: layer.window_attention(q, k, v, **how), lambda: layer.window_attention_backward(o, q, k, v, o, lse, **how))
    product("enc-attention-dense", saved["o"].flatten(2), p["dense"])
    product("enc-MLP-GEMM-1", saved["y2"], p["up"])
    both("enc-MLP-gelu", lambda: torch.nn.functional.gelu(saved["u"]), lambda: torch.ops.aten.gelu_backward(saved["g"], saved["u"]))
    product("enc-MLP-GEMM-2", saved["g"], p["down"])
    table = torch.randn(vocab // tp, h, device=device).bfloat16()
    tokens = torch.randint(0, table.shape[0], (micro_batch * s,), device=device)
    rows = d.view(-1, h)
    both("encoder-embedding", lambda: table[tokens], lambda: torch.zeros_like(table).index_add_(0, tokens, rows))
    product("gpt-post-process", x, table.t())
    return out


def sizes(w, name, micro_batch, tp):
    """(input, output, weights, activations) MB of a row: those of synth, with attention as one operator that keeps its answer and a
    log-sum for every query, and norms that take the residual stream and a block's output, and keep the stream, its norm and four
    statistics of every row."""
    u = micro_batch * w.seq * w.hidden * 2 * MB
    if "layernorm" in name:
        return 2 * u, 2 * u, 2 * w.hidden * 2 * MB, 2 * u + micro_batch * w.seq * 16 * MB
    if name == "enc-attention-score":
        lse = micro_batch * (w.hidden // HEAD / tp) * w.seq * 4 * MB
        return 4 * u / tp + u, u / tp + u, 0.0, u / tp + lse
    if name in CONTAINED[:3]:
        return u / tp + u, u / tp + u, 0.0, 0.0
    if name in CONTAINED:
        return 2 * u, 2 * u, 0.0, 0.0
    return synth._shape_mb(w, name, micro_batch, tp)


def database(w, graph, measured, base):
    """The database `base` of workload `w` with the rows of `measured` ({(micro-batch, tp): measure's result}) in their places; of
    rows that are two times only, the reserved memory stays that of `base`."""
    db = ProfileDB.empty(w.model_name, base.op_names, base.mbs_list, base.tp_list, base.n_algo)
    db.collectives, db.intra_band, db.inter_band = base.collectives, base.intra_band, base.inter_band
    for f in FIELDS:
        db.tables[f][...] = base.tables[f]
    for (b, tp), rows in measured.items():
        at = db.mbs_list.index(b), db.tp_list.index(tp)
        for name, row in rows.items():
            values = dict(zip(FIELDS[2:6], sizes(w, name, b, tp)), **dict(zip(FIELDS[:2] + FIELDS[6:], row)))
            for f, v in values.items():
                db.tables[f][(db.op_names.index(name),) + at] = round(v, 3)
    return db


def write(db, stem, directory, measured=None):
    """The database's operator tables as files that ProfileDB.from_directory reads (profiler/op_profiler.py:461-482).  `measured`: the
    (micro-batch, tp) that were, to be listed with the others in a file of their own, <stem>_origin.csv."""
    os.makedirs(directory, exist_ok=True)
    if measured is not None:
        with open(os.path.join(directory, f"{stem}_origin.csv"), "w", newline="") as f:
            csv.writer(f).writerows([["mbs", "tp", "origin"]] + [[b, tp, "measured" if (b, tp) in measured else "synthetic"] for b in db.mbs_list for tp in db.tp_list])
    for mi, mbs in enumerate(db.mbs_list):
        for ti, tp in enumerate(db.tp_list):
            for algo in range(db.n_algo):
                with open(os.path.join(directory, f"{stem}_mbs{mbs}_tp{tp}_algo{algo}.csv"), "w", newline="") as f:
                    out = csv.writer(f)
                    out.writerow(["op_name", "forward-compute", "backward-compute", "input_size", "output_size", "weights", "activations", "fwd_reserved", "bwd_reserved"])
                    for t, name in enumerate(db.op_names):
                        out.writerow([name] + ["%.3f" % db.tables[c][t, mi, ti, algo] for c in FIELDS])


@dataclasses.dataclass
class EightBitSettings(CostModelSettings):
    """Settings of a training run whose optimizer keeps its two moments in 8 bits: 2 bytes and a little per weight of 2 bytes, where
    the reference's settings have 8."""
    @property
    def memory_optimizer(self):
        return 1


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--workload", default="gpt3_13b", choices=[n for n, w in synth.WORKLOADS.items() if w.model_name == "gpt"])
    ap.add_argument("--micro-batches", type=int, nargs="+", default=None, help="sizes to measure (default: the workload's)")
    ap.add_argument("--tp", type=int, nargs="+", default=None, help="tensor-parallel degrees to measure (default: all)")
    ap.add_argument("--window", type=int, default=None)
    ap.add_argument("--sinks", type=int, default=0)
    ap.add_argument("--reps", type=int, default=10)
    ap.add_argument("--plans", type=int, default=65536)
    ap.add_argument("--steps", type=int, default=0, help="train one layer for this many steps, moments in 32 and in 8 bits")
    ap.add_argument("--out", default=None, help="directory for the database's files")
    args = ap.parse_args(argv)

    from .aceso_cost_model import CostModel
    w = synth.WORKLOADS[args.workload]
    graph = synth.make_graph(w)
    base = synth.make_db(w, graph)
    heads = w.hidden // HEAD
    for what, asked, there in (("--micro-batches", args.micro_batches, base.mbs_list), ("--tp", args.tp, [t for t in base.tp_list if heads % t == 0])):
        if any(v not in there for v in asked or ()):
            ap.error(f"{what}: of workload {w.name} there are {there}")
    measured = {(b, tp): measure(w, b, tp, args.window, args.sinks, reps=args.reps)
                for b in (args.micro_batches or base.mbs_list) for tp in (args.tp or base.tp_list) if heads % tp == 0}
    db = database(w, graph, measured, base)
    result = {"workload": w.name, "ops": graph.num_ops, "window": args.window, "sinks": args.sinks, "measured": len(measured)}
    (b, tp), rows = next(iter(measured.items()))
    result["forward_backward_us"] = {f"micro-batch {b}, tp {tp}": {n: [round(t, 1) for t in row[:2]] for n, row in rows.items()}}
    result["synthetic"] = [[b, tp] for b in base.mbs_list for tp in base.tp_list if (b, tp) not in measured]
    if args.out:
        write(db, f"{w.model_name}_{w.name}", args.out, measured)
    for bits, kind in ((32, CostModelSettings), (8, EightBitSettings)):
        cm = CostModel(kind(**dataclasses.asdict(synth.make_settings(w))), db, graph)
        ms, mb, feasible = cm.score_batch(synth.make_plans(w, cm.tables, n_plans=args.plans))
        best = np.where((feasible > 0) & (not result["synthetic"]), ms, np.inf)
        result[f"plans_with_{bits}_bit_moments"] = {"scored": len(ms), "feasible": int((feasible > 0).sum()),
                                                    "best_ms": float(best.min()) if np.isfinite(best.min()) else None, "median_peak_mb": float(np.nanmedian(mb))}
        cm.close()
        if args.steps:
            losses = train(min(w.hidden, 2048), 512, 2, args.steps, bits, args.window, args.sinks)
            result[f"losses_with_{bits}_bit_moments"] = [losses[0], losses[-1]]
    print(json.dumps(result))


if __name__ == "__main__":
    main()
