"""The layer that the training-layer operators are profiled in: its gradients, its training, the database it becomes."""
import csv
import json
import math
import os

import numpy as np
import pytest
import torch

from superscaler_amd import opgraph, profile_layer, synth
from superscaler_amd.profile_db import FIELDS, CostModelSettings, ProfileDB
from superscaler_amd.tables import compile_tables

gpu = pytest.mark.gpu


def rows(scale):
    return {name: (scale * (i + 1.0), scale * (i + 2.5)) for i, name in enumerate(opgraph.GPT_TYPES)}


def test_measured_rows_become_a_database_and_its_files(tmp_path):
    w = synth.WORKLOADS["gpt3_1_3b"]
    graph = synth.make_graph(w)
    base = synth.make_db(w, graph)
    db = profile_layer.database(w, graph, {(2, 1): rows(1.0), (4, 2): rows(3.0)}, base)
    at = db.op_names.index("enc-MLP-GEMM-1")
    assert (db.tables["fwd"][at, 1, 0] == 1.0 * (opgraph.GPT_TYPES.index("enc-MLP-GEMM-1") + 1)).all()
    assert (db.tables["bwd"][at, 2, 1] == 3.0 * (opgraph.GPT_TYPES.index("enc-MLP-GEMM-1") + 2.5)).all()
    for f in FIELDS:      # what was not measured stays
        assert np.array_equal(db.tables[f][:, 0], base.tables[f][:, 0])
    for name in ("enc-attention-softmax", "enc-attention-dropout", "enc-attention-context"):
        assert (db.tables["activations"][db.op_names.index(name), 1, 0] == 0).all()
    assert (db.tables["activations"][db.op_names.index("enc-attention-score"), 1, 0] < base.tables["activations"][db.op_names.index("enc-attention-score"), 1, 0]).all()
    profile_layer.write(db, "gpt_1.3B", str(tmp_path))
    settings = synth.make_settings(w)
    for prim, groups in db.collectives.items():
        for n, table in groups.items():
            with open(tmp_path / f"prim_gpt_1.3B_{prim}_{n}gpus.csv", "w", newline="") as f:
                csv.writer(f).writerows([["size", "time"]] + [[k, v] for k, v in table.items()])
    with open(tmp_path / "p2p_intra_node.csv", "w", newline="") as f:
        csv.writer(f).writerows([list(range(len(db.intra_band))), db.intra_band])
    again = ProfileDB.from_directory("gpt", "1.3B", str(tmp_path) + os.sep, settings)
    assert again.op_names == db.op_names
    for f in FIELDS:
        assert np.array_equal(again.tables[f], db.tables[f])


def test_moments_in_8_bits_take_a_quarter_of_the_optimizer_s_memory():
    w = synth.WORKLOADS["gpt3_1_3b"]
    graph = synth.make_graph(w)
    db = synth.make_db(w, graph)
    import dataclasses
    wide = synth.make_settings(w)
    small = profile_layer.EightBitSettings(**dataclasses.asdict(wide))
    assert isinstance(small, CostModelSettings) and wide.memory_optimizer == 4 * small.memory_optimizer and wide.memory_main_params == small.memory_main_params
    assert compile_tables(graph, db, small).as_struct().optimizer == 1.0 and compile_tables(graph, db, wide).as_struct().optimizer == 4.0


def test_a_layer_is_whole_heads():
    with pytest.raises(ValueError):
        profile_layer.GptLayer(640, tp=4, device="cpu")


@gpu
def test_layer_gradients():
    """Against automatic differentiation of the same layer in 64 bits.  Some twenty tensors between input and gradient are rounded to
    bfloat16 (2^-9 of their norm each at most, taken as independent): 2^-9 sqrt(20) < 1%, doubled for what sums of them cancel."""
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    net = profile_layer.GptLayer(256, window=20, sinks=2, seed=5)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, block, dr, db = (torch.randn(2, 70, 256, device="cuda", generator=gen).bfloat16() for _ in range(4))
    r, b, saved = net.forward(x, block)
    d_x, d_block, grads = net.backward(dr, db, saved)
    p = {n: t.cpu().double().requires_grad_() for n, t in net.params.items()}
    xs, bs = x.cpu().double().requires_grad_(), block.cpu().double().requires_grad_()
    pos = torch.arange(70)
    seen = (pos[None] <= pos[:, None]) & ((pos[:, None] - pos[None] < 20) | (pos[None] < 2))

    def norm(t, name):
        return torch.nn.functional.layer_norm(t, (256,), p[name], p[name + "_bias"])
    r1 = xs + bs
    q, k, v = (norm(r1, "norm1") @ p["qkv"]).view(2, 70, 3, 2, 128).permute(2, 0, 3, 1, 4)
    s = (q @ k.transpose(2, 3) / math.sqrt(128)).masked_fill(~seen, -math.inf).softmax(-1)
    r2 = r1 + (s @ v).transpose(1, 2).reshape(2, 70, 256) @ p["dense"]
    out = torch.nn.functional.gelu(norm(r2, "norm2") @ p["up"]) @ p["down"]
    ((r2 * dr.cpu().double()).sum() + (out * db.cpu().double()).sum()).backward()
    for name, got, want in [("r", r, r2.detach()), ("out", b, out.detach()), ("x", d_x, xs.grad), ("block", d_block, bs.grad)] + [(n, grads[n], p[n].grad) for n in p]:
        off = float((got.cpu().double() - want).norm() / want.norm())
        assert off < 0.02, (name, off)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_layer_learns(bits):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    losses = profile_layer.train(256, 64, 2, 40, bits, window=16, sinks=1)
    assert losses[-1] < 0.5 * losses[0]


@gpu
def test_the_command(capsys, tmp_path):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    profile_layer.main(["--workload", "gpt3_1_3b", "--micro-batches", "1", "--tp", "1", "2", "--window", "256", "--sinks", "4", "--reps", "2", "--plans", "512", "--out",
                        str(tmp_path)])
    r = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    assert r["measured"] == 2 and r["plans_with_8_bit_moments"]["feasible"] >= r["plans_with_32_bit_moments"]["feasible"]
    times = next(iter(r["forward_backward_us"].values()))
    assert set(times) == set(opgraph.GPT_TYPES) and all(f > 0 and b > 0 for n, (f, b) in times.items() if n not in profile_layer.CONTAINED)
    assert len(list(tmp_path.glob("gpt_gpt3_1_3b_mbs*_tp*_algo*.csv"))) == 5 * 3 * 2
