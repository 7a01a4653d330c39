"""What a measured profile database says of itself: times of the card and not of the host, reserved memory, what a layer keeps, and which rows were
measured."""
import csv
import json
import time

import numpy as np
import pytest
import torch

from superscaler_amd import opgraph, profile_layer, synth

gpu = pytest.mark.gpu


def database(row):
    w = synth.WORKLOADS["gpt3_1_3b"]
    base = synth.make_db(w, synth.make_graph(w))
    return base, profile_layer.database(w, synth.make_graph(w), {(2, 4): {name: row for name in opgraph.GPT_TYPES}}, base)


def test_reserved_memory_is_what_was_measured():
    base, db = database((1.0, 2.0, 3.5, 4.25))
    assert (db.tables["reserved_fwd"][:, 1, 2] == 3.5).all() and (db.tables["reserved_bwd"][:, 1, 2] == 4.25).all()
    assert (db.tables["fwd"][:, 1, 2] == 1.0).all() and (db.tables["bwd"][:, 1, 2] == 2.0).all()
    base, db = database((1.0, 2.0))      # times only: nothing is known of the rest
    for f in ("reserved_fwd", "reserved_bwd"):
        assert base.tables[f].any() and np.array_equal(db.tables[f], base.tables[f])


def test_files_say_which_of_them_were_measured(tmp_path):
    _, db = database((1.0, 2.0, 0.0, 0.0))
    profile_layer.write(db, "gpt_x", str(tmp_path), {(2, 4): None})
    with open(tmp_path / "gpt_x_origin.csv") as f:
        rows = list(csv.reader(f))
    assert rows[0] == ["mbs", "tp", "origin"] and len(rows) == 1 + len(db.mbs_list) * len(db.tp_list)
    assert [r[:2] for r in rows if r[2] == "measured"] == [["2", "4"]]


@pytest.mark.parametrize("args", [["--tp", "3"], ["--tp", "1", "16"], ["--micro-batches", "5"]])
def test_sizes_that_the_database_does_not_have(args, capsys):
    with pytest.raises(SystemExit) as e:
        profile_layer.main(["--workload", "gpt3_1_3b"] + args)
    assert e.value.code == 2 and "gpt3_1_3b there are [1, 2, 4" in capsys.readouterr().err


@gpu
def test_times_are_the_card_s():
    """A call whose host part takes 300 us and whose kernels take a few."""
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    x = torch.zeros(1 << 16, device="cuda")

    def call():
        end = time.perf_counter() + 3e-4
        while time.perf_counter() < end:
            pass
        x.add_(1.0)
    assert 0.5 < profile_layer._time_us(call, 10) < 100
    big = torch.zeros(1 << 28, device="cuda")      # 1 GiB read and written: 0.27 ms at the card's peak, some 0.41 at a copy's rate
    assert 250 < profile_layer._time_us(lambda: big.add_(1.0), 10) < 1000


@gpu
def test_reserved_memory_is_what_a_call_gives_back():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")

    def mb(n):
        return torch.empty(n << 20, dtype=torch.uint8, device="cuda")

    def call():
        kept, scratch = mb(64), mb(96)
        del scratch
        return kept
    assert profile_layer._reserved_mb(call) == 96.0
    assert profile_layer._reserved_mb(call, left=40.0) == 120.0
    assert profile_layer._reserved_mb(lambda: mb(32)) == 0.0


@gpu
@pytest.mark.parametrize("tp", [1, 4])
def test_rows_keep_what_the_layer_keeps(tp):
    """The activations of a layer's rows add up to what its forward pass leaves for the backward one and the next layer."""
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    w = synth.WORKLOADS["gpt3_1_3b"]
    net = profile_layer.GptLayer(w.hidden, tp, window=256, sinks=4)
    x, block = (torch.randn(3, w.seq, w.hidden, device="cuda").bfloat16() for _ in range(2))
    r, out, saved = net.forward(x, block)
    kept = {t.untyped_storage().data_ptr(): t.untyped_storage().nbytes() for t in [r, out, *saved.values()] if t is not x and t is not block}
    rows = {n: profile_layer.sizes(w, n, 3, tp) for n in opgraph.GPT_TYPES if n.startswith("enc-")}
    assert abs(sum(s[3] for s in rows.values()) - sum(kept.values()) / 2 ** 20) < 1e-6
    assert rows["enc-1st-layernorm"][2] == sum(net.params[n].nbytes for n in ("norm1", "norm1_bias")) / 2 ** 20
    assert all(rows[n][3] == 0 for n in profile_layer.CONTAINED)


@gpu
def test_a_partly_measured_database_has_no_best_plan(capsys, tmp_path):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    profile_layer.main(["--workload", "gpt3_1_3b", "--micro-batches", "2", "--tp", "4", "--reps", "2", "--plans", "256", "--out", str(tmp_path)])
    r = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    assert len(r["synthetic"]) == 14 and [2, 4] not in r["synthetic"]
    assert all(r[f"plans_with_{bits}_bit_moments"]["best_ms"] is None for bits in (8, 32))
    assert sum("measured" in line for line in open(tmp_path / "gpt_gpt3_1_3b_origin.csv")) == 1
