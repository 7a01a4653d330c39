"""What packed attention's gradients need for first keys and queries beyond their window: memory by the tokens that there are, not by the longest sequence,
and sequences of every length about the window."""
import ctypes
import random as pyrandom

import pytest

from superscaler_amd import layer
from tests.test_layer_packed import attend, case, check, cuda_or_skip, pack

gpu = pytest.mark.gpu


def floats(tokens, sequences, longest, kv_heads, window, sinks, dim=128):
    """Of the workspace, without the queries' deltas."""
    lib = layer.load_library()
    lib.ace_packed_attend_backward_workspace_bytes.restype = ctypes.c_size_t
    blocks = tokens // 128 + sequences
    p = pack(tokens, sequences, blocks, longest)
    whole = lib.ace_packed_attend_backward_workspace_bytes(attend(tokens, kv_heads, kv_heads, dim, window, sinks), p)
    none = lib.ace_packed_attend_backward_workspace_bytes(attend(tokens, kv_heads, kv_heads, dim, window, 0), p)
    assert none == 4 * ((kv_heads * tokens + 3) // 4 * 4)
    return (whole - none) // 4


def needed(lengths, window, sinks):
    """Blocks of first keys that queries beyond their window see."""
    return sum(max(0, (min(sinks, n - window) + 31) // 32) for n in lengths if n > window)


@pytest.mark.parametrize("window,sinks,most", [(256, 37, 150e6), (256, 1024, 560e6), (512, 37, 150e6), (2048, 4, 11e6)])
def test_memory_goes_by_the_tokens(window, sinks, most):
    """32,768 tokens in 256 sequences, one of them of 4,096, 20 key heads of 128."""
    assert floats(32768, 256, 4096, 20, window, sinks) * 4 <= most


def test_there_is_memory_for_every_sequence():
    """Never less than the sequences need, and never more than as many blocks as the longest needs for each."""
    rng = pyrandom.Random(1)
    for _ in range(300):
        lengths = [rng.choice([1, rng.randint(1, 90), rng.randint(1, 600)]) for _ in range(rng.randint(1, 400))]
        window, sinks = rng.choice([1, 5, 31, 32, 33, rng.randint(1, 300)]), rng.choice([1, 32, 33, 100, rng.randint(1, 700)])
        kv_heads = 1024      # (one part each)
        if max(lengths) <= window or len(lengths) * kv_heads * ((min(sinks, max(lengths)) + 31) // 32) > 1 << 22:
            continue
        slots, rest = divmod(floats(sum(lengths), len(lengths), max(lengths), kv_heads, window, sinks), kv_heads * 2 * 32 * 128)
        assert rest == 0 and needed(lengths, window, sinks) <= slots <= len(lengths) * ((min(sinks, max(lengths)) + 31) // 32)


@gpu
@pytest.mark.parametrize("window,sinks", [(1, 200), (20, 100), (31, 33), (32, 64), (33, 65), (64, 300), (100, 7)])
@pytest.mark.parametrize("kv_heads", [1, 20])
def test_sequences_about_as_long_as_the_window(window, sinks, kv_heads):
    cuda_or_skip()
    rng = pyrandom.Random(window)
    lengths = [rng.choice([0, window - 1, window, window + 1, window + 31, window + 32, window + 33, rng.randint(1, 160)]) for _ in range(60)]
    check(*case(window, sum(lengths) + 5, kv_heads, kv_heads, 64), lengths, only=set(range(0, 60, 7)) | {57, 58, 59}, window=window, sinks=sinks)


@gpu
def test_one_long_sequence_among_short_ones():
    cuda_or_skip()
    lengths = [10] * 40 + [900] + [40] * 30 + [1, 0, 65]
    check(*case(8, sum(lengths), 4, 2, 128), lengths, only={0, 39, 40, 41, 70, 71, 73}, window=64, sinks=400)
