"""Rows of 16-bit elements that begin at an odd element: the kernels' 16-byte loads at addresses that are no multiples of four."""
import pytest
import torch

from superscaler_amd import layer

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def shifted(seed, *shape, dtype, by, at=0.0):
    """A contiguous tensor `by` elements into its memory, with others' elements on both sides, and a copy of it in memory of its own."""
    n = torch.Size(shape).numel()
    flat = torch.randn(n + 32, generator=torch.Generator().manual_seed(seed)).add_(at).to(dtype).cuda()
    t = flat[16 + by:16 + by + n].view(shape)
    assert t.is_contiguous() and t.data_ptr() % 16 == by * t.element_size() % 16
    return t, t.clone()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,by", [(BF16, 1), (F16, 3), (BF16, 7), (F16, 2), (F32, 3)])
@pytest.mark.parametrize("width", [8, 264, 2048, 7168, 12288, 20000, 513])
def test_norm_rows_that_begin_anywhere(dtype, by, width):
    """Whole vectors and not, with the parameters in LDS and in memory: the same bits as of aligned copies."""
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    rows = 5
    big = [shifted(i, rows, width, dtype=dtype, by=by) for i in range(4)]
    small = [shifted(10 + i, width, dtype=dtype, by=by, at=1.0) for i in range(5)]

    def calls(which):
        x, block, dr, dy = (t[which] for t in big)
        how = dict(zip(("gate", "exit_weight", "exit_bias", "entry_weight", "entry_bias"), (t[which] for t in small)))
        r = layer.block_norm(x, block, **how)
        return [*r, *layer.block_norm_backward(dr, dy, x, block, r.stats, **how)]
    for a, b in zip(calls(0), calls(1)):
        assert torch.equal(a, b)
