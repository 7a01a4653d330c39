"""8-bit moments of blocks that have all but decayed."""
import pytest
import torch

from superscaler_amd import layer


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-28, 3e-30, 1e-31, 1e-35, 0.0])
def test_first_moments_below_a_reciprocal_s_range(size):
    """Without a gradient m becomes b1 m, to half a step of the block's unit: of its largest value, or of 1e-30."""
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    p = torch.ones(512, device="cuda")
    opt = layer.AdamW([p], state_bits=8)
    opt.state["m"].copy_(torch.linspace(-127, 127, 512).round())
    opt.state["m_scale"].fill_(size / 127)
    before = opt.moments()[0].double().cpu()
    opt.step([torch.zeros(512, device="cuda")], lr=0.0, betas=(0.5, 0.9))
    off = (opt.moments()[0].double().cpu() - 0.5 * before).view(2, 256).abs()
    unit = (0.5 * before).view(2, 256).abs().amax(1, keepdim=True).clamp(min=1e-30)
    assert float((off - 0.5 * unit / 127 * (1 + 2.0 ** -12) - 127 * 2.0 ** -22 * unit / 127).max()) <= 0
    if size > 1e-29:
        assert (opt.state["m"].view(2, 256).abs().amax(1) == 127).all()
    if size == 0.0:
        assert not opt.state["m_scale"].any()
