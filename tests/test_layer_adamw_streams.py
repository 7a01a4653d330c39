"""An AdamW that goes away while another stream is at work on its step."""
import pytest
import torch

from superscaler_amd import layer
from tests.test_layer_packing_memory import busy

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_memory_stays_until_the_step_is_done(bits):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    gen = torch.Generator(device="cuda").manual_seed(1)
    start, grad = (torch.randn(3000, device="cuda", generator=gen) for _ in range(2))
    want = start.clone()
    layer.AdamW([want], state_bits=bits).step([grad], lr=0.1)
    got, side = start.clone(), torch.cuda.Stream()
    opt = layer.AdamW([got], state_bits=bits)
    places = {t.data_ptr() for t in (opt._tensors, opt._chunk_tensor, *opt.state.values())}
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        busy()
        opt.step([grad], lr=0.1)
        done = side.record_event()
    del opt
    others = [torch.full((n,), 1 << 20, dtype=torch.int32, device="cuda") for n in (10, 100, 770, 768, 3100) for _ in range(40)]
    assert not done.query() and not places & {t.data_ptr() for t in others}
    torch.cuda.synchronize()
    assert torch.equal(got, want)
