"""AdamW writes to the memory that it was made with: a tensor that has been given other memory since is refused, not written where it was."""
import pytest
import torch

from superscaler_amd import layer


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["params", "copies"])
def test_a_tensor_that_has_moved(which):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    params = [torch.ones(n, device="cuda") for n in (300, 0, 1000)]
    copies = [p.bfloat16() for p in params]
    opt = layer.AdamW(params, copies=copies)
    grads = [torch.ones_like(p) for p in params]
    opt.step(grads, lr=0.1)
    held = {"params": params, "copies": copies}[which]
    old = held[2].data      # (kept, so that new memory is other memory)
    held[2].data = old.clone()
    before = [t.clone() for t in params + copies + [old, *opt.state.values()]]
    with pytest.raises(ValueError, match=rf"{which}\[2\] has moved"):
        opt.step(grads, lr=0.1, step=2)
    assert all(torch.equal(a, b) for a, b in zip(before, params + copies + [old, *opt.state.values()]))
    held[2].data = old
    opt.step(grads, lr=0.1, step=2)
    assert float(params[0][0]) < float(before[0][0])
