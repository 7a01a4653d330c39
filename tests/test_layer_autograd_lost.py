"""Where automatic differentiation would lose a gradient of the packed step's operators, it is told, and what to call instead."""
import pytest
import torch

from superscaler_amd import layer
from superscaler_amd.evaluator import AceError

gpu = pytest.mark.gpu


def cuda_or_skip():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


@pytest.mark.parametrize("name", ["block_norm", "window_attention", "packed_attention", "token_logprobs", "policy_loss", "gradient_norm"])
def test_the_message_names_calls_that_are_there(name):
    a = torch.ones(3, requires_grad=True)
    made, = layer._untracked(name, (torch.ones(2),), (a,))
    with pytest.raises(AceError) as e:
        made.sum().backward()
    words = [w.strip("():") for w in str(e.value).split() if "_" in w and "." not in w]
    assert name in words and all(hasattr(layer, w) for w in words)
