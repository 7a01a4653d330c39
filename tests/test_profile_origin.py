"""What a measured profile database says of itself: times of the card and not of the host."""
import time

import pytest
import torch

from superscaler_amd import profile_layer

gpu = pytest.mark.gpu


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
