"""Kernels that need more LDS than a launch has by itself ask for it on every device that they run on, and again after a failure.  On the CPU: the
library's host part over a stand-in for HIP."""
import pytest

from tests import layer_host as host

CALLS = [host.norm_forward(), host.norm_backward(), host.norm_backward(width=8192, dtype=0), host.attend_forward(), host.attend_forward(queries=1, keys=8192), host.attend_backward(window=64, sinks=3),
         host.attend_backward(batch=64, heads=8, kv_heads=8), host.attend_forward(dim=96, dtype=2)]


def test_every_device_is_asked(tmp_path):
    order = [0, 1, 0, 5, 70, 1]
    done = host.run(tmp_path, [host.call(*c, device=d) for d in order for c in CALLS])
    assert all(r["rc"] == 0 and r["launches"] > 0 for r in done)
    assert [r["unprepared"] for r in done] == [0] * len(done)


@pytest.mark.parametrize("at", range(len(CALLS)))
def test_a_failure_is_not_kept(tmp_path, at):
    first, second = host.run(tmp_path, [host.call(*CALLS[at], fail=1), host.call(*CALLS[at])])
    if first["rc"] == 0:      # (a kernel with no more LDS than it has anyway)
        assert first["unprepared"] == 0
    else:
        assert first["rc"] == -3 and first["launches"] == 0
    assert second["rc"] == 0 and second["launches"] > 0 and second["unprepared"] == 0
