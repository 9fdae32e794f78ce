"""A cache that is refused by its arguments is refused before any device call."""
import pytest

from test_gpu_paged import side_stream
from test_gpu_paged_calls import captured

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_a_refused_cache_leaves_a_capture_alone():
    import qw_amd

    x = torch.zeros(8, device="cuda")

    def refused():
        for args in (("fp16", 2, 64), ("fp16", 0, 128), ("turbo4", 2, 96)):
            with pytest.raises(qw_amd.QwError):
                qw_amd.KVCache(*args)
        x.add_(1)

    _, g = captured(refused, side_stream(6))
    g.replay()
    torch.cuda.synchronize()
    assert torch.all(x == 1)
