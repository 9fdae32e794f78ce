"""Calls over pages that need no workspace make none, and take their tensors as they lie."""
import numpy as np
import pytest

from conftest import rng
from test_gpu_paged import Sequences, dev, ints, queries, side_stream

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def captured(f, stream):
    """f's outputs and its graph, from a first call inside a capture."""
    torch.cuda.synchronize()
    stream.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        out = f()
    return out, g


@pytest.mark.parametrize("mode,lengths", [("affine8", [1300, 0, 300]), ("fp16", [40, 1100]), ("int8", [0, 2100] + [5, 260, 0, 17] * 17)])
def test_rows_that_fill_the_card_need_no_workspace(mode, lengths):
    """8192 rows of a KV head: a workgroup for each 32 takes all sequences, and nothing is cut."""
    r = rng(sum(lengths))
    s = Sequences(r, mode, 1, 128, 16, lengths)
    B = len(lengths)
    q, t, n = dev((2 * r.standard_normal((1, 32, 256, 128))).astype(np.float16)).expand(B, -1, -1, -1), ints(s.table), ints(lengths)
    out, g = captured(lambda: s.cache.attention(q, t, n, 0.09), side_stream(4))
    for less in (0, 3):
        now = [max(x - less, 0) for x in lengths]
        n.copy_(ints(now))
        g.replay()
        torch.cuda.synchronize()
        s.check(out[:, 31:], q[:, 31:], 0.09, lengths=now)
        assert torch.equal(out, s.cache.attention(q, t, n, 0.09))
