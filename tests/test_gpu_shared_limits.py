"""Sizes and values at the ends of what the shared, scored and evicting calls take."""
import ctypes

import numpy as np
import pytest

from conftest import rng
from test_gpu_shared import dev, filled, queries

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

INT_MAX = 2 ** 31 - 1


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("n_seq,n_rows,group", [(INT_MAX, INT_MAX, 1), (INT_MAX, INT_MAX, 4), (INT_MAX, INT_MAX, 6), (INT_MAX, INT_MAX, 8),
                                                (2 ** 30, 2 ** 30, 8), (2 ** 24, 1, 1), (1, 2 ** 24 - 1, 2), (INT_MAX, 1, INT_MAX)])
def test_row_counts_whose_product_wraps(n_seq, n_rows, group):
    """Refused on the host, by the declared sizes alone: (2^31 - 1)^2 * 4 is -2^34 + 4 in 64 bits."""
    import qw_amd

    prefix = filled("fp16", 1, 128, 20, rng(3))
    x = torch.zeros(128, dtype=torch.float16, device="cuda")
    call = qw_amd.lib().qw_kv_shared_attention
    assert call(prefix._h, None, n_seq, None, x.data_ptr(), group, n_rows, 0.1, x.data_ptr(), stream()) in (1, 2)
    torch.cuda.synchronize()
    assert prefix.offset == 20 and not x.any()
