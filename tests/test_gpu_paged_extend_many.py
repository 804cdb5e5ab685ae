"""Block tables of requests that ask for more tokens than a call has rows: starts are the sums of what was asked for, and
positions count from them."""
import numpy as np
import pytest
import torch

import jero_hip as J
import paged_oracle as P
from test_gpu_paged import Pool, step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seqs", [3, 2000])
def test_requests_of_more_than_2_24_tokens(dev, seqs):
    """Granted (blocks of 2^20 positions) and refused; by one launch and by two."""
    hist, asked = [5, 1 << 20, 7], [(1 << 24) + 9, (1 << 25) + 1, 3]
    p = Pool(8, hist + [1] * (seqs - 3), 64, 1 << 20, 60).device(dev)
    want = step(p, dev, np.array(asked + [0] * (seqs - 3), np.int32), tokens=40)
    assert want["starts"][1] == (1 << 24) + 9 and want["starts"][3] == 3 * (1 << 24) + 13
    assert want["granted"][0] == 1 and want["lens"][0] == (1 << 24) + 14


def test_sums_past_31_bits_stop_there(dev):
    """Three requests of 2^31 - 1 tokens, none of which fits: starts stop at 2^31 - 1."""
    p = Pool(9, [1, 1, 1, 1], 4, 16, 8).device(dev)
    most = (1 << 31) - 1
    new = torch.tensor([most, most, most, 2], dtype=torch.int32, device=dev)
    T = 8
    out = [torch.zeros(T, dtype=torch.int32, device=dev), torch.zeros(T, dtype=torch.int64, device=dev),
           torch.zeros(5, dtype=torch.int32, device=dev)]
    granted = torch.zeros(4, dtype=torch.int32, device=dev)
    J.paged_extend(p.pool, new, *out, granted=granted)
    torch.cuda.synchronize()
    assert out[2].tolist() == [0, most, most, most, most] and granted.tolist() == [0, 0, 0, 1]
    assert (out[0] == -1).all() and (out[1] == -1).all()
    assert p.d["lens"].tolist() == [1, 1, 1, 3]
