"""Keys and values that are not finite near the start of a cache, in steps that some of a tile's rows see whole and others do
not: who attends to them gets nothing finite, the others what they got without them."""
import numpy as np
import pytest
import torch

from test_gpu_paged_attention import TYPES, Problem

pytestmark = pytest.mark.gpu


def spoil(p, block, at, what):
    p.v[block, at, 0, 3] = what
    p.k[block, at, 1, 5] = np.nan


def check(p, ref, sees, what):
    out = p.run()
    half = p.H // 2
    assert not torch.isfinite(out[sees, :half, 3]).any(), f"{what}: a value that was attended to is lost"
    assert not torch.isfinite(out[sees, half:]).any(), f"{what}: a key that was attended to is lost"
    good = torch.from_numpy(ref[0]).to(out)
    out[sees] = good[sees]
    p.check(out, ref, what=what)


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("pos", [0, 5, 40])
@pytest.mark.parametrize("heads,dim", [(2, 64), (2, 128), (4, 80), (2, 256)])
def test_a_prompt(dev, heads, dim, pos, act, kv):
    """One prompt from its first token on: its rows' tiles hold waves that begin before the position and behind it."""
    for what in (np.inf, np.nan):
        p = Problem(31, [130], [130], heads, 2, dim, 16, 0, act, kv, one=False)
        ref = p.oracle()
        spoil(p, p.table[0, pos // 16], pos % 16, what)
        p.device(dev)
        print(f"paged_attention {act} {kv} {heads} heads of {dim}, {what} at {pos}", flush=True)
        check(p, ref, torch.arange(p.T, device=dev) >= pos, f"{what}")


@pytest.mark.parametrize("act,kv", TYPES)
def test_shared_positions(dev, act, kv):
    """One sequence ends before the position, in the first wave's rows; the others, in other waves too, see it."""
    p = Problem(32, [3] + [600] * 44, [1] * 45, 16, 8, 128, 32, 16, act, kv)
    ref = p.oracle()
    b = p.shared[0]
    p.v[b, 5, 2, 7] = np.inf
    p.device(dev)
    out = p.run()
    assert not torch.isfinite(out[1:, 4:6, 7]).any()
    out[1:, 4:6] = torch.from_numpy(ref[0][1:, 4:6]).to(out)
    p.check(out, ref)
