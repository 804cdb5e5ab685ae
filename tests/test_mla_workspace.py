"""Workspace sizes of the expanded form, without a GPU, and what a call makes of them, on one."""
import ctypes as C

import pytest
import torch

import jero_hip as J
from mla_oracle import THETA, Problem


def size(n_heads, total, max_len, act=J.F32, nope=32, v=40):
    c = J.HipLatentCache(rows_dev=1 << 16, table_dev=1 << 16, lens_dev=1 << 16, n_blocks=8, table_stride=1 << 12, n_seqs=2,
                         max_len=max_len, block_size=1024, kv_dtype=J.KV_F16, rank=64, rope_dim=16)
    return J.lib().jero_hip_mla_prefill_workspace_bytes(C.byref(c), act, n_heads, nope, v, total)


def test_sizes_of_one_head_and_of_the_least():
    """One head's call gets room for partial rows like any other's, where positions may be cut; 0 heads: the least."""
    assert size(0, 5000, 5000) == size(0, 5000, 200) == size(1, 5000, 200) < size(1, 5000, 5000)
    assert size(2, 5000, 5000) - size(2, 5000, 200) == size(1, 5000, 5000) - size(1, 5000, 200)
    assert size(0, 1 << 20, 1 << 20, J.F16, 128, 128) == size(1, 1 << 20, 256, J.F16, 128, 128)
    assert size(-1, 5000, 5000) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "f16"])
def test_one_head_is_cut_into_runs_as_two_are(dev, act):
    """A token at the end of 3000 positions: of one head, the bits of the same head among two."""
    p = Problem(80, [3000], [1], heads=2, act=act, block=64).device(dev)
    both = p.run("expanded")
    out = torch.zeros_like(both[:, :1])
    got = J.mla_prefill_attention(out, p.d["q"][:, :1].contiguous(), p.cache, p.d["kv_b"][:1].contiguous(), p.total(),
                                  p.scale, THETA)
    least = torch.empty(J.lib().jero_hip_mla_prefill_workspace_bytes(
        p.cache.ref, J.F16 if act == "f16" else J.F32, 0, p.N, p.V, p.total()), dtype=torch.uint8, device=dev)
    whole = p.run("expanded", workspace=least)
    torch.cuda.synchronize()
    p.check(both)
    p.check(whole)
    assert torch.equal(got, both[:, :1])
    if act == "f32":  # (f16's rounding hides the order of the sums)
        assert not torch.equal(whole, both)


@pytest.mark.gpu
def test_heads_that_do_not_fit_at_once_leave_the_partial_rows_their_room(dev):
    """A workspace of two heads' rows and of partial rows, for six heads: two at a time and cut, not all six in the
    partial rows' place and not cut."""
    p = Problem(81, [3000], [1], heads=6, block=64).device(dev)
    want = p.run("expanded")
    c = J.HipLatentCache.from_buffer_copy(p.cache.c)
    L = J.lib()
    two = L.jero_hip_mla_prefill_workspace_bytes(p.cache.ref, J.F32, 2, p.N, p.V, p.total())
    got = p.run("expanded", workspace=torch.empty(two, dtype=torch.uint8, device=dev))
    c.max_len = 1  # without partial rows
    rows = L.jero_hip_mla_prefill_workspace_bytes(C.byref(c), J.F32, 6, p.N, p.V, p.total())
    whole = p.run("expanded", workspace=torch.empty(rows, dtype=torch.uint8, device=dev))
    torch.cuda.synchronize()
    p.check(got)
    assert torch.equal(got, want) and not torch.equal(whole, want)


@pytest.mark.gpu
@pytest.mark.parametrize("total", [-1, 0, (1 << 23) + 1, 1 << 40])
def test_totals_are_refused_before_their_workspace_is_made(dev, total):
    p = Problem(82, [20], [2]).device(dev)
    with pytest.raises(J.K3Error) as ei:
        p.run("expanded", total=total)
    assert ei.value.variant == "TensorBoundsError"
