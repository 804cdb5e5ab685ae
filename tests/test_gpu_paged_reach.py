"""Paged operators at sizes where another way is taken: chunks over more blocks than a wave keeps ids of, batches whose
sequences fill the card with wide tiles, more sequences than a workgroup's copies in LDS hold."""
import numpy as np
import pytest
import torch

from test_gpu_paged import Pool, step
from test_gpu_paged_attention import TYPES, Problem

pytestmark = pytest.mark.gpu


def run(p, dev, what):
    print(what, flush=True)
    p.device(dev)
    print("  off by", p.check(p.run(), what=what), flush=True)


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("block", [1, 2, 4, 8])
@pytest.mark.parametrize("heads,dim", [(4, 64), (8, 128), (2, 256)])
def test_chunks_over_many_blocks(dev, heads, dim, block, act, kv):
    """Single tokens (narrow tiles), more of them so that chunks get longer, and prompts (wide tiles); a block that is none,
    beyond the first 64."""
    lens = [1100, 700, 64 * block + 1] + [530] * 13
    for n, new, what in ((lens, [1] * 16, "16 single tokens"), (lens * 9, [1] * 144, "144 single tokens"),
                         (lens[:3], [150, 140, 2], "prompts")):
        p = Problem(41, n, new, heads, 2, dim, block, 0, act, kv)
        p.table[1, 600 // block] = p.n_blocks
        run(p, dev, f"paged_attention {act} {kv} {heads} heads of {dim}, blocks of {block}, {what}")


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("block", [1, 4])
def test_shared_chunks_over_many_blocks(dev, block, act, kv):
    lens = [700 + 3 * i for i in range(40)]
    run(Problem(42, lens, [1] * 40, 16, 8, 128, block, 640 // block, act, kv), dev,
        f"paged_attention {act} {kv} behind 640 shared positions, blocks of {block}")


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("kv_heads,group,dim", [(4, 8, 64), (4, 8, 128), (4, 24, 80), (8, 3, 256)])
def test_wide_tiles_that_fill_the_card(dev, kv_heads, group, dim, act, kv):
    """512 workgroups and more of 17 rows a sequence and more, with and without shared positions."""
    S = 130
    r = np.random.default_rng(dim)
    new = r.integers(1, 6, S) * -(-24 // group)
    for shared in (0, 2):
        lens = [int(shared * 32 + r.integers(0, 70)) + int(n) for n in new]
        run(Problem(43, lens, list(new), kv_heads * group, kv_heads, dim, 32, shared, act, kv, pad_rows=2), dev,
            f"paged_attention {act} {kv} {kv_heads} x {group} heads of {dim}, {S} sequences, {shared} shared blocks")


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("shared", [0, 12])
def test_more_than_1024_sequences(dev, shared, act, kv):
    """Their starts are searched in memory; some are empty, and rows before and behind them are nobody's."""
    S = 1100
    r = np.random.default_rng(3)
    new = [int(n) for n in r.integers(0, 3, S)]
    lens = [int(shared * 16 + r.integers(0, 40)) + n for n in new]
    lens[5], lens[1090] = 0, 1
    run(Problem(44, lens, new, 4, 1, 64, 16, shared, act, kv, pad_rows=3, before=2, one=False), dev,
        f"paged_attention {act} {kv} {S} sequences, {shared} shared blocks")
    run(Problem(45, lens, [1] * S, 4, 1, 64, 16, shared, act, kv), dev, f"paged_attention {act} {kv} {S} single tokens")


@pytest.mark.parametrize("seqs", [4096, 4097, 6000])
def test_extend_more_than_4096_requests(dev, seqs):
    r = np.random.default_rng(seqs)
    p = Pool(seqs, r.integers(0, 40, seqs), 12, 8, seqs * 2).device(dev)
    for i in range(4):
        new = r.integers(0, 9, seqs)
        new[r.random(seqs) < 0.2] = -1
        step(p, dev, new, np.minimum(r.integers(0, 3, seqs), p.lens) if i % 2 else None)


def test_extend_that_gives_back_many_blocks(dev):
    """1024 requests of 200 blocks each end in one launch, and others take them."""
    p = Pool(7, [800] * 1024, 256, 4, 3).device(dev)
    new = np.where(np.arange(1024) % 8 == 5, 4, -1)
    want = step(p, dev, new)
    assert want["granted"].all() and want["n_free"][0] == 3 + 896 * 200 - 128
