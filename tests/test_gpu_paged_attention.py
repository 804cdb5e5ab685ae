"""Attention over a paged cache with shared first positions on the GPU, against the 64-bit oracle.

Pool rows that no sequence owns, and those past a length, hold NaN unless a test says otherwise, so a row read where
it must not be shows in the output."""
import numpy as np
import pytest
import torch

import jero_hip as J
import paged_oracle as P

pytestmark = pytest.mark.gpu

TYPES = [("f32", "f16"), ("f16", "f16"), ("f32", "f32")]
DTYPE = {"f32": torch.float32, "f16": torch.float16}


class Problem:
    """Sequences of lens positions, new[s] tokens each, whose first shared blocks are the same."""

    def __init__(self, seed, lens, new, heads, kv_heads, dim, block=16, shared=0, act="f32", kv="f16", rest=np.nan, pad_rows=0,
                 before=0, max_len=None, one=None, gain=1.0):
        r = np.random.default_rng(seed)
        self.H, self.KV, self.D, self.block, self.act, self.kv = heads, kv_heads, dim, block, act, kv
        self.lens, self.new, self.max_len = np.array(lens, np.int32), list(new), max_len
        self.one = all(n == 1 for n in new) if one is None else one
        S = len(lens)
        need = [max(-(-n // block) - shared, 0) for n in lens]
        self.n_blocks = shared + sum(need) + 2
        order = r.permutation(self.n_blocks).astype(np.int32)
        self.cols = max(max(need) + shared, -(-(max_len or 1) // block))
        self.shared = order[:shared]
        self.table = np.full((S, self.cols), 2 ** 30, np.int32)  # (columns of shared blocks are not read)
        kv_type = np.float32 if kv == "f32" else np.float16
        self.k, self.v = (np.full((self.n_blocks, block, kv_heads, dim), rest, kv_type) for _ in range(2))

        def fill(ids, n):
            for i, b in enumerate(ids):
                m = min(block, n - i * block)
                for pool in (self.k, self.v):
                    pool[b, :m] = r.normal(size=(m, kv_heads, dim)) * gain

        fill(self.shared, shared * block)
        at = shared
        for s in range(S):
            ids = order[at:at + need[s]]
            self.table[s, shared:shared + need[s]] = ids
            fill(ids, lens[s] - shared * block)
            at += need[s]
        self.before = before
        starts = before + np.concatenate([[0], np.cumsum(new)])
        self.starts = None if self.one else starts.astype(np.int32)
        self.T = int(starts[-1]) + pad_rows if not self.one else S
        self.q = (r.normal(size=(self.T, heads, dim)) * 1.5).astype(np.float32 if act == "f32" else np.float16)
        self.scale = dim ** -0.5

    def device(self, dev):
        self.d = {n: torch.from_numpy(getattr(self, n)).to(dev) for n in ("k", "v", "table", "lens", "q")}
        self.d["starts"] = None if self.starts is None else torch.from_numpy(self.starts).to(dev)
        self.d["shared"] = torch.from_numpy(self.shared).to(dev) if len(self.shared) else None
        self.cache = J.PagedCache(self.d["k"], self.d["v"], self.d["table"], self.d["lens"], starts=self.d["starts"],
                                  max_len=self.max_len, shared=self.d["shared"])
        return self

    def run(self, out=None, **kw):
        if out is None:
            out = torch.full(self.d["q"].shape, 7.0, dtype=self.d["q"].dtype, device=self.d["q"].device)
        J.paged_attention(out, self.d["q"], self.cache, self.scale, **kw)
        torch.cuda.synchronize()
        return out

    def oracle(self):
        return P.attend(self.q, self.k, self.v, self.table, self.lens, self.starts, self.scale, self.block, self.n_blocks,
                        self.shared, self.max_len)

    def check(self, got, ref=None, what=""):
        """Each result within a bound of its own.  With d the error of a score and w the sum of |v| under the softmax:
        scores are off by their largest sum of |q k| times 2^-22 for each factor of two parts and (D + 8) 2^-24 for the
        sums and the scaling (f32 additions, one after another at worst), plus 2^-22 of the score's size for the
        exponential's argument; numerators by 2^-21 (exponential, two parts) or 2^-11 (f16), twice (themselves and
        their sum), those below 2^-36 of the largest altogether; the sums over n positions by (n + 32) 2^-24 twice
        (rescalings and joins among the 32); then the result's own rounding."""
        out, size, most, seen = ref or self.oracle()
        got = got.double().cpu().numpy()
        live = ~np.isnan(out[:, 0, 0])
        assert (got[~live] == 7).all(), f"{what}: rows of no sequence"
        two = self.act == "f32"
        parts = 2.0 ** -22 * (two + (self.kv == "f32"))
        d = most * (parts + (self.D + 8) * 2.0 ** -24 + 2.0 ** -22)
        p = 2.0 ** -21 if two else 2.0 ** -11 + 2.0 ** -21
        n = seen[:, None]
        w = 2 * d + 2 * p + 2 * (n + 32) * 2.0 ** -24 + n * 2.0 ** -36 + (2.0 ** -22 if self.kv == "f32" else 0)
        half = 2.0 ** -24 if two else 2.0 ** -11
        bound = size * w[:, :, None] + np.abs(out) * half + (2.0 ** -25 if not two else 0) + \
            (2.0 ** -25 if self.kv == "f32" else 0)
        err = np.abs(got - out)[live] / np.maximum(bound[live], 1e-300)
        assert np.isfinite(got[live]).all(), f"{what}: not finite"
        assert err.max() <= 1, f"{what}: off by {err.max()} of the bound"
        return err.max()


# lens, new, heads, kv_heads, dim, block, shared blocks: each edge of the tiles (16, 32, 64 positions; 16, 32, 64, 128
# rows), pages that end inside one, sequences of one token and of none, one and many heads of a group
CASES = [
    ([1], [1], 1, 1, 8, 16, 0),
    ([2], [2], 3, 3, 64, 1, 0),
    ([15, 16, 17], [1, 1, 1], 10, 2, 64, 4, 0),
    ([31, 32, 33, 34], [1, 3, 0, 2], 8, 2, 40, 16, 0),
    ([63, 64, 65], [1, 1, 1], 8, 8, 128, 64, 0),
    ([127, 128, 129, 1], [2, 1, 1, 1], 32, 8, 128, 32, 0),
    ([300], [1], 17, 1, 80, 16, 0),
    ([1300], [1], 64, 1, 128, 64, 0),
    ([257, 40], [1, 4], 40, 2, 96, 256, 0),
    ([130, 131], [1, 1], 4, 2, 256, 8, 0),
    ([700], [2], 40, 2, 200, 16, 0),
    ([17, 18, 40], [1, 1, 1], 8, 2, 64, 16, 1),          # a shared block
    ([200] * 9, [1] * 9, 4, 2, 128, 64, 3),              # 18 rows over the shared positions
    ([131, 140, 128, 129, 300], [1, 2, 0, 1, 4], 8, 1, 80, 16, 8),
    ([600] * 20, [1] * 20, 8, 2, 64, 32, 16),            # 80 rows
    ([600, 513, 530] * 13, [1] * 39, 16, 4, 128, 16, 32),  # 156 rows, more than a tile
    ([100, 70, 66] * 3, [1, 2, 1] * 3, 32, 1, 256, 64, 1),
    ([80, 90], [1, 1], 128, 1, 128, 16, 4),              # 128 rows of a token
    ([65], [1], 8, 2, 128, 64, 1),                       # one sequence: nobody to share with
]
PROMPTS = [
    ([130], [130], 2, 2, 64, 16, 0),
    ([64, 65, 129], [64, 65, 129], 6, 2, 128, 32, 0),
    ([300, 20, 257], [17, 20, 200], 8, 2, 128, 16, 0),
    ([97, 256], [31, 128], 3, 1, 72, 4, 0),
    ([140], [140], 4, 1, 256, 64, 0),
    ([400, 330, 390, 321], [40, 9, 60, 1], 4, 2, 96, 32, 10),   # 55 rows a sequence on average
    ([700, 520, 612], [180, 6, 100], 8, 2, 128, 64, 8),         # tiles filled by sequences
    ([1100], [70], 16, 2, 64, 16, 0),
]


def ids(c):
    return "-".join(map(str, c[0][:5])) + f"_n{len(c[0])}_h{c[2]}.{c[3]}.{c[4]}_b{c[5]}_s{c[6]}"


def problem(case, act="f32", kv="f16", **kw):
    lens, new, H, KV, D, block, shared = case
    return Problem(sum(lens) + H, lens, new, H, KV, D, block, shared, act, kv, **kw)


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("case", CASES + PROMPTS, ids=ids)
def test_against_the_oracle(dev, case, act, kv):
    print(f"paged_attention {act} {kv} {case}", flush=True)
    p = problem(case, act, kv).device(dev)
    print("  off by", p.check(p.run()), flush=True)
    q = problem(case, act, kv, pad_rows=3, before=2, one=False).device(dev)  # the same with starts, and rows of nobody
    q.check(q.run(), what="with starts")


# Batches that go over their shared positions together (which pays from 48 MB spared on): few rows, 17 to 32 of them, more
# than a tile of 128; one and several tiles of a sequence's own rows, narrow and wide ones
SHARED = [
    ([780] + [770] * 8, [1] * 9, 16, 16, 128, 16, 48),
    ([1600] * 12, [1] * 12, 32, 16, 64, 64, 24),
    ([850, 834, 833, 840] * 6, [1] * 24, 16, 16, 80, 32, 26),
    ([515, 600, 513] * 14, [1] * 42, 32, 8, 128, 16, 32),
    ([530, 514, 513, 640] * 5, [1, 2, 0, 5] * 5, 40, 8, 256, 64, 8),
    ([800, 705, 720] * 8, [4, 5, 1] * 8, 64, 8, 96, 64, 11),
    ([1100, 1054] * 14, [12, 14] * 14, 16, 4, 128, 16, 65),
]


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("case", SHARED, ids=ids)
def test_shared_positions(dev, case, act, kv):
    print(f"paged_attention {act} {kv} {case}", flush=True)
    p = problem(case, act, kv, pad_rows=0 if case[1] == [1] * len(case[1]) else 2).device(dev)
    print("  off by", p.check(p.run()), flush=True)


@pytest.mark.parametrize("act,kv", TYPES)
def test_shared_positions_that_not_all_see(dev, act, kv):
    """Empty sequences, the first among them, sequences that end within the shared positions, ids that are none, positions
    from max_len on; values that are not finite are for those who see them."""
    lens = [0, 600, 513, 100, 1, 530, 0, 512, 511] * 5
    p = Problem(21, lens, [1] * 45, 16, 8, 128, 32, 16, act, kv, max_len=520)
    p.shared[3] = -5
    p.shared[9] = p.n_blocks
    p.table[1, 16] = p.n_blocks
    ref = p.oracle()
    b = p.shared[512 // 32 - 1]
    p.v[b, 30, 2, 7] = np.inf  # position 510: for the sequences of 511 positions and more
    p.k[b, 29, 5, 1] = np.nan  # position 509
    p.device(dev)
    out = p.run()
    sees = torch.tensor([n >= 511 for n in lens], device=dev)
    assert not torch.isfinite(out[sees][:, 4:6, 7]).any() and not torch.isfinite(out[sees][:, 10:12]).any()
    good = torch.from_numpy(ref[0]).to(out)
    out[sees, 4:6] = good[sees, 4:6]
    out[sees, 10:12] = good[sees, 10:12]
    p.check(out, ref)
    assert (out[0] == 0).all() and (out[6] == 0).all()


def test_shared_positions_captured(dev):
    """Replays over other lengths, tables and queries, with eager calls between; two graphs that share a workspace."""
    p = Problem(22, [600] * 40, [1] * 40, 16, 8, 128, 16, 32).device(dev)
    n = J.lib().jero_hip_paged_attention_workspace_bytes(p.cache.ref, J.F32, p.T, p.H)
    assert n > 0
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    outs = [torch.zeros_like(p.d["q"]) for _ in range(2)]
    graphs = []
    for out in outs:
        J.paged_attention(out, p.d["q"], p.cache, p.scale, workspace=ws)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            J.paged_attention(out, p.d["q"], p.cache, p.scale, workspace=ws)
        graphs.append(g)
    r = np.random.default_rng(3)
    for i in range(4):
        p.lens = r.integers(0, 601, 40).astype(np.int32)
        p.q = np.roll(p.q, 1, 0)
        p.d["lens"].copy_(torch.from_numpy(p.lens))
        p.d["q"].copy_(torch.from_numpy(p.q))
        for g, out in zip(graphs, outs):
            out.fill_(5)
            g.replay()
        torch.cuda.synchronize()
        eager = p.run(workspace=ws)
        assert torch.equal(outs[0], eager) and torch.equal(outs[1], eager)
    p.check(eager)


@pytest.mark.parametrize("shared", [0, 2])
@pytest.mark.parametrize("dim", [64, 128])
def test_rows_that_see_nothing_get_zeros(dev, shared, dim):
    """An empty sequence, a sequence of more tokens than positions, and one without tokens."""
    p = Problem(5, [0, 3, 70, 100, -5], [1, 5, 0, 2, 1], 6, 2, dim, 16, shared, pad_rows=3).device(dev)
    out = p.run()
    p.check(out)
    assert (out[0] == 0).all() and (out[1:3] == 0).all() and (out[8] == 0).all() and (out[3] != 0).any()


def test_a_padded_batch(dev):
    """Half of the sequences of a step are empty, among them the first, beside shared positions."""
    lens = [0, 90, 0, 64, 0, 200, 65, 0]
    for kv in ("f16", "f32"):
        p = Problem(6, lens, [1] * 8, 16, 4, 128, 16, 4, kv=kv).device(dev)
        out = p.run()
        p.check(out)
        assert all((out[s] == 0).all() == (lens[s] == 0) for s in range(8))


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("shared", [0, 3])
def test_bad_blocks_are_masked(dev, shared, act, kv):
    """Ids outside the pool are not followed: their positions are masked."""
    p = Problem(7, [100, 90, 60], [1, 2, 1], 10, 2, 64, 16, shared, act, kv)
    p.table[0, 4] = p.n_blocks
    p.table[0, 6] = -1
    p.table[1, 3] = 2 ** 31 - 1
    p.table[2, shared:] = -(2 ** 31)
    if shared:
        p.shared[1] = -1
    p.device(dev)
    p.check(p.run())


@pytest.mark.parametrize("shared", [0, 2, 4])
def test_positions_from_max_len_on_are_not_attended_to(dev, shared):
    p = Problem(8, [100, 70, 64], [3, 1, 1], 6, 3, 64, 16, shared, max_len=50).device(dev)
    p.check(p.run())


@pytest.mark.parametrize("case", [([50, 17, 129], [2, 1, 1], 4, 2, 64, 16, 1), ([200, 150], [90, 40], 4, 2, 128, 16, 0)], ids=ids)
def test_masked_places_may_hold_anything(dev, case):
    """The rows past each length and the blocks of others hold infinities, or the type's lowest value."""
    for rest in (np.inf, -np.inf, np.finfo(np.float16).min):
        p = problem(case, rest=rest).device(dev)
        p.check(p.run(), what=str(rest))


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("new,heads,dim", [(4, 4, 64), (5, 8, 128), (70, 4, 128), (4, 2, 256)])
def test_values_that_are_not_finite_stay_with_those_who_see_them(dev, new, heads, dim, act, kv):
    """An infinite value and a NaN key at the position of the last token but one: the tokens before it get what they got
    without, it and the one after it nothing finite (in the heads of its group)."""
    p = Problem(9, [200, 77], [new, 1], heads, 2, dim, 16, 0, act, kv)
    ref = p.oracle()
    pos = 200 - 2
    b = p.table[0, pos // 16]
    p.v[b, pos % 16, 0, 3] = np.inf
    p.k[b, pos % 16, 1, 5] = np.nan
    p.device(dev)
    out = p.run()
    assert not torch.isfinite(out[new - 2:new, :heads // 2, 3]).any()
    assert not torch.isfinite(out[new - 2:new, heads // 2:]).any()
    out[new - 2:new] = torch.from_numpy(ref[0][new - 2:new]).to(out)
    p.check(out, ref)


def test_scores_far_apart(dev):
    """Peaks, and rows whose largest score comes last: 60 nats between positions."""
    for act, kv in TYPES:
        p = Problem(10, [500, 700, 300], [1, 1, 1], 8, 2, 64, 16, 4, act, kv)
        p.q *= 6
        p.device(dev)
        p.check(p.run(), what=f"{act} {kv}")


def test_queries_of_any_size_and_either_sign_of_scale(dev):
    p = Problem(11, [150, 70], [1, 1], 4, 2, 128, 16, 0)
    p.q[0] *= np.float32(2.0 ** 40)
    p.q[1] *= np.float32(2.0 ** -40)
    p.scale = -2.0 ** -40 / 11
    p.device(dev)
    p.check(p.run())


def test_tensors_apart_and_a_workspace_of_ones_own(dev):
    """Tokens' rows apart in q and out, a workspace that held something else, on a stream of its own."""
    p = Problem(12, [900, 650, 700], [1, 2, 1], 16, 4, 128, 64, 8).device(dev)
    want = p.run()
    wide = torch.full((p.T, 2, p.H, p.D), 3.0, device=dev)
    wide[:, 1] = p.d["q"]
    out = torch.full((p.T, p.H + 1, p.D), 7.0, device=dev)
    n = J.lib().jero_hip_paged_attention_workspace_bytes(p.cache.ref, J.F32, p.T, p.H)
    assert n > 0
    ws = torch.full((n,), 255, dtype=torch.uint8, device=dev)
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream())
    J.paged_attention(out[:, :p.H], wide[:, 1], p.cache, p.scale, workspace=ws, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(out[:, :p.H], want) and (out[:, p.H] == 7).all()
    with pytest.raises(J.K3Error):
        J.paged_attention(out[:, :p.H], wide[:, 1], p.cache, p.scale, workspace=ws[:n - 256])


def test_captured(dev):
    """One step captured, replayed over other lengths, tables and queries, with eager calls between."""
    p = Problem(13, [300, 200, 260], [1, 1, 1], 8, 2, 64, 16, 8).device(dev)
    out = torch.zeros_like(p.d["q"])
    ws = torch.empty(J.lib().jero_hip_paged_attention_workspace_bytes(p.cache.ref, J.F32, p.T, p.H), dtype=torch.uint8, device=dev)
    J.paged_attention(out, p.d["q"], p.cache, p.scale, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        J.paged_attention(out, p.d["q"], p.cache, p.scale, workspace=ws)
    for i, lens in enumerate(([300, 200, 260], [129, 0, 200], [250, 199, 130], [300, 200, 1])):
        p.lens = np.array(lens, np.int32)
        p.q = np.roll(p.q, 1, 0)
        p.d["lens"].copy_(torch.from_numpy(p.lens))
        p.d["q"].copy_(torch.from_numpy(p.q))
        out.fill_(5)
        g.replay()
        torch.cuda.synchronize()
        eager = p.run(workspace=ws)
        assert torch.equal(out, eager)
        p.check(out, what=f"replay {i}")


def test_runs_repeat(dev):
    """The same bits each time, whatever the workspace held."""
    for case in (CASES[15], PROMPTS[5], PROMPTS[6], SHARED[0], SHARED[4]):
        p = problem(case).device(dev)
        a = p.run()
        for _ in range(3):
            assert torch.equal(a, p.run())
