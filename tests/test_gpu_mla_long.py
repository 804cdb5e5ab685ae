"""Latent attention over long caches on the GPU: what only runs of many steps reach.

A workgroup of the absorbed form takes a run of 32-position steps, and all CUs get one: a run has several
steps only where the call's sequences hold some 70000 positions together.  Here the sequences share one
set of blocks, so that the oracle works on one set of rows, all tokens at a time.
"""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import jero_hip as J
from mla_oracle import Problem, THETA, rotate

pytestmark = pytest.mark.gpu

TYPES = [("f32", "f16"), ("f16", "f16"), ("f32", "f32")]


class Shared(Problem):
    """Sequences of `lens` positions, all over the blocks of the longest.  `stairs` nats are added to the scores of
    every second head at three places (by the key part, whose queries come rotated: theta 0)."""

    def __init__(self, seed, lens, new, stairs=0.0, **kw):
        super().__init__(seed, [max(lens)], [1], max_len=max(lens), **kw)
        g = np.random.default_rng(seed + 1)
        self.theta = 0.0 if stairs else THETA
        self.lens, self.new = list(lens), list(new)
        self.c = self.visible(0, max(lens) - 1)
        self.table = np.repeat(self.table, len(lens), 0)
        self.starts = np.cumsum([0] + self.new).astype(np.int32)
        self.T = int(self.starts[-1])
        q = g.standard_normal((self.T, self.H, self.N + self.P)) * 1.5
        if stairs:
            self.c[:, self.R] = np.searchsorted([3300, 3860, 4420], np.arange(max(lens)), side="right")
            for j in range(max(lens)):
                self.rows[self.table[0, j // self.block], j % self.block, self.R] = self.c[j, self.R]
            q[:, :, self.N] = 0
            q[:, ::2, self.N] = stairs / self.scale
        self.q = q.astype(self.q.dtype)

    def attention(self, theta=None):
        """Problem.attention and Problem.bound for all tokens of a head at once; a score's own error weighs its own
        position, so that positions far below the maximum do not widen the bounds."""
        theta = self.theta if theta is None else theta
        half = self.act == "f16"
        u, f = 2.0 ** (-11 if half else -22) / math.sqrt(3), 2.0 ** -24
        n, c, c2, s, R, N = self.R + self.P + self.N, self.c, self.c ** 2, self.scale, self.R, self.N
        out, far = np.zeros((self.T, self.H, self.V)), np.zeros((self.T, self.H, 2))
        pos = np.array([p for _, _, p in self.tokens()])
        hidden = np.arange(len(c))[None, :] > pos[:, None]
        for h in range(self.H):
            wk, wv, q = self.wk[h].astype(np.float64), self.wv[h].astype(np.float64), self.q[:, h].astype(np.float64)
            qp = np.stack([rotate(x, p, theta) for x, p in zip(q[:, N:], pos)]) if theta else q[:, N:]
            q = np.concatenate([q[:, :N], qp], 1)
            qa = np.concatenate([q[:, :N] @ wk, qp], 1)
            k, v = c[:, :R] @ wk.T, c[:, :R] @ wv.T
            a = np.where(hidden, -np.inf, s * (qa @ c.T))
            under = a.max(1, keepdims=True) - a
            p = np.exp(-under)
            p /= p.sum(1, keepdims=True)
            o = p @ v
            prod = np.sqrt(np.maximum((qa ** 2 @ c2.T).max(1), (q ** 2 @ np.concatenate([k ** 2, c2[:, R:]], 1).T).max(1)))
            inner = np.sqrt((q[:, :N] ** 2 @ wk ** 2).max(1) * c2.sum(1).max())
            ds = s * (math.sqrt(2) * u * prod + f * math.sqrt(n) * (prod + inner))[:, None] + \
                np.where(hidden, 0, under) * 2.0 ** -22
            w = (p * ds) ** 2
            apart = w @ v ** 2 - 2 * o * (w @ v) + o ** 2 * w.sum(1, keepdims=True)
            lat = ((p ** 2) @ c2[:, :R] + (p @ c[:, :R]) ** 2) @ (wv ** 2).T
            each = np.maximum(apart, 0) + (2 * u * u + f * f * (n + len(c))) * ((p ** 2) @ v ** 2 + lat + o * o)
            each = each + (2.0 ** -11 / math.sqrt(3) * o if half else f * o) ** 2
            out[:, h], far[:, h, 0], far[:, h, 1] = o, 8 * np.sqrt(each.max(1)), np.sqrt(each.mean(1))
        return out, far

    def steps(self):
        """Steps of the longest run, by the plan's rule: equal runs of the items' units (steps, and 3 an item)."""
        share = min(64 // self.H, -(-self.T // len(self.lens))) if self.T > len(self.lens) and self.H <= 32 else 1
        rows = share * self.H
        at = 16 if rows <= 16 else 32 if rows <= 32 else 128 if rows > 64 and self.act == "f16" else 64
        groups = -(-rows // at)
        runs = 8 if groups >= 32 else 256 // groups // 8 * 8
        items = []
        for n, L in zip(self.new, self.lens):
            items += [-(-min(L, L - n + i + share) // 32) + 3 for i in range(0, n, share)]
        return -(-sum(items) // runs) - 3


# sixteen sequences of odd lengths; one token each and several
LENS = [4700 - 13 * i for i in range(16)]
ONE, TWO_ = [1] * 16, [2] * 16
BIG = dict(rank=512, rope=64, nope=16, v=24)
LONG = [(h, new, t, BIG) for t in TYPES for h, new in ((5, ONE), (20, ONE), (40, ONE), (5, TWO_), (20, TWO_))]
LONG += [(66, ONE, ("f16", "f16"), BIG), (128, ONE, ("f16", "f16"), BIG), (66, ONE, ("f32", "f32"), BIG)]
LONG += [(h, ONE, t, d) for d in (dict(rank=120, rope=24), dict(rank=248, rope=40)) for t in TYPES for h in (5, 40, 66)
         if h < 66 or t[0] == "f16"]


@pytest.mark.parametrize("stairs", [0.0, 6.5], ids=["level", "stairs"])
@pytest.mark.parametrize("heads,new,types,dims", LONG, ids=lambda x: "-".join(map(str, x.values() if isinstance(x, dict) else x))
                         if not isinstance(x, int) else f"h{x}")
def test_runs_of_many_steps(dev, heads, new, types, dims, stairs):
    """Every ring buffer is used again, maxima grow by 2^9 within runs (stairs), and block ids are read anew."""
    act, kv = types
    print(f"mla absorbed {act} {kv} {heads} heads, {new[0]} tokens, {dims}, stairs {stairs}", flush=True)
    p = Shared(50, LENS, new, heads=heads, act=act, kv=kv, block=2 if heads in (5, 66) else 64, stairs=stairs,
               **{**dict(nope=16, v=24), **dims})
    assert p.steps() >= 5
    p.device(dev, starts=new != ONE)
    print("  off by", p.check(p.run("absorbed", theta=p.theta), what="long"), flush=True)


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("heads,new", [(5, ONE), (20, ONE), (7, TWO_), (35, ONE), (70, ONE)], ids=lambda x: str(x) if isinstance(x, int) else f"new{x[0]}")
def test_bits_do_not_hang_on_what_the_workspace_held(dev, heads, new, act, kv):
    """Heads that do not fill 16s: the same bits over workspaces of zeros, of NaN, and of any values."""
    print(f"mla absorbed {act} {kv} {heads} heads, {new[0]} tokens", flush=True)
    p = Shared(52, LENS, new, heads=heads, act=act, kv=kv, block=64, rank=64, rope=16, nope=16, v=24).device(dev, starts=new != ONE)
    need = J.lib().jero_hip_mla_absorbed_workspace_bytes(p.cache.ref, p.T, heads)
    want = p.run("absorbed", workspace=torch.zeros(need, dtype=torch.uint8, device=dev))
    g = torch.Generator(device=dev).manual_seed(1)
    for ws in [torch.full((need,), 255, dtype=torch.uint8, device=dev)] + \
            [torch.randint(0, 256, (need,), dtype=torch.uint8, device=dev, generator=g) for _ in range(4)]:
        got = p.run("absorbed", workspace=ws)
        torch.cuda.synchronize()
        assert torch.equal(got, want), (got != want).sum().item()


# ---------------------------------------------------------------- one peak over a long tail


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("peak", [0, 5000, 8192])
@pytest.mark.parametrize("nats", [10.0, 13.0, 16.0, 17.375])
@pytest.mark.parametrize("form,heads", [("absorbed", 1), ("absorbed", 20), ("absorbed", 40), ("absorbed", 70), ("expanded", 1)])
def test_a_peak_over_thousands_of_small_numerators(dev, form, heads, nats, peak, act, kv):
    """One position of value 0, and 8192 of value 1 with scores `nats` below it, in one run: their small
    numerators add up to what is seen of them.

    Scores and values are exact.  A numerator's relative error: the exponent's three f32 roundings and its
    exponential's (nats 3 2^-24 + 2^-23), its parts' (2^-22, with f16 activations 2^-11), and, as f16 holds
    numerators 2^9 (expanded: 2^11) above their value, half its last place: 2^-34 (2^-36) of the peak.  The f32 sums
    of equal terms: 2^-24 a step of 32, for numerators and total."""
    print(f"mla {form} {act} {kv} {heads} heads: peak at {peak}, {nats} nats", flush=True)
    n, T = 8192, 512 if form == "absorbed" else 1
    p = Problem(51, [1], [1], heads=heads, rank=64, rope=16, nope=8, v=8, act=act, kv=kv, block=256)
    p.lens, p.new, p.T, p.max_len = [n + 1] * T, [1] * T, T, n + 1
    p.n_blocks = 33
    rows = np.zeros((33 * 256, 80), p.rows.dtype)
    rows[:, 1] = 1
    rows[peak] = 0
    rows[peak, 0] = nats
    p.rows = rows.reshape(33, 256, 80)
    p.table = np.repeat(np.arange(33, dtype=np.int32)[None], T, 0)
    p.starts = np.arange(T + 1, dtype=np.int32)
    p.wk[:], p.wv[:] = 0, 0
    p.wk[:, 0, 0] = 1
    p.wv[:, :, 1] = 1
    p.q = np.zeros((T, heads, 24), p.q.dtype)
    p.q[..., 0] = 1
    p.scale = 1.0
    p.device(dev, starts=False)
    kw = {}
    if form == "expanded":  # a workspace without room for partial rows: the positions stay in one run
        c = J.HipLatentCache.from_buffer_copy(p.cache.c)
        c.max_len = 1
        need = J.lib().jero_hip_mla_prefill_workspace_bytes(C.byref(c), J.F16 if act == "f16" else J.F32, 1, 8, 8, n + 1)
        kw = dict(workspace=torch.empty(need, dtype=torch.uint8, device=dev))
    got = p.run(form, theta=0.0, **kw).double().cpu().numpy()
    small = math.exp(-nats)
    exact = n * small / (1 + n * small)
    half = act == "f16"
    each = nats * 3 * 2.0 ** -24 + 2.0 ** -23 + (2.0 ** -11 if half else 2.0 ** -22) + \
        2.0 ** (-34 if form == "absorbed" else -36) / small
    far = exact * each + 2 * exact * (n / 32 + 64) * 2.0 ** -24 + exact * (2.0 ** -11 if half else 2.0 ** -22)
    print(f"  {np.abs(got - exact).max() / far:.3g} of {far / exact:.3g}", flush=True)
    assert (np.abs(got - exact) <= far).all()


# ---------------------------------------------------------------- the largest calls


@pytest.mark.parametrize("act,kv", TYPES)
def test_the_most_heads(dev, act, kv):
    print(f"mla {act} {kv} 1024 heads", flush=True)
    p = Problem(53, [70, 33], [1, 2], heads=1024, nope=8, v=8, act=act, kv=kv, pad_rows=1).device(dev)
    ref = p.attention()
    for form in ("absorbed", "expanded"):
        p.check(p.run(form), ref, form)


@pytest.mark.parametrize("starts", [False, True])
def test_the_most_tokens(dev, starts):
    """2^19 sequences of a token each, of 0 to 2 positions over one block, whose 192 different rows repeat."""
    print(f"mla append and absorbed, 2^19 sequences, starts {starts}", flush=True)
    n, few = 1 << 19, 192
    p = Problem(54, [2], [1], heads=1, nope=8, v=8, rank=8, rope=8)
    p.lens, p.new, p.T = [i % 3 for i in range(few)], [1] * few, few
    p.table = np.repeat(p.table, few, 0)
    p.starts = np.arange(few + 1, dtype=np.int32)
    p.q = np.random.default_rng(1).standard_normal((few, 1, 16)).astype(np.float32)
    ref = p.attention()
    p.device(dev, starts=starts)
    p.check(p.run("absorbed"), ref, "few")
    d = p.d
    again = lambda t: t.repeat((n + few - 1) // few, *[1] * (t.dim() - 1))[:n].contiguous()  # noqa: E731
    cache = J.LatentCache(d["rows"], again(d["table"]), again(d["lens"]), 8, max_len=p.max_len,
                          starts=torch.arange(n + 1, dtype=torch.int32, device=dev) if starts else None)
    out = torch.full((n, 1, 8), 7.0, device=dev)
    J.mla_absorbed_attention(out, again(d["q"]), cache, d["k_b"], d["v_b"], p.scale, THETA)
    torch.cuda.synchronize()
    p.check(out[:few], ref, "first")
    whole = out[:n // few * few].view(-1, few, 8)
    assert torch.equal(whole, whole[:1].expand_as(whole)) and torch.equal(out[n // few * few:, 0], whole[0, :n % few])
    # each token into a row of its own
    rows = torch.zeros((n // 16, 16, 16), dtype=torch.float16, device=dev)
    table = torch.arange(n, dtype=torch.int32, device=dev).view(-1, 1) // 16
    lens = torch.arange(n, dtype=torch.int32, device=dev) % 16 + 1
    x = torch.randn((n, 16), device=dev)
    J.mla_append(J.LatentCache(rows, table, lens, 8, starts=cache.starts), x, None, 0.0, 0.0)
    torch.cuda.synchronize()
    assert torch.equal(rows.view(n, 16), x.half())


def test_the_most_sequences_of_the_expanded_form(dev):
    print("mla expanded, 4096 sequences", flush=True)
    n = 4096
    lens = [(37 * i) % 19 for i in range(n)]
    p = Problem(55, lens, [min(L, 1 + i % 3) for i, L in enumerate(lens)], heads=1, nope=8, v=8, rank=8, rope=8, block=4,
                pad_rows=1).device(dev)
    p.check(p.run("expanded"), what="expanded")
