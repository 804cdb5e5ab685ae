"""Block tables, rotation and storing, and drafted tokens on the GPU, against the 64-bit oracle."""
import numpy as np
import pytest
import torch

import jero_hip as J
import paged_oracle as P

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- block tables


class Pool:
    """Requests that hold hist positions, in blocks of a random order; the rest of the pool free but for `others`."""

    def __init__(self, seed, hist, cols, block, free, shared=0, others=3):
        r = np.random.default_rng(seed)
        S = len(hist)
        self.block, self.shared, self.cols = block, shared, cols
        need = [max(-(-h // block), shared) for h in hist]
        own = [n - shared for n in need]
        self.n_blocks = shared + sum(own) + free + others
        ids = r.permutation(self.n_blocks).astype(np.int32)
        self.table = np.full((S, cols), -7, np.int32)
        at = shared
        for s in range(S):
            self.table[s, :shared] = ids[:shared]
            self.table[s, shared:need[s]] = ids[at:at + own[s]]
            at += own[s]
        self.free = np.full(self.n_blocks, -9, np.int32)
        self.free[:free] = ids[at:at + free]
        self.n_free = np.array([free], np.int32)
        self.lens, self.owned = np.array(hist, np.int32), np.array(need, np.int32)

    def device(self, dev):
        self.d = {n: torch.from_numpy(getattr(self, n).copy()).to(dev) for n in ("table", "lens", "owned", "free", "n_free")}
        self.pool = J.BlockPool(self.d["table"], self.d["lens"], self.d["owned"], self.d["free"], self.d["n_free"],
                                self.n_blocks, self.block, self.shared)
        return self


def put(dev, a, dtype=torch.int32):
    return None if a is None else torch.tensor(np.asarray(a), dtype=dtype, device=dev)


def step(p, dev, new, drop=None, spare=3, tokens=None, into=False, stream=None):
    """One call, checked in everything it writes; the pool's own arrays become what the call left."""
    T = tokens or max(1, int(np.maximum(new, 0).sum()) + spare)
    want = P.extend(p.table, p.lens, p.owned, p.free, p.n_free[0], new, drop, T, p.block, p.n_blocks, p.shared)
    got = dict(positions=torch.full((T + 2,), 77, dtype=torch.int32, device=dev), slots=torch.full((T + 2,), 77, device=dev),
               starts=torch.zeros(len(new) + 1, dtype=torch.int32, device=dev),
               granted=torch.zeros(len(new), dtype=torch.int32, device=dev))
    outs = None
    if into:
        outs = [torch.full_like(p.d[n], 55) for n in ("lens", "owned", "n_free")]
    J.paged_extend(p.pool, put(dev, new), got["positions"][:T], got["slots"][:T], got["starts"], drop=put(dev, drop),
                   granted=got["granted"], into=outs, stream=stream)
    torch.cuda.synchronize()
    assert (got["positions"][T:] == 77).all() and (got["slots"][T:] == 77).all()
    got["positions"], got["slots"] = got["positions"][:T], got["slots"][:T]
    got.update(p.d)
    if into:
        for n, t in zip(("lens", "owned", "n_free"), outs):
            assert np.array_equal(p.d[n].cpu().numpy(), getattr(p, n)), f"{n} changed"
            got[n] = t
    for n, w in want.items():
        assert np.array_equal(got[n].cpu().numpy(), w), (n, got[n].cpu().numpy(), w)
    for n in ("table", "free"):
        setattr(p, n, want[n])
    if not into:
        for n in ("lens", "owned", "n_free"):
            setattr(p, n, want[n])
    return want


EXTEND = [
    # hist, new, block, cols, free, shared
    ([0], [1], 16, 4, 4, 0),
    ([15, 16, 17, 0], [1, 1, 1, 0], 16, 4, 9, 0),
    ([5, 9, 3], [-1, 20, 0], 4, 16, 0, 0),            # what one gives back another takes
    ([5, 9, 3], [-1, 20, 13], 4, 16, 1, 0),           # the second finds too few left
    ([7, 7, 7, 7], [9, 40, 1, 1], 8, 8, 3, 0),        # a refused request keeps the later ones that need blocks waiting
    ([32, 40, 48], [3, -1, 17], 16, 8, 6, 2),         # two shared blocks each
    ([100], [29], 1, 128, 40, 0),
    ([100, 20], [29, 108], 1, 128, 200, 0),
    ([100, 20], [29, 109], 1, 128, 200, 0),           # past the table row
    ([0] * 70, [1] * 70, 256, 2, 70, 0),
    ([3, 1], [-5, -1], 2, 4, 2, 0),
    ([10], [-1], 16, 1, 0, 1),                        # only a shared block: nothing goes back
]


@pytest.mark.parametrize("into", [False, True])
@pytest.mark.parametrize("case", EXTEND, ids=lambda c: f"{c[0][:4]}-{c[1][:4]}-b{c[2]}-f{c[4]}-s{c[5]}")
def test_extend(dev, case, into):
    hist, new, block, cols, free, shared = case
    step(Pool(1, hist, cols, block, free, shared).device(dev), dev, new, into=into)


@pytest.mark.parametrize("seqs,block,most", [(1, 16, 5000), (64, 16, 3), (500, 4, 30), (1024, 16, 3), (1025, 16, 2), (3000, 8, 40)])
def test_extend_many_steps(dev, seqs, block, most):
    """Steps after each other, with drafts taken back, requests that end and are admitted again, and a stack that runs
    dry; the larger ones by two launches."""
    r = np.random.default_rng(seqs)
    hist = r.integers(0, 60, seqs)
    p = Pool(seqs, hist, 6000 // block if seqs == 1 else 64, block, seqs * 2 + 10).device(dev)
    for i in range(5):
        new = r.integers(0, most + 1, seqs)
        new[r.random(seqs) < 0.15] = -1
        drop = np.minimum(r.integers(0, 4, seqs), p.lens) if i % 2 else None
        step(p, dev, new, drop, tokens=None if i != 3 else max(1, int(np.maximum(new, 0).sum()) // 2))
    assert (p.n_free[0] >= 0)


def test_extend_values_out_of_range(dev):
    """Counts beyond their arrays are taken as the arrays' ends, ids beyond the pool give no slot."""
    p = Pool(3, [5, 6, 7, 8], 4, 4, 6).device(dev)
    for name, v in (("owned", [9, -3, 2, 2]), ("lens", [5, 6, -4, 8]), ("n_free", [1000])):
        setattr(p, name, np.array(v, np.int32))
        p.d[name].copy_(torch.from_numpy(getattr(p, name)))
    p.table[0, :] = [-1, p.n_blocks, 2 ** 31 - 1, 0]
    p.d["table"].copy_(torch.from_numpy(p.table))
    step(p, dev, [7, 3, 2, 1], drop=[0, 100, 1, -5])


def test_extend_captured(dev):
    """A captured step, replayed with other requests each time."""
    p = Pool(5, [3, 30, 17], 16, 8, 40).device(dev)
    new = torch.zeros(3, dtype=torch.int32, device=dev)
    T = 12
    out = [torch.zeros(T, dtype=torch.int32, device=dev), torch.zeros(T, dtype=torch.int64, device=dev),
           torch.zeros(4, dtype=torch.int32, device=dev)]
    J.paged_extend(p.pool, new, *out)  # (nothing asked for)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        J.paged_extend(p.pool, new, *out)
    for asked in ([1, 1, 1], [0, 9, 2], [-1, 1, 0], [10, 0, 1]):
        new.copy_(put(dev, asked))
        g.replay()
        torch.cuda.synchronize()
        want = P.extend(p.table, p.lens, p.owned, p.free, p.n_free[0], asked, None, T, p.block, p.n_blocks)
        for n in ("table", "lens", "owned", "free", "n_free"):
            assert np.array_equal(p.d[n].cpu().numpy(), want[n]), n
            setattr(p, n, want[n])
        for n, t in zip(("positions", "slots", "starts"), out):
            assert np.array_equal(t.cpu().numpy(), want[n]), n


# ---------------------------------------------------------------- rotation and storing

F16 = np.float16
# half a step of each type, relative
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11}


def held(got, ref, size, dtype, steps32):
    """Each element within its own rounding to dtype (half a step, or half the least step near zero) and `steps32`
    half steps of 32 bits of the row's size."""
    got, tiny = got.double().cpu().numpy(), (2.0 ** -25 if dtype is torch.float16 else 0.0)
    bound = np.abs(ref) * HALF[dtype] * (1 + 1e-6) + size * steps32 * 2.0 ** -24 * (1 + 2.0 ** -10) + tiny
    worst = np.max(np.abs(got - ref) / np.maximum(bound, 1e-300))
    assert worst <= 1, f"off by {worst} of the bound"


APPEND = [
    # tokens, heads, kv, dim, rot, layout, scaling
    (1, 1, 1, 8, 8, "half", "none"),
    (3, 4, 2, 64, 64, "half", "yarn"),
    (5, 6, 3, 80, 24, "interleaved", "linear"),
    (130, 3, 1, 128, 128, "interleaved", "wavelength"),
    (33, 8, 8, 96, 72, "half", "ntk"),
    (17, 5, 1, 256, 256, "half", "none"),
    (7, 40, 4, 200, 8, "half", "linear"),
    (1100, 2, 1, 72, 40, "interleaved", "yarn"),
]


@pytest.mark.parametrize("act", [torch.float32, torch.float16])
@pytest.mark.parametrize("kv_type", [torch.float32, torch.float16])
@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("case", APPEND, ids=lambda c: "-".join(map(str, c)))
def test_append(dev, case, normed, act, kv_type):
    """Queries, keys and values out of a wider row.  In half steps of 32 bits (2^-24) of a pair's size: the angle,
    2 turns rounded to 32 bits, is off by pi 2^-25, 1.6; cosine and sine by 2 units in the last place, 4, and the product
    with the magnitude, 1: each by 6.6, together sqrt(2) of that, 9.3; the two products 1, their sum 1: below 13.  The
    norm: 8 squares a lane and 5 sums over lanes, half of their 13 through the root; mean and eps likewise 1; root,
    quotient and two products 4: below 12."""
    T, H, KV, D, rot, layout, scaling = case
    print(f"paged_append {case} {act} {kv_type} norm {normed}", flush=True)
    g = torch.Generator(device=dev).manual_seed(T + H)
    x = (torch.randn((T, 8 + (H + 2 * KV) * D + 16), generator=g, device=dev) * 1.5).to(act)
    q, k, v = (x[:, 8 + a * D:8 + b * D].unflatten(1, (b - a, D)) for a, b in ((0, H), (H, H + KV), (H + KV, H + 2 * KV)))
    r = np.random.default_rng(T)
    pos = r.integers(0, 1 << 20, T).astype(np.int32)
    pos[0] = 0
    n_slots = 2 * T + 9
    slots = r.permutation(n_slots)[:T].astype(np.int64)
    if T > 4:
        pos[2], slots[1], slots[3], slots[4] = -1, -1, n_slots, 1 << 40
    args = dict(scaling=scaling, factor=4.0, original=4096)
    rope = J.Rope(rot, 1e4, layout=layout, **args)
    pools = [torch.full((n_slots, KV, D), 3.25, dtype=kv_type, device=dev) for _ in range(2)]
    norms = [1 + 0.2 * torch.randn(D, generator=g, device=dev) for _ in range(2)] if normed else [None, None]
    out = torch.full((T, H + 1, D), 9.0, dtype=act, device=dev)
    J.paged_append(*pools, out[:, :H], q, k, v, torch.from_numpy(pos).to(dev), torch.from_numpy(slots).to(dev), rope,
                   q_norm=norms[0], k_norm=norms[1], eps=1e-5)
    torch.cuda.synchronize()
    freq, m = P.frequencies(rot, 1e4, **args)
    steps = 13 + (12 if normed else 0)
    live = pos >= 0
    assert (out[:, H] == 9).all() and (out[:, :H].cpu()[~live] == 9).all()
    nm = [None if n is None else n.cpu().numpy() for n in norms]
    want = P.rotated(q.cpu().numpy(), pos, freq, m, layout, nm[0], 1e-5)

    def size(w):  # of each element's pair
        n, z = rot // 2, np.abs(w).copy()
        a, b = (z[..., :n], z[..., n:rot]) if layout == "half" else (z[..., 0:rot:2], z[..., 1:rot:2])
        both = np.hypot(a, b)
        if layout == "half":
            z[..., :n], z[..., n:rot] = both, both
        else:
            z[..., 0:rot:2], z[..., 1:rot:2] = both, both
        return z

    held(out[:, :H].cpu()[live], want[live], size(want)[live], act, steps)
    stored = live & (slots >= 0) & (slots < n_slots)
    kw = P.rotated(k.cpu().numpy(), pos, freq, m, layout, nm[1], 1e-5)
    for rows, ref, s in ((pools[0], kw, steps), (pools[1], v.double().cpu().numpy(), 0)):
        rows = rows.cpu()
        held(rows[slots[stored]], ref[stored], size(ref)[stored], kv_type, s)
        rest = np.setdiff1d(np.arange(n_slots), slots[stored])
        assert (rows[rest] == 3.25).all()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_alone_and_in_place(dev, layout):
    """rope is paged_append's rotation of queries; onto its own input it gives the same bits."""
    g = torch.Generator(device=dev).manual_seed(2)
    x = torch.randn((37, 5, 96), generator=g, device=dev)
    pos = torch.randint(0, 3000, (37,), generator=g, device=dev).int()
    r = J.Rope(64, 5e5, layout=layout, scaling="wavelength", factor=8.0, original=2048)
    out = J.rope(torch.zeros_like(x), x, pos, r)
    freq, m = P.frequencies(64, 5e5, "wavelength", 8.0, 2048)
    want = P.rotated(x.cpu().numpy(), pos.cpu().numpy(), freq, m, layout)
    assert np.max(np.abs(out.double().cpu().numpy() - want)) < 13 * 2.0 ** -24 * np.max(np.abs(want)) * 1.5
    assert torch.equal(out[..., 64:], x[..., 64:])
    y = x.clone()
    J.rope(y, y, pos, r)
    torch.cuda.synchronize()
    assert torch.equal(y, out)
    z = J.rope(torch.zeros_like(x), x, torch.zeros_like(pos), r)
    torch.cuda.synchronize()
    assert torch.equal(z, x)


def test_append_rows_far_apart(dev):
    """A pool whose rows pass 2^31 elements, and one query row 2^31 elements behind another."""
    KV, D = 8, 128
    n = (1 << 31) // (KV * D) + 100
    pools = [torch.zeros((n, KV, D), dtype=torch.float16, device=dev) for _ in range(2)]
    base = torch.zeros(((1 << 31) + 4096,), dtype=torch.float16, device=dev)
    q = base.as_strided((2, 2, D), (1 << 31, D, 1))
    q.copy_(torch.arange(4 * D, device=dev).view(2, 2, D) % 7)
    k = torch.ones((2, KV, D), dtype=torch.float16, device=dev)
    out = torch.zeros((2, 2, D), dtype=torch.float16, device=dev)
    slots = torch.tensor([n - 1, 5], device=dev)
    J.paged_append(*pools, out, q, k, 2 * k, torch.tensor([0, 0], dtype=torch.int32, device=dev), slots, J.Rope(D, 1e4))
    torch.cuda.synchronize()
    assert torch.equal(out, q) and (pools[0][[n - 1, 5]] == 1).all() and (pools[1][[n - 1, 5]] == 2).all()
    assert pools[0].count_nonzero() == 2 * KV * D


# ---------------------------------------------------------------- drafted tokens


def drafts(seed, rows, V, near=0.5, draft=True):
    r = np.random.default_rng(seed)
    T = sum(rows)
    N = sum(max(n - 1, 0) for n in rows)
    soft = lambda x: (np.exp(x - x.max(-1, keepdims=True)) / np.exp(x - x.max(-1, keepdims=True)).sum(-1, keepdims=True))  # noqa: E731
    z = r.normal(size=(T, V)) * 2
    target = soft(z).astype(np.float32)
    starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    tokens = r.integers(0, V, T).astype(np.int32)
    q = np.zeros((N, V), np.float32)
    i = 0
    for s, n in enumerate(rows):
        for j in range(1, n):
            q[i] = soft(z[starts[s] + j - 1] + near * r.normal(size=V))
            tokens[starts[s] + j] = r.choice(V, p=q[i].astype(np.float64) / q[i].astype(np.float64).sum())
            i += 1
    return dict(target=target, draft=q if draft else None, tokens=tokens, starts=starts, u=r.random(N, dtype=np.float32),
                u_last=r.random(len(rows), dtype=np.float32))


def check_verify(dev, d, pad=2):
    """The call against the oracle; draft, target and outputs have rows and columns more than the call's."""
    V = d["target"].shape[1]
    T = len(d["tokens"])

    def wide(a):
        if a is None:
            return None
        w = torch.full((a.shape[0], V + pad), 0.5, device=dev)
        w[:, :V] = torch.from_numpy(a)
        return w[:, :V]

    out = torch.full((T,), -2, dtype=torch.int32, device=dev)
    acc, dropped = (torch.full((len(d["starts"]) - 1,), 9, dtype=torch.int32, device=dev) for _ in range(2))
    J.verify_drafts(out, acc, wide(d["target"]), wide(d["draft"]), put(dev, d["tokens"]), put(dev, d["starts"]),
                    put(dev, d["u"], torch.float32), put(dev, d["u_last"], torch.float32), dropped=dropped)
    torch.cuda.synchronize()
    want = P.verify(**d)
    for n, g, w in zip(("out", "accepted", "dropped"), (out, acc, dropped), want):
        assert np.array_equal(g.cpu().numpy(), w), (n, g.cpu().numpy(), w)
    return want


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("rows,V", [([1], 1), ([1], 50), ([2], 7), ([4], 4096), ([3, 1, 5], 4097), ([2, 0, 4, 0, 0, 3], 1000),
                                    ([6] * 20, 333), ([70, 2, 130], 65), ([3] * 4, 40000), ([2] * 300, 90)])
def test_verify(dev, rows, V, draft):
    for seed in range(3):
        want = check_verify(dev, drafts(seed, rows, V, draft=draft, near=(0.1, 0.7, 2.0)[seed]))
    assert (want[0][want[0] != -2] < V).all()


def test_verify_borders(dev):
    """Numbers at 0 and just below 1, probabilities of 0 and 1, a draft that is the target, a drafted token that is none,
    and weights that are not finite."""
    d = drafts(1, [3, 3, 3, 3, 3, 3], 100)
    below = np.nextafter(np.float32(1), np.float32(0))
    d["draft"][0:2] = d["target"][0:2]              # always accepted while u < 1
    d["u"][0:2], d["u_last"][0] = below, below
    d["draft"][2, :] = d["target"][3, :]            # refused with nothing left over: the target itself
    d["target"][3, d["tokens"][4]] = 0
    d["draft"][2, d["tokens"][4]] = 0.5
    d["u"][2], d["u_last"][1] = 0, 0
    d["tokens"][7] = -1
    d["tokens"][10] = 100
    d["target"][6, 5], d["target"][9, 3], d["target"][9, 4] = np.nan, np.inf, -1
    d["target"][12:15] = 0                          # nothing to draw from
    d["u"][8:10] = 0
    d["target"][15:18, :] = 0
    d["target"][15:18, 42] = 1                      # one token has it all
    d["u_last"][5] = below
    want = check_verify(dev, d)
    assert want[1][0] == 2 and want[0][12] == -1
    for v in (0.0, below):
        d["u_last"][:] = v
        check_verify(dev, d)
    d["draft"] = None
    check_verify(dev, d)


@pytest.mark.parametrize("V", [50, 70000])
def test_verify_starts_out_of_order(dev, V):
    """Starts that fall and whose counts of drafts add up to 2^32 - 4: no number is read before the first, so the
    sequence behind them has no drafts of its own, and stands on its last token alone."""
    d = drafts(5, [4], V)
    top = (1 << 31) - 1
    starts = torch.tensor([0, top, 0, top, 0, 4], dtype=torch.int32, device=dev)
    out, acc, dropped = (torch.full((n,), 9, dtype=torch.int32, device=dev) for n in (4, 5, 5))
    J.verify_drafts(out, acc, put(dev, d["target"], torch.float32), put(dev, d["draft"], torch.float32), put(dev, d["tokens"]),
                    starts, put(dev, d["u"], torch.float32), torch.full((5,), 0.5, device=dev), dropped=dropped)
    torch.cuda.synchronize()
    assert acc.tolist()[1::2] == [0, 0] and acc[4] == 0 and dropped.tolist()[1::2] == [0, 0] and dropped[4] == 3


def test_verify_is_the_targets_distribution(dev):
    """What stands or is drawn for the first place is distributed as the target's row, whatever the draft: over 20000
    chats of one drafted token, each of 8 tokens' counts within 5 standard deviations."""
    n, V = 20000, 8
    r = np.random.default_rng(4)
    p, q = r.dirichlet(np.ones(V)).astype(np.float32), r.dirichlet(np.ones(V)).astype(np.float32)
    tokens = np.zeros(2 * n, np.int32)
    tokens[1::2] = r.choice(V, size=n, p=q.astype(np.float64) / q.astype(np.float64).sum())
    out, acc = torch.zeros(2 * n, dtype=torch.int32, device=dev), torch.zeros(n, dtype=torch.int32, device=dev)
    J.verify_drafts(out, acc, torch.from_numpy(np.tile(p, (2 * n, 1))).to(dev), torch.from_numpy(np.tile(q, (n, 1))).to(dev),
                    put(dev, tokens), put(dev, np.arange(n + 1) * 2), put(dev, r.random(n), torch.float32).clamp(max=1 - 2 ** -24),
                    put(dev, r.random(n), torch.float32).clamp(max=1 - 2 ** -24))
    counts = np.bincount(out[::2].cpu().numpy(), minlength=V)
    assert np.all(np.abs(counts - n * p) < 5 * np.sqrt(n * p * (1 - p)) + 1)
