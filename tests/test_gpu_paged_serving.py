"""The paged operators as a server uses them, together: steps of requests with drafted tokens behind a shared prompt, a layer
of attention in between; every step against a plain 64-bit run of each request by itself."""
import numpy as np
import pytest
import torch

import jero_hip as J
import paged_oracle as P

pytestmark = pytest.mark.gpu

V, E, H, KV, D, BLOCK, SHARED, COLS = 97, 48, 8, 2, 64, 16, 3, 24
DRAFTS = 3
THETA, SCALE = 1e4, D ** -0.5


class Layer:
    """Embeddings and projections in f32, and the same in 64 bits for the plain run."""

    def __init__(self, seed):
        r = np.random.default_rng(seed)
        self.emb = r.normal(size=(V, E)).astype(np.float32)
        self.wq, self.wk, self.wv = (r.normal(size=(E, n * D)).astype(np.float32) / 7 for n in (H, KV, KV))
        self.wo = r.normal(size=(H * D, V)).astype(np.float32) / 12
        self.freq, self.m = P.frequencies(D, THETA, "yarn", 4.0, 32)

    def rows(self, token, pos):
        """(q, k, v) of one token in 64 bits, q and k rotated, k and v as the f16 cache holds them."""
        x = self.emb[token].astype(np.float64)
        q, k, v = ((x @ w.astype(np.float64)).reshape(1, -1, D) for w in (self.wq, self.wk, self.wv))
        q, k = (P.rotated(a, [pos], self.freq, self.m, "half") for a in (q, k))
        return q[0], k[0], v[0]

    def attend(self, tokens):
        """Attention of the last token of `tokens` over all of them, [H][D]."""
        rows = [self.rows(t, i) for i, t in enumerate(tokens)]
        k, v = np.stack([r[1] for r in rows]), np.stack([r[2] for r in rows])
        out = np.zeros((H, D))
        for h in range(H):
            a = k[:, h * KV // H] @ rows[-1][0][h] * SCALE
            e = np.exp(a - a.max())
            out[h] = (e @ v[:, h * KV // H]) / e.sum()
        return out


class Server:
    def __init__(self, dev, seqs, seed, captured):
        self.dev, self.S, self.captured = dev, seqs, captured
        self.r = np.random.default_rng(seed)
        self.layer = Layer(seed)
        L = self.layer
        self.w = {n: torch.from_numpy(getattr(L, n)).to(dev) for n in ("emb", "wq", "wk", "wv", "wo")}
        self.n_blocks = SHARED + seqs * 6 + 5
        i32 = dict(dtype=torch.int32, device=dev)
        self.prompt = self.r.integers(0, V, SHARED * BLOCK)
        self.shared = torch.arange(SHARED, **i32)
        self.table = torch.full((seqs, COLS), -1, **i32)
        self.lens, self.owned, self.drop = (torch.zeros(seqs, **i32) for _ in range(3))
        self.free, self.n_free = torch.arange(SHARED, self.n_blocks + SHARED, **i32), torch.tensor([self.n_blocks - SHARED], **i32)
        self.free = self.free[:self.n_blocks].contiguous()
        self.k, self.v = (torch.full((self.n_blocks, BLOCK, KV, D), float("nan"), dtype=torch.float16, device=dev)
                          for _ in range(2))
        self.rope = J.Rope(D, THETA, scaling="yarn", factor=4.0, original=32)
        self.pool = J.BlockPool(self.table, self.lens, self.owned, self.free, self.n_free, self.n_blocks, BLOCK, SHARED)
        self.T = seqs * (1 + DRAFTS) + 40
        T = self.T
        self.new, self.starts, self.granted = torch.zeros(seqs, **i32), torch.zeros(seqs + 1, **i32), torch.zeros(seqs, **i32)
        self.positions, self.slots = torch.zeros(T, **i32), torch.zeros(T, dtype=torch.int64, device=dev)
        self.q, self.qr, self.out = (torch.zeros((T, H, D), device=dev) for _ in range(3))
        self.kn, self.vn = (torch.zeros((T, KV, D), device=dev) for _ in range(2))
        self.tokens, self.stand, self.accepted = torch.zeros(T, **i32), torch.zeros(T, **i32), torch.zeros(seqs, **i32)
        self.target, self.draft = torch.zeros((T, V), device=dev), torch.zeros((T - 1, V), device=dev)
        self.u, self.u_last = torch.zeros(T - 1, device=dev), torch.zeros(seqs, device=dev)
        self.text = [None] * seqs  # what stands, the last token not yet in the cache
        self.graphs = None
        # the shared prompt's rows
        x = self.w["emb"][torch.from_numpy(self.prompt).to(dev)]
        n = SHARED * BLOCK
        q, k, v = ((x @ self.w[w]).view(n, -1, D) for w in ("wq", "wk", "wv"))
        J.paged_append(self.k, self.v, torch.empty_like(q), q, k, v, torch.arange(n, **i32), torch.arange(n, device=dev), self.rope)

    def admit(self, s):
        self.text[s] = list(self.prompt) + list(self.r.integers(0, V, 1))
        self.table[s, :SHARED] = self.shared
        self.lens[s], self.owned[s], self.drop[s] = SHARED * BLOCK, SHARED, 0

    def first_half(self):
        J.paged_extend(self.pool, self.new, self.positions, self.slots, self.starts, drop=self.drop, granted=self.granted)
        J.paged_append(self.k, self.v, self.qr, self.q, self.kn, self.vn, self.positions, self.slots, self.rope)
        cache = J.PagedCache(self.k, self.v, self.table, self.lens, starts=self.starts, shared=self.shared)
        J.paged_attention(self.out, self.qr, cache, SCALE)

    def second_half(self):
        J.verify_drafts(self.stand, self.accepted, self.target, self.draft, self.tokens, self.starts, self.u, self.u_last,
                        dropped=self.drop)

    def call(self, which):
        if not self.captured:
            return (self.first_half, self.second_half)[which]()
        if self.graphs is None:
            # (captured while nothing is asked for: requests without tokens leave everything as it is)
            keep = self.new.clone(), self.drop.clone(), self.tokens.clone()
            self.new.zero_()
            self.drop.zero_()
            self.first_half()
            self.second_half()
            torch.cuda.synchronize()
            self.graphs = []
            for f in (self.first_half, self.second_half):
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    f()
                self.graphs.append(g)
            for t, was in zip((self.new, self.drop, self.tokens), keep):
                t.copy_(was)
        self.graphs[which].replay()

    def step(self, end):
        """One step: `end`, the requests that end with it."""
        rows, new = [], []
        for s in range(self.S):
            if self.text[s] is None or s in end:
                new.append(-1 if s in end else 0)
                continue
            n = int(self.r.integers(0, DRAFTS + 1))
            rows.append((s, [self.text[s][-1]] + list(self.r.integers(0, V, n))))
            new.append(n + 1)
        tokens = [t for _, ts in rows for t in ts]
        self.new.copy_(torch.tensor(new, dtype=torch.int32))
        self.tokens[:len(tokens)] = torch.tensor(tokens, dtype=torch.int32)
        x = self.w["emb"][self.tokens.long()]
        for dst, w in ((self.q, "wq"), (self.kn, "wk"), (self.vn, "wv")):
            torch.mm(x, self.w[w], out=dst.view(self.T, -1))
        self.call(0)
        assert (self.granted.cpu().numpy()[[s for s, _ in rows]] == 1).all()
        # the layer's output, and probabilities
        self.target.copy_(torch.softmax(2 * self.out.view(self.T, -1) @ self.w["wo"], 1))
        drafted = sum(len(ts) - 1 for _, ts in rows)
        q = self.r.dirichlet(np.ones(V), max(drafted, 1)).astype(np.float32)
        for i, t in enumerate(t for _, ts in rows for t in ts[1:]):  # the draft was fond of what it drafted
            q[i] *= 0.5
            q[i, t] += 0.5
        self.draft[:drafted] = torch.from_numpy(q[:drafted]).to(self.dev)
        # often enough accepted
        self.u.copy_(torch.from_numpy(self.r.random(self.T - 1, dtype=np.float32) * np.float32(0.05)))
        self.u_last.copy_(torch.from_numpy(self.r.random(self.S, dtype=np.float32)))
        self.call(1)
        torch.cuda.synchronize()
        self.check(rows, len(tokens))
        for s in end:
            self.text[s] = None

    def check(self, rows, n):
        starts = self.starts.cpu().numpy()
        out = self.out.double().cpu().numpy()
        lens, drop, owned = (t.cpu().numpy() for t in (self.lens, self.drop, self.owned))
        target = self.target.cpu().numpy()
        want, accepted, dropped = P.verify(target[:n], self.draft.cpu().numpy(), self.tokens.cpu().numpy()[:n], starts,
                                           self.u.cpu().numpy(), self.u_last.cpu().numpy())
        stand = self.stand.cpu().numpy()
        assert np.array_equal(stand[:n], want) and np.array_equal(drop, dropped)
        assert np.array_equal(self.accepted.cpu().numpy(), accepted)
        at = 0
        for s, ts in rows:
            assert starts[s] == at
            text = self.text[s]
            assert lens[s] == len(text) - 1 + len(ts)
            for i in (0, len(ts) - 1):  # attention of the first and the last of its tokens
                full = text[:-1] + ts[:i + 1]
                ref = self.layer.attend(full)
                # keys and values of the cache are f16 (2^-11 of each, keys' part in a score of 8 nats at most), the rest f32
                assert np.max(np.abs(out[at + i] - ref)) < 2.0 ** -11 * (2 * 8 + 2) * np.max(np.abs(ref)) + 1e-4
            a = accepted[s]
            self.text[s] = text[:-1] + ts[:a + 1] + [int(stand[at + a])]
            assert len(self.text[s]) - 1 == lens[s] - drop[s]
            at += len(ts)
        # every block is in one place
        ids = [i for s in range(self.S) for i in self.table[s, SHARED:max(owned[s], SHARED)].cpu().tolist()]
        ids += self.free[:int(self.n_free)].cpu().tolist()
        assert sorted(ids) == list(range(SHARED, self.n_blocks)), "blocks lost or held twice"


@pytest.mark.parametrize("captured", [False, True])
def test_requests_with_drafts_behind_a_shared_prompt(dev, captured):
    sv = Server(dev, 6, 3, captured)
    for s in range(6):
        sv.admit(s)
    grown = 0
    for i in range(12):
        end = {i % 6} if i % 4 == 3 else set()
        before = [0 if t is None else len(t) for t in sv.text]
        sv.step(end)
        grown = max(grown, max(len(t) - b for t, b in zip(sv.text, before) if t is not None and b))
        for s in end:  # its place is taken by another from the next step on
            sv.admit(s)
    assert grown >= 2, "no drafted token was ever accepted"
