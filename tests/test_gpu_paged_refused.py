"""Requests that paged_extend refuses while drafted tokens are under way: verify_drafts takes nothing off them, and a server
whose pool runs dry keeps every position it has stored."""
import numpy as np
import pytest
import torch

import jero_hip as J
import paged_oracle as P
from test_gpu_paged import drafts, put
from test_gpu_paged_serving import DRAFTS, SHARED, V, Server

pytestmark = pytest.mark.gpu


def refused(want, starts, granted):
    """The oracle's results, but -1 and 0, 0 for the sequences that were refused."""
    out, accepted, dropped = (a.copy() for a in want)
    for s, ok in enumerate(granted):
        if not ok:
            out[starts[s]:max(starts[s + 1], starts[s])] = -1
            accepted[s] = dropped[s] = 0
    return out, accepted, dropped


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("rows,vocab", [([4], 50), ([3, 1, 5, 0, 2, 4], 333), ([3, 4, 1, 70], 70000), ([2, 5] * 40, 90)])
def test_verify_granted(dev, rows, vocab, draft):
    """By one launch and by two; the others' drafts keep their places behind a refused sequence's."""
    d = drafts(3, rows, vocab, draft=draft, near=0.3)
    n = len(rows)
    for granted in (np.ones(n, int), np.arange(n) % 2, np.zeros(n, int), (np.arange(n) + 1) % 2 * 5):
        out = torch.full((len(d["tokens"]),), -2, dtype=torch.int32, device=dev)
        acc, dropped = (torch.full((n,), 9, dtype=torch.int32, device=dev) for _ in range(2))
        J.verify_drafts(out, acc, put(dev, d["target"], torch.float32), put(dev, d["draft"], torch.float32),
                        put(dev, d["tokens"]), put(dev, d["starts"]), put(dev, d["u"], torch.float32),
                        put(dev, d["u_last"], torch.float32), dropped=dropped, granted=put(dev, granted))
        torch.cuda.synchronize()
        for name, got, want in zip(("out", "accepted", "dropped"), (out, acc, dropped),
                                   refused(P.verify(**d), d["starts"], granted)):
            assert np.array_equal(got.cpu().numpy(), want), (name, granted, got.cpu().numpy(), want)


class DryServer(Server):
    """A server of which all but `blocks` free blocks are held by others."""

    def __init__(self, dev, seqs, seed, captured, blocks):
        super().__init__(dev, seqs, seed, captured)
        self.held = self.free[blocks:int(self.n_free)].cpu().tolist()
        self.n_free.fill_(blocks)
        self.refusals = self.with_drafts = self.granted_again = 0
        self.asked = [None] * seqs  # the tokens that a refused request asks for again

    def second_half(self):
        J.verify_drafts(self.stand, self.accepted, self.target, self.draft, self.tokens, self.starts, self.u, self.u_last,
                        dropped=self.drop, granted=self.granted)

    def step(self, end):
        rows, new = [], []
        for s in range(self.S):
            if self.text[s] is None or s in end:
                new.append(-1 if s in end else 0)
                self.asked[s] = None
                continue
            ts = self.asked[s] or [self.text[s][-1]] + list(self.r.integers(0, V, int(self.r.integers(0, DRAFTS + 1))))
            rows.append((s, ts))
            new.append(len(ts))
        tokens = [t for _, ts in rows for t in ts]
        self.new.copy_(torch.tensor(new, dtype=torch.int32))
        self.tokens[:len(tokens)] = torch.tensor(tokens, dtype=torch.int32)
        x = self.w["emb"][self.tokens.long()]
        for dst, w in ((self.q, "wq"), (self.kn, "wk"), (self.vn, "wv")):
            torch.mm(x, self.w[w], out=dst.view(self.T, -1))
        self.call(0)
        self.target.copy_(torch.softmax(2 * self.out.view(self.T, -1) @ self.w["wo"], 1))
        drafted = len(tokens) - len(rows)
        q = self.r.dirichlet(np.ones(V), max(drafted, 1)).astype(np.float32)
        self.draft[:drafted] = torch.from_numpy(q[:drafted]).to(self.dev)
        self.u.copy_(torch.from_numpy(self.r.random(self.T - 1, dtype=np.float32) * np.float32(0.05)))
        self.u_last.copy_(torch.from_numpy(self.r.random(self.S, dtype=np.float32)))
        self.call(1)
        torch.cuda.synchronize()
        self.check(rows, len(tokens))
        for s in end:
            self.text[s] = None

    def check(self, rows, n):
        starts, granted = self.starts.cpu().numpy(), self.granted.cpu().numpy()
        out = self.out.double().cpu().numpy()
        lens, drop, owned = (t.cpu().numpy() for t in (self.lens, self.drop, self.owned))
        want, accepted, dropped = refused(P.verify(self.target.cpu().numpy()[:n], self.draft.cpu().numpy(),
                                                   self.tokens.cpu().numpy()[:n], starts, self.u.cpu().numpy(),
                                                   self.u_last.cpu().numpy()), starts, granted)
        stand = self.stand.cpu().numpy()
        assert np.array_equal(stand[:n], want) and np.array_equal(drop, dropped)
        assert np.array_equal(self.accepted.cpu().numpy(), accepted)
        for s, ts in rows:
            text, at = self.text[s], starts[s]
            if not granted[s]:
                self.refusals += 1
                self.with_drafts += len(ts) > 1
                self.asked[s] = ts
                assert lens[s] == len(text) - 1 and drop[s] == 0, "a refused request lost or gained positions"
                continue
            self.granted_again += self.asked[s] is not None
            self.asked[s] = None
            assert lens[s] == len(text) - 1 + len(ts)
            for i in (0, len(ts) - 1):
                ref = self.layer.attend(text[:-1] + ts[:i + 1])
                # keys and values of the cache are f16 (2^-11 of each, keys' part in a score of 8 nats at most), the rest f32
                assert np.max(np.abs(out[at + i] - ref)) < 2.0 ** -11 * (2 * 8 + 2) * np.max(np.abs(ref)) + 1e-4
            a = accepted[s]
            self.text[s] = text[:-1] + ts[:a + 1] + [int(stand[at + a])]
            assert len(self.text[s]) - 1 == lens[s] - drop[s]
        ids = [i for s in range(self.S) for i in self.table[s, SHARED:max(owned[s], SHARED)].cpu().tolist()]
        ids += self.free[:int(self.n_free)].cpu().tolist() + self.held
        assert sorted(ids) == list(range(SHARED, self.n_blocks)), "blocks lost or held twice"


@pytest.mark.parametrize("captured", [False, True])
def test_a_pool_that_runs_dry_with_drafts_under_way(dev, captured):
    sv = DryServer(dev, 6, 5, captured, 7)
    for s in range(6):
        sv.admit(s)
    for i in range(24):
        end = {i // 4 % 6} if i % 4 == 3 else set()
        sv.step(end)
        for s in end:
            sv.admit(s)
            sv.asked[s] = None
    print(f"{sv.refusals} refusals, {sv.with_drafts} with drafts, {sv.granted_again} granted later", flush=True)
    assert sv.with_drafts > 0 and sv.granted_again > 0
