"""Latent attention in 64 bits from its definition, problems to run it on, and the tolerances.

The oracle works a sequence and a head at a time in the expanded form (a head's keys and values made
from the latents), on the values the device holds (f16 or f32 caches and weights, widened).
"""
import math

import numpy as np

THETA, EPS = 10000.0, 1e-6


def rotate(x, pos, theta=THETA):
    """x [..., P] at position pos: pairs (2i, 2i + 1) turned by pos * theta^(-2i/P)."""
    P = x.shape[-1]
    a = pos * theta ** (-2.0 * np.arange(P // 2) / P)
    c, s = np.cos(a), np.sin(a)
    out = np.empty_like(x)
    out[..., 0::2] = x[..., 0::2] * c - x[..., 1::2] * s
    out[..., 1::2] = x[..., 0::2] * s + x[..., 1::2] * c
    return out


def off(got, exact, bounds):
    """The largest error of an element, over what its row allows, and the root mean square of all errors, over
    twice what is expected: each has to be at most 1."""
    err = np.abs(got - exact)
    far = (err.max(-1) / np.maximum(bounds[..., 0], 1e-300)).max() if err.any() else 0.0
    rms = np.sqrt((err ** 2).mean()) / max(2 * np.sqrt((bounds[..., 1] ** 2).mean()), 1e-300)
    return far, rms


class Problem:
    """Sequences of `lens` positions whose last `new` are the call's tokens, over a pool with its blocks in a
    random order.  Every pool row that no sequence owns, and every one past a length, holds `rest`."""

    def __init__(self, seed, lens, new, heads=4, rank=64, rope=16, nope=32, v=40, block=16, act="f32", kv="f16", rest=np.nan,
                 max_len=None, gain=1.5, pad_rows=0):
        g = np.random.default_rng(seed)
        self.lens, self.new, self.H, self.R, self.P, self.N, self.V, self.block = \
            list(lens), list(new), heads, rank, rope, nope, v, block
        self.act, self.kv = act, kv
        A = np.float32 if act == "f32" else np.float16
        K = np.float32 if kv == "f32" else np.float16
        self.max_len = max_len or max(1, max(self.lens))
        need = [-(-max(n, 0) // block) for n in self.lens]
        self.n_blocks = sum(need) + 2
        order = g.permutation(self.n_blocks)
        stride = max(max(need), -(-self.max_len // block))
        self.table = np.full((len(self.lens), stride), -1, np.int32)
        self.rows = np.full((self.n_blocks, block, rank + rope), rest, K)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
            for p in range(max(self.lens[i], 0)):
                self.rows[self.table[i, p // block], p % block] = g.standard_normal(rank + rope).astype(K)
        self.starts = np.cumsum([0] + self.new).astype(np.int32)
        self.T = int(self.starts[-1]) + pad_rows
        self.q = (g.standard_normal((self.T, heads, nope + rope)) * gain).astype(A)
        self.x = (g.standard_normal((self.T, rank + rope)) * 1.7).astype(A)
        self.norm = (1 + 0.1 * g.standard_normal(rank)).astype(np.float32)
        self.wk = (g.standard_normal((heads, nope, rank)) / math.sqrt(rank)).astype(np.float16)
        self.wv = (g.standard_normal((heads, v, rank)) / math.sqrt(rank)).astype(np.float16)
        self.scale = float(np.float32(1 / math.sqrt(nope + rope)))

    def tokens(self):
        """(row, sequence, position) of the call's tokens."""
        for s, (n, L) in enumerate(zip(self.new, self.lens)):
            for i in range(n):
                yield int(self.starts[s]) + i, s, L - n + i

    def visible(self, s, pos):
        """The positions a token at pos attends to, and their rows in 64 bits."""
        js = [j for j in range(min(pos + 1, self.max_len)) if 0 <= self.table[s, j // self.block] < self.n_blocks]
        return np.array([self.rows[self.table[s, j // self.block], j % self.block] for j in js],
                        np.float64).reshape(-1, self.R + self.P)

    def attention(self, theta=THETA, causal=True, turn=True):
        """(out [T][H][V], bounds [T][H][2]): the attention of every token in 64 bits (rows of no sequence NaN), and
        how far a computed row may be off (see bound)."""
        out = np.full((self.T, self.H, self.V), np.nan)
        far = np.zeros((self.T, self.H, 2))
        wk, wv = self.wk.astype(np.float64), self.wv.astype(np.float64)
        for t, s, pos in self.tokens():
            c = self.visible(s, pos if causal else self.lens[s] - 1)
            if not len(c):
                out[t] = 0
                continue
            q = self.q[t].astype(np.float64)
            qp = rotate(q[:, self.N:], pos, theta) if turn and theta else q[:, self.N:]
            for h in range(self.H):
                k = c[:, :self.R] @ wk[h].T
                v = c[:, :self.R] @ wv[h].T
                a = self.scale * (k @ q[h, :self.N] + c[:, self.R:] @ qp[h])
                p = np.exp(a - a.max())
                p /= p.sum()
                out[t, h] = p @ v
                qa = np.concatenate([wk[h].T @ q[h, :self.N], qp[h]])
                far[t, h] = self.bound(c, qa, q[h], qp[h], k, v, p, a, wk[h], wv[h])
        return out, far

    def bound(self, c, qa, q, qp, k, v, p, a, wk, wv):
        """(far, std): how far an element of an output row may be from the exact one, and the standard deviation
        expected of it.

        u is half a step of the factors: 2^-22 for the two-part products of f32 activations, 2^-11 for f16;
        f = 2^-24 one f32 rounding.  A rounding is uniform within its half step (deviation / sqrt 3) and
        independent of the others.  A score is a sum of n products of two rounded factors (2 u^2 of their squares),
        summed in f32 (f sqrt(n) of their root of squares, and the same for the absorbed query or expanded key
        inside it), its hardware exponential adds |a - max| 2^-22.  With scores off by ds_j, out is off by
        sum p_j ds_j (v_j - out); the rounded numerators, values (and the absorbed form's latent) by u of the root
        of the squares that they weigh, the f32 sums over positions and rank by f sqrt of their number, and the
        output's own rounding by half its step.  far is eight of these deviations."""
        half = self.act == "f16"
        u, f = 2.0 ** (-11 if half else -22) / math.sqrt(3), 2.0 ** -24
        n, o = self.R + self.P + self.N, p @ v
        prod = max(np.sqrt((qa ** 2 * c ** 2).sum(1).max()),
                   np.sqrt((k ** 2 * q[:self.N] ** 2).sum(1).max() + (c[:, self.R:] ** 2 * qp ** 2).sum(1).max()))
        inner = np.sqrt((q[:self.N] ** 2 @ wk ** 2).max() * (c ** 2).sum(1).max())
        ds = self.scale * (math.sqrt(2) * u * prod + f * math.sqrt(n) * (prod + inner)) + \
            np.abs(a - a.max()).max() * 2.0 ** -22
        apart = (p[:, None] * (v - o)) ** 2
        wide = (p[:, None] * v) ** 2
        lat = ((p[:, None] * c[:, :self.R]) ** 2).sum(0) @ (wv ** 2).T + (p @ c[:, :self.R]) ** 2 @ (wv ** 2).T
        each = ds ** 2 * apart.sum(0) + (2 * u * u + f * f * (n + len(c))) * (wide.sum(0) + lat + o * o)
        each = each + (2.0 ** -11 / math.sqrt(3) * o if half else f * o) ** 2
        return 8 * np.sqrt(each.max()), np.sqrt(each.mean())

    def appended(self, theta=THETA, norm=True):
        """The pool after mla_append, in 64 bits before the rounding to its type: (rows, touched)."""
        rows = self.rows.astype(np.float64)
        hit = np.zeros(rows.shape[:2], bool)
        for t, s, pos in self.tokens():
            if not 0 <= pos < self.max_len or not 0 <= self.table[s, pos // self.block] < self.n_blocks:
                continue
            x = self.x[t].astype(np.float64)
            c = x[:self.R]
            if norm:
                c = c / np.sqrt((c ** 2).mean() + EPS) * self.norm.astype(np.float64)
            b = self.table[s, pos // self.block]
            rows[b, pos % self.block] = np.concatenate([c, rotate(x[self.R:], pos, theta) if theta else x[self.R:]])
            hit[b, pos % self.block] = True
        return rows, hit

    # ---------------------------------------------------------------- on the device

    def device(self, dev, starts=True):
        import torch
        import jero_hip as J
        up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
        self.d = dict(rows=up(self.rows), table=up(self.table), lens=up(np.array(self.lens, np.int32)), q=up(self.q),
                      x=up(self.x), norm=up(self.norm), k_b=up(self.wk.transpose(0, 2, 1)), v_b=up(self.wv),
                      kv_b=up(np.concatenate([self.wk, self.wv], 1)), starts=up(self.starts) if starts else None)
        self.cache = J.LatentCache(self.d["rows"], self.d["table"], self.d["lens"], self.R, starts=self.d["starts"],
                                   max_len=self.max_len)
        return self

    def total(self):
        return max(1, sum(min(max(n, 0), self.max_len) for n in self.lens))

    def run(self, form, out=None, theta=THETA, **kw):
        import torch
        import jero_hip as J
        d = self.d
        if out is None:
            out = torch.full((self.T, self.H, self.V), 7.0, dtype=d["q"].dtype, device=d["q"].device)
        if form == "absorbed":
            return J.mla_absorbed_attention(out, kw.pop("q", d["q"]), self.cache, d["k_b"], d["v_b"], self.scale, theta, **kw)
        return J.mla_prefill_attention(out, kw.pop("q", d["q"]), self.cache, d["kv_b"], kw.pop("total", self.total()),
                                       self.scale, theta, **kw)

    def check(self, out, ref=None, what=""):
        """out [T][H][V] against the oracle; rows of no sequence must hold the 7 they were given."""
        exact, far = ref or self.attention()
        got = out.float().cpu().numpy().astype(np.float64)
        rows = sorted(t for t, _, _ in self.tokens())
        rest = sorted(set(range(self.T)) - set(rows))
        assert (got[rest] == 7).all(), f"{what}: rows of no sequence were written"
        assert np.isfinite(got[rows]).all(), f"{what}: not finite"
        far_, rms = off(got[rows], exact[rows], far[rows])
        assert far_ <= 1, f"{what}: an element is off by {far_:.3g} of what is allowed"
        assert rms <= 1, f"{what}: off by {rms:.3g} of what is allowed over all elements"
        return far_, rms
