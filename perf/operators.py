"""The latent-attention operators, measured: what a program that serves a model whose cache holds one
shared latent vector a token has the library do.

Each case is a dict of plain values; `kind` names the operator:

- append: `mla_append`, a step's or a prompt's rows normalised, rotated and stored in the paged cache;
- absorbed: `mla_absorbed_attention`, the attention of single tokens straight over the latent rows;
- expanded: `mla_prefill_attention`, a prompt's causal attention over keys and values made from them.

`seqs` sequences have between hist_lo and hist_hi positions in the cache before the call and between
new_lo and new_hi tokens in it.  Cached latents, queries and keys have unit variance per element, the
projections keep it, so scores spread as a model's do.
"""
import math
import os
import sys

import torch

own = False

_J = None


def _lib():
    global _J
    if _J is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "jero-engine_amd"))
        import jero_hip
        _J = jero_hip
    return _J


EPS, THETA = 1e-6, 10000.0
DTYPE = {"f32": torch.float32, "f16": torch.float16}
WIDE = dict(rank=512, rope=64, nope=128, v=128)
NARROW = dict(rank=128, rope=32, nope=64, v=64)


def listed():
    return [
        # a decode step of 64 sequences: one row each, from f32 projections into a 16-bit cache
        dict(name="append_step_64", kind="append", **WIDE, act="f32", kv="f16", block=16, seqs=64, hist_lo=0, hist_hi=8000,
             new_lo=1, new_hi=1, before=0),
        # three prompts' rows at once, the tail of a wider fused projection, in 16 bits
        dict(name="append_prompts", kind="append", **WIDE, act="f16", kv="f16", block=64, seqs=3, hist_lo=0, hist_hi=0,
             new_lo=2900, new_hi=8191, before=1536),
        # continued prompts of odd lengths, odd widths, into the reference's f32 cache
        dict(name="append_odd_f32", kind="append", rank=328, rope=24, nope=64, v=64, act="f32", kv="f32", block=16, seqs=5,
             hist_lo=3, hist_hi=700, new_lo=1, new_hi=901, before=8),
        # the start of a chat with a small model: one token, 77 positions, where latency counts
        dict(name="absorbed_short", kind="absorbed", **NARROW, heads=8, act="f32", kv="f16", block=16, seqs=1, hist_lo=76,
             hist_hi=76, new_lo=1, new_hi=1),
        # a serving step: 32 sequences of mixed lengths, pages of 16
        dict(name="absorbed_batch_32", kind="absorbed", **WIDE, heads=32, act="f32", kv="f16", block=16, seqs=32, hist_lo=900,
             hist_hi=6000, new_lo=1, new_hi=1),
        # one token of a large model at the end of the longest context
        dict(name="absorbed_long", kind="absorbed", **WIDE, heads=128, act="f32", kv="f16", block=64, seqs=1, hist_lo=131071,
             hist_hi=131071, new_lo=1, new_hi=1),
        # the large model's serving step with 16-bit activations
        dict(name="absorbed_f16_64", kind="absorbed", **WIDE, heads=128, act="f16", kv="f16", block=64, seqs=64, hist_lo=100,
             hist_hi=4100, new_lo=1, new_hi=1),
        # four drafted tokens a sequence checked at once, over the f32 cache
        dict(name="absorbed_draft_f32", kind="absorbed", **WIDE, heads=20, act="f32", kv="f32", block=16, seqs=7, hist_lo=40,
             hist_hi=2500, new_lo=2, new_hi=4),
        # a short prompt of the small model
        dict(name="expanded_short", kind="expanded", **NARROW, heads=8, act="f32", kv="f32", block=16, seqs=1, hist_lo=0,
             hist_hi=0, new_lo=31, new_hi=31),
        # a prompt with f32 activations, as the library's own decode path has them
        dict(name="expanded_prompt", kind="expanded", **WIDE, heads=32, act="f32", kv="f16", block=64, seqs=1, hist_lo=0,
             hist_hi=0, new_lo=2048, new_hi=2048),
        # a long prompt of the large model in 16 bits
        dict(name="expanded_f16_4097", kind="expanded", **WIDE, heads=128, act="f16", kv="f16", block=64, seqs=1, hist_lo=0,
             hist_hi=0, new_lo=4097, new_hi=4097),
        # chunks of six prompts, each with a history of its own
        dict(name="expanded_chunks", kind="expanded", **WIDE, heads=20, act="f32", kv="f16", block=16, seqs=6, hist_lo=0,
             hist_hi=1500, new_lo=17, new_hi=600),
    ]


def _between(rng, lo, hi, step=1):
    """A multiple of `step` from [lo, hi], spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step))


def draw(rng):
    kind = rng.choice(["append", "absorbed", "absorbed", "expanded"])
    case = dict(kind=kind)
    form = rng.random()
    if form < 0.5:
        case.update(WIDE)
    elif form < 0.7:
        case.update(NARROW)
    else:
        case.update(rank=_between(rng, 64, 512, 8), rope=rng.choice([16, 24, 32, 64]), nope=_between(rng, 32, 128, 8),
                    v=_between(rng, 32, 128, 8))
    case["act"], case["kv"] = rng.choice([("f32", "f16"), ("f32", "f16"), ("f16", "f16"), ("f32", "f32")])
    case["block"] = rng.choice([16, 32, 64, 256])
    if kind == "append":
        case["seqs"] = _between(rng, 1, 64)
        case["hist_lo"], case["hist_hi"] = 0, rng.choice([0, _between(rng, 10, 2000)])
        case["new_hi"] = 1 if rng.random() < 0.4 else _between(rng, 2, 16000 // case["seqs"])
        case["new_lo"] = rng.randint(1, case["new_hi"])
        case["before"] = rng.choice([0, 0, 8, 1536])
        return case
    case["heads"] = rng.choice([1, 3, 8, 20, 32, 40, 64, 128])
    if kind == "absorbed":
        case["seqs"] = _between(rng, 1, 64)
        longest = min(100000, 400000 // case["seqs"], 6000000 // (case["seqs"] * case["heads"]))
        case["hist_hi"] = _between(rng, 1, longest)
        case["hist_lo"] = rng.randint(0, case["hist_hi"])
        case["new_hi"] = rng.choice([1, 1, 1, 2, 4])
        case["new_lo"] = rng.randint(1, case["new_hi"])
        return case
    case["seqs"] = _between(rng, 1, 8)
    case["new_hi"] = _between(rng, 2, 2048 // case["seqs"])
    case["new_lo"] = rng.randint(1, case["new_hi"])
    case["hist_hi"] = rng.choice([0, _between(rng, 1, 2048 // case["seqs"])])
    case["hist_lo"] = rng.randint(0, case["hist_hi"])
    return case


def _spread(n, lo, hi, mul):
    """n lengths from lo to hi, both ends among them, in a mixed order."""
    if n == 1:
        return [hi]
    return [lo + (hi - lo) * ((i * mul + 1) % n) // (n - 1) for i in range(n)]


def _lengths(case):
    n = case["seqs"]
    return _spread(n, case["new_lo"], case["new_hi"], 5 if n % 5 else 7), \
        _spread(n, case["hist_lo"], case["hist_hi"], 3 if n % 3 else 11)


def _size(name):
    return 4 if name == "f32" else 2


def work(case):
    new, hist = _lengths(case)
    tokens, total = sum(new), sum(new) + sum(hist)
    R, P = case["rank"], case["rope"]
    a, c = _size(case["act"]), _size(case["kv"])
    if case["kind"] == "append":
        return {"bytes": tokens * (R + P) * (a + c) + 4 * R, "flops": tokens * (4 * R + 6 * (P // 2))}
    H, N, V = case["heads"], case["nope"], case["v"]
    data = total * (R + P) * c + tokens * H * (N + P + V) * a + 2 * H * R * (N + V)
    pairs = sum(n * h + n * (n + 1) // 2 for n, h in zip(new, hist))
    if case["kind"] == "absorbed":
        return {"bytes": data, "flops": 2 * H * (pairs * (2 * R + P) + tokens * R * (N + V))}
    return {"bytes": data, "flops": 2 * H * (pairs * (N + P + V) + total * R * (N + V))}


# ------------------------------------------------------------------ inputs


def _normal(g, shape, dtype, gain=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * gain).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)
    new, hist = _lengths(case)
    lens = [n + h for n, h in zip(new, hist)]
    R, P, bs = case["rank"], case["rope"], case["block"]
    act, kv = DTYPE[case["act"]], DTYPE[case["kv"]]
    tokens = sum(new)
    # the pool: every sequence's blocks, in a random order, and a few that belong to others
    need = [-(-n // bs) for n in lens]
    n_blocks = sum(need) + 3
    order = torch.randperm(n_blocks, generator=g, device="cuda").int()
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    s = dict(case=case, table=table, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), max_len=max(lens),
             total_len=sum(lens), max_new=max(new), tokens=tokens, scale=1.0 / math.sqrt(case["nope"] + P))
    s["rows"] = _normal(g, (n_blocks, bs, R + P), kv)
    # one token a sequence, or the tokens of each from starts[i] to starts[i + 1]
    one = case["kind"] != "expanded" and max(new) == 1
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s["starts"] = None if one else torch.tensor(starts, dtype=torch.int32, device="cuda")
    if case["kind"] == "append":
        x = _normal(g, (tokens, case["before"] + R + P), act, 1.7)
        s["x"] = x[:, case["before"]:]
        s["norm"] = 1.0 + 0.1 * torch.randn(R, generator=g, device="cuda")
        return s
    H, N, V = case["heads"], case["nope"], case["v"]
    s["q"] = _normal(g, (tokens, H, N + P), act, 1.5)
    k = _normal(g, (H, N, R), torch.float16, R ** -0.5)
    v = _normal(g, (H, V, R), torch.float16, R ** -0.5)
    if case["kind"] == "absorbed":
        s["k_b"], s["v_b"] = k.transpose(1, 2).contiguous(), v
    else:
        s["kv_b"] = torch.cat([k, v], 1)
    return s


# ------------------------------------------------------------------ the plain forms


def _tokens(s):
    """(sequence, place in it, position) of each token, and each sequence's token count."""
    dev = s["lens"].device
    t = torch.arange(s["tokens"], device=dev)
    lens = s["lens"].long()
    if s["starts"] is None:
        return t, torch.zeros_like(t), lens - 1, torch.ones_like(lens)
    starts = s["starts"].long()
    seq = torch.bucketize(t, starts[1:], right=True)
    n = starts[1:] - starts[:-1]
    place = t - starts[seq]
    return seq, place, lens[seq] - n[seq] + place, n


def _rotate(x, pos, P):
    """x [..., P] (f32), one position per leading row: pairs (2i, 2i + 1) turned by pos * theta^(-2i/P)."""
    i = torch.arange(P // 2, dtype=torch.float64, device=x.device)
    angle = pos.double()[:, None] * THETA ** (-2.0 * i / P)
    c, n = angle.cos().float(), angle.sin().float()
    while c.dim() < x.dim():
        c, n = c.unsqueeze(1), n.unsqueeze(1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * n, a * n + b * c], -1).flatten(-2)


def _gathered(s):
    """The sequences' cache rows in f32, [seqs][max_len][R + P], with zeros past each length."""
    bs = s["case"]["block"]
    t = torch.arange(s["max_len"], device="cuda")
    rows = s["rows"].flatten(0, 1)
    live = t[None, :] < s["lens"][:, None]
    at = s["table"].long().clamp(min=0)[:, t // bs] * bs + t % bs
    return torch.where(live[:, :, None], rows[at].float(), 0.0)


def _softmax(scores, pos_padded):
    """Rows of softmax over positions up to each query's own; scores [B][n][H][L], pos_padded [B][n]."""
    t = torch.arange(scores.shape[-1], device=scores.device)
    hidden = t[None, None, None, :] > pos_padded[:, :, None, None]
    scores = scores.masked_fill_(hidden, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _plain(s):
    case = s["case"]
    R, P = case["rank"], case["rope"]
    seq, place, pos, n = _tokens(s)
    if case["kind"] == "append":
        x = s["x"].float()
        c = x[:, :R]
        c = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS) * s["norm"]
        row = torch.cat([c, _rotate(x[:, R:], pos, P)], 1)
        bs = case["block"]
        s["rows"][s["table"].long()[seq, pos // bs], pos % bs] = row.to(s["rows"].dtype)
        return s["rows"]
    H, N, V = case["heads"], case["nope"], case["v"]
    B, m = case["seqs"], s["max_new"]
    rows = _gathered(s)
    q = s["q"].float()
    q = torch.cat([q[..., :N], _rotate(q[..., N:], pos, P)], -1)
    # queries by sequence, [B][m][H][N + P]; a short sequence's spare places see the first position
    qp = torch.zeros((B, m, H, N + P), device="cuda")
    qp[seq, place] = q
    pp = torch.zeros((B, m), dtype=torch.long, device="cuda")
    pp[seq, place] = pos
    if case["kind"] == "absorbed":
        k_b, v_b = s["k_b"].float(), s["v_b"].float()  # [H][R][N], [H][V][R]
        qn = qp[..., :N].permute(2, 0, 1, 3).reshape(H, B * m, N).contiguous()
        qa = torch.bmm(qn, k_b.transpose(1, 2).contiguous()).reshape(H, B, m, R).permute(1, 2, 0, 3)
        qa = torch.cat([qa, qp[..., N:]], -1).reshape(B, m * H, R + P)
        scores = torch.bmm(qa, rows.transpose(1, 2).contiguous()).mul_(s["scale"]).view(B, m, H, -1)
        p = _softmax(scores, pp).view(B, m * H, -1)
        o = torch.bmm(p, rows[..., :R].contiguous()).view(B, m, H, R)[seq, place]  # [T][H][R]
        out = torch.bmm(o.transpose(0, 1).contiguous(), v_b.transpose(1, 2).contiguous()).transpose(0, 1)
        return out.to(s["q"].dtype).contiguous()
    kv = rows[..., :R].reshape(-1, R) @ s["kv_b"].float().reshape(H * (N + V), R).t().contiguous()
    kv = kv.view(B, -1, H, N + V).transpose(1, 2)  # [B][H][L][N + V]
    k = torch.cat([kv[..., :N], rows[:, None, :, R:].expand(-1, H, -1, -1)], -1)
    k = k.transpose(2, 3).contiguous().view(B * H, N + P, -1)
    scores = torch.bmm(qp.transpose(1, 2).reshape(B * H, m, N + P).contiguous(), k).mul_(s["scale"])
    p = _softmax(scores.view(B, H, m, -1).transpose(1, 2), pp).transpose(1, 2).reshape(B * H, m, -1)
    out = torch.bmm(p.contiguous(), kv[..., N:].reshape(B * H, -1, V).contiguous())
    return out.view(B, H, m, V).transpose(1, 2)[seq, place].to(s["q"].dtype).contiguous()


def _kernels(s):
    J, case = _lib(), s["case"]
    cache = J.LatentCache(s["rows"], s["table"], s["lens"], case["rank"], starts=s["starts"], max_len=s["max_len"])
    if case["kind"] == "append":
        J.mla_append(cache, s["x"], s["norm"], EPS, THETA)
        return s["rows"]
    out = torch.empty((s["tokens"], case["heads"], case["v"]), dtype=s["q"].dtype, device=s["q"].device)
    if case["kind"] == "absorbed":
        return J.mla_absorbed_attention(out, s["q"], cache, s["k_b"], s["v_b"], s["scale"], THETA)
    return J.mla_prefill_attention(out, s["q"], cache, s["kv_b"], s["total_len"], s["scale"], THETA)


def run(state):
    return _kernels(state) if own else _plain(state)


# ------------------------------------------------------------------ 64 bits


def exact(case, seed):
    """From the definition, a sequence and a head at a time in 64 bits: the absorbed cases in the expanded form."""
    s = prepare(case, seed)
    new, hist = _lengths(case)
    R, P, bs = case["rank"], case["rope"], case["block"]

    def turned(x, first):  # x [n][...][P] at positions first, first + 1, ...
        z = torch.view_as_complex(x.reshape(*x.shape[:-1], P // 2, 2).contiguous())
        f = THETA ** (-torch.arange(0, P, 2, dtype=torch.float64, device=x.device) / P)
        ph = torch.arange(first, first + x.shape[0], dtype=torch.float64, device=x.device)[:, None] * f
        w = torch.polar(torch.ones_like(ph), ph)
        return torch.view_as_real(z * w.view(x.shape[0], *([1] * (x.dim() - 2)), P // 2)).flatten(-2)

    if case["kind"] == "append":
        rows = s["rows"].double()
    else:
        H, N, V = case["heads"], case["nope"], case["v"]
        out = torch.zeros((sum(new), H, V), dtype=torch.float64, device="cuda")
    at = 0
    for i, (n, h) in enumerate(zip(new, hist)):
        blocks = s["table"][i, :-(-(n + h) // bs)].long()
        if case["kind"] == "append":
            x = s["x"][at:at + n].double()
            c = x[:, :R] / torch.sqrt(x[:, :R].pow(2).sum(1, keepdim=True) / R + EPS) * s["norm"].double()
            p = torch.arange(h, h + n, device="cuda")
            rows[blocks[p // bs], p % bs] = torch.cat([c, turned(x[:, R:], h)], 1)
        else:
            c = s["rows"][blocks].reshape(-1, R + P)[:n + h].double()
            q = s["q"][at:at + n].double()
            qr = turned(q[..., N:], h)
            later = torch.arange(n + h, device="cuda")[None, :] > torch.arange(h, h + n, device="cuda")[:, None]
            for j in range(H):
                wk = s["k_b"][j].double() if "k_b" in s else s["kv_b"][j, :N].double().t()
                wv = s["v_b"][j].double() if "v_b" in s else s["kv_b"][j, N:].double()
                a = (q[:, j, :N] @ (c[:, :R] @ wk).t() + qr[:, j] @ c[:, R:].t()) * s["scale"]
                out[at:at + n, j] = torch.softmax(a.masked_fill(later, -math.inf), 1) @ (c[:, :R] @ wv.t())
        at += n
    return rows if case["kind"] == "append" else out
