"""The operators of a serving step over a paged key/value cache, measured: what a program that serves many
requests of a model with grouped-query attention has the library do, step after step.

Each case is a dict of plain values; `kind` names the operator:

- extend: `paged_extend`, the requests' block tables, lengths and their tokens' positions and slots, made on the
  GPU from how many tokens each request gets;
- append: `paged_append`, the tokens' queries and keys rotated to their positions, keys and values stored;
- attend: `paged_attention`, the attention of a batch whose sequences share their first `shared` positions;
- verify: `verify_drafts`, drafted tokens accepted or replaced by given random numbers.

`seqs` sequences have between hist_lo and hist_hi positions in the cache before the call (in `attend`: behind the
shared ones) and between new_lo and new_hi tokens in it.
"""
import functools
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


EPS = 1e-6
DTYPE = {"f32": torch.float32, "f16": torch.float16}


def listed():
    return [
        # a decode step of 64 requests: one token each, four of them on a new block
        dict(name="extend_step_64", kind="extend", seqs=64, block=16, cols=512, hist_lo=1, hist_hi=8000, new_lo=1, new_hi=1,
             ends=0, drop=0, free=4096),
        # the mixed step of a large server: prompts beside single tokens, requests that end, drafts taken back
        dict(name="extend_mixed_1500", kind="extend", seqs=1500, block=64, cols=160, hist_lo=0, hist_hi=8000, new_lo=1,
             new_hi=401, ends=97, drop=3, free=9000),
        # a decode step of 64 sequences of the 8B shape, from f32 projections: norms of queries and keys, a scaled context
        dict(name="append_step_64", kind="append", tokens=64, heads=32, kv_heads=8, dim=128, rot=128, layout="half",
             scaling="yarn", theta=1e6, factor=4.0, original=32768, far=131072, norm=True, act="f32", kv="f16", block=16,
             before=0),
        # prompts' rows in 16 bits, parts of one fused projection's output
        dict(name="append_prompts_f16", kind="append", tokens=12001, heads=32, kv_heads=8, dim=128, rot=128, layout="half",
             scaling="wavelength", theta=5e5, factor=8.0, original=8192, far=16000, norm=False, act="f16", kv="f16",
             block=64, before=0),
        # odd widths: pairs side by side in part of the head, positions far out, the reference's f32 cache
        dict(name="append_part_f32", kind="append", tokens=901, heads=20, kv_heads=4, dim=80, rot=24, layout="interleaved",
             scaling="linear", theta=1e4, factor=16.0, original=4096, far=1000000, norm=True, act="f32", kv="f32", block=16,
             before=8),
        # two chats on a short system prompt, where latency counts
        dict(name="attend_two_short", kind="attend", seqs=2, shared=64, hist_lo=3, hist_hi=40, new_lo=1, new_hi=1, heads=32,
             kv_heads=8, dim=128, act="f32", kv="f16", block=16),
        # a serving step of the 8B shape: 64 chats behind one long instruction
        dict(name="attend_step_64", kind="attend", seqs=64, shared=8192, hist_lo=30, hist_hi=1500, new_lo=1, new_hi=1,
             heads=32, kv_heads=8, dim=128, act="f32", kv="f16", block=16),
        # a large batch that answers questions about one document, 16-bit activations
        dict(name="attend_step_f16_256", kind="attend", seqs=256, shared=32768, hist_lo=10, hist_hi=700, new_lo=1, new_hi=1,
             heads=64, kv_heads=8, dim=128, act="f16", kv="f16", block=64),
        # drafted tokens over the f32 cache, odd group of heads
        dict(name="attend_drafts_f32", kind="attend", seqs=7, shared=2048, hist_lo=3, hist_hi=900, new_lo=2, new_hi=5,
             heads=20, kv_heads=4, dim=64, act="f32", kv="f32", block=32),
        # chunks of nine prompts behind a shared one
        dict(name="attend_chunks_f16", kind="attend", seqs=9, shared=4096, hist_lo=0, hist_hi=900, new_lo=17, new_hi=1500,
             heads=32, kv_heads=4, dim=128, act="f16", kv="f16", block=64),
        # one chat with three drafted tokens that come with no probabilities (looked up in its own text)
        dict(name="verify_looked_up", kind="verify", seqs=1, new_lo=4, new_hi=4, vocab=32000, draft=False, near=2.0),
        # 64 chats with up to four drafted tokens of a small model
        dict(name="verify_64", kind="verify", seqs=64, new_lo=1, new_hi=5, vocab=151936, draft=True, near=0.7),
    ]


def _between(rng, lo, hi, step=1):
    """A multiple of `step` from [lo, hi], spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step))


def draw(rng):
    kind = rng.choice(["extend", "append", "append", "attend", "attend", "attend", "verify"])
    case = dict(kind=kind)
    if kind == "extend":
        case.update(seqs=_between(rng, 1, 2000), block=rng.choice([4, 16, 32, 64, 256]), drop=rng.choice([0, 0, 4]))
        case["cols"] = max(8, 8192 // case["block"])
        case["hist_hi"] = _between(rng, 1, case["cols"] * case["block"] - 600)
        case["hist_lo"] = rng.randint(0, case["hist_hi"])
        case["new_hi"] = rng.choice([1, _between(rng, 1, 500)])
        case["new_lo"] = rng.randint(0, case["new_hi"])
        case["ends"] = rng.randint(0, case["seqs"] // 8)
        # (at times fewer free blocks than asked for)
        case["free"] = _between(rng, 1, 2 + case["seqs"] * (2 + 2 * case["new_hi"] // case["block"]))
        return case
    case["act"], case["kv"] = rng.choice([("f32", "f16"), ("f32", "f16"), ("f16", "f16"), ("f32", "f32")])
    case["block"] = rng.choice([16, 32, 64, 256])
    if kind == "append":
        case["kv_heads"] = rng.choice([1, 2, 4, 8])
        case["heads"] = case["kv_heads"] * rng.choice([1, 2, 4, 5, 8])
        case["dim"] = rng.choice([64, 80, 128, 128, 256])
        case["tokens"] = _between(rng, 1, min(8000, 30000000 // (case["dim"] * (case["heads"] + case["kv_heads"]))))
        case["rot"] = case["dim"] if rng.random() < 0.5 else _between(rng, 8, case["dim"], 8)
        case["layout"] = rng.choice(["half", "interleaved"])
        case["scaling"] = rng.choice(["none", "linear", "ntk", "yarn", "wavelength"])
        case["theta"] = rng.choice([1e4, 5e5, 1e6])
        case["factor"] = rng.choice([2.0, 4.0, 8.0])
        case["original"] = rng.choice([4096, 8192, 32768])
        case["far"] = _between(rng, 8, 2000000)
        case["norm"] = rng.random() < 0.5
        case["before"] = rng.choice([0, 0, 8, 1024])
        return case
    if kind == "verify":
        case["seqs"] = _between(rng, 1, 64)
        case["new_hi"] = rng.randint(1, 6)
        case["new_lo"] = rng.randint(1, case["new_hi"])
        case["vocab"] = _between(rng, 50, 151936)
        case["draft"] = rng.random() < 0.7
        case["near"] = rng.choice([0.3, 0.7, 1.5])
        return case
    case["dim"] = rng.choice([64, 80, 96, 128, 128, 128, 256])
    case["kv_heads"] = rng.choice([1, 2, 4, 8])
    case["heads"] = case["kv_heads"] * rng.choice([1, 2, 4, 5, 8])
    case["seqs"] = _between(rng, 1, 128)
    case["new_hi"] = rng.choice([1, 1, 1, 4, _between(rng, 2, 2048 // case["seqs"])])
    case["new_lo"] = rng.randint(1, case["new_hi"])
    tokens = case["seqs"] * case["new_hi"]
    pairs = 200000000 // (case["heads"] * tokens) * 128 // case["dim"]  # positions a token, at most
    case["shared"] = 0 if rng.random() < 0.2 else _between(rng, case["block"], max(case["block"], min(32768, pairs // 2)),
                                                         case["block"])
    case["shared"] = case["shared"] // case["block"] * case["block"]
    rows = 60000000 // (case["kv_heads"] * case["dim"])
    case["hist_hi"] = _between(rng, 1, max(2, min(4000, pairs // 4, rows // case["seqs"])))
    case["hist_lo"] = rng.randint(0, case["hist_hi"])
    return case


def _spread(n, lo, hi, mul):
    """n lengths from lo to hi, both ends among them, in a mixed order."""
    if n == 1:
        return [hi]
    return [lo + (hi - lo) * ((i * mul + 1) % n) // (n - 1) for i in range(n)]


def _lengths(case):
    n = case["seqs"]
    new = _spread(n, case["new_lo"], case["new_hi"], 5 if n % 5 else 7)
    hist = _spread(n, case.get("hist_lo", 0), case.get("hist_hi", 0), 3 if n % 3 else 11)
    if case["kind"] == "extend":  # the requests that end, spread over the batch
        for i in range(case["ends"]):
            new[i * n // case["ends"]] = -1
    return new, hist


def _size(name):
    return 4 if name == "f32" else 2


def work(case):
    if case["kind"] == "append":
        q, k, D = case["tokens"] * case["heads"], case["tokens"] * case["kv_heads"], case["dim"]
        a, c = _size(case["act"]), _size(case["kv"])
        flops = (q + k) * (3 * case["rot"] + (4 * D if case["norm"] else 0))
        return {"bytes": q * D * 2 * a + 2 * k * D * (a + c) + case["tokens"] * 12, "flops": flops}
    new, hist = _lengths(case)
    n = len(new)
    if case["kind"] == "extend":
        tokens, bs = sum(max(x, 0) for x in new), case["block"]
        fresh = sum(-(-(h + x) // bs) - -(-h // bs) for x, h in zip(new, hist) if x > 0)
        pages = sum(-(-x // bs) for x in new if x > 0)
        back = sum(-(-h // bs) for x, h in zip(new, hist) if x < 0)
        return {"bytes": 24 * n + 12 * tokens + 4 * pages + 8 * (fresh + back), "flops": 8 * (n + tokens)}
    if case["kind"] == "verify":  # a sequence's last row of the target's and of the draft's probabilities
        V = case["vocab"]
        return {"bytes": n * V * 4 * (2 if case["draft"] else 1), "flops": n * V * 3}
    H, KV, D, P = case["heads"], case["kv_heads"], case["dim"], case["shared"]
    tokens = sum(new)
    pairs = sum(x * (P + h) + x * (x + 1) // 2 for x, h in zip(new, hist))
    rows = P + sum(new) + sum(hist)
    return {"bytes": rows * KV * D * 2 * _size(case["kv"]) + tokens * H * D * 2 * _size(case["act"]),
            "flops": 4 * H * D * pairs}


# ------------------------------------------------------------------ inputs


def _normal(g, shape, dtype, gain=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * gain).to(dtype)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _starts(new):
    at = [0]
    for x in new:
        at.append(at[-1] + max(x, 0))
    return at


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)
    s = dict(case=case)
    make = dict(extend=_prepare_extend, append=_prepare_append, attend=_prepare_attend, verify=_prepare_verify)
    make[case["kind"]](s, case, g)
    return s


def _prepare_extend(s, case, g):
    """Requests between steps: a table of the blocks they hold, their lengths, and the stack of the free ones."""
    new, hist = _lengths(case)
    n, bs, cols = case["seqs"], case["block"], case["cols"]
    n_blocks = sum(-(-(h + 6) // bs) for h in hist) + case["free"]  # those in neither table nor stack are others'
    # lengths of another seed are others; a draft's rejected tokens stand at the end of a length
    hist = torch.tensor(hist, device="cuda")
    lens = (hist + torch.randint(0, 7, (n,), generator=g, device="cuda")).clamp(min=0).int()
    s["drop"] = None
    if case["drop"]:
        s["drop"] = torch.minimum(torch.randint(0, case["drop"] + 1, (n,), generator=g, device="cuda").int(), lens)
    owned = (lens + bs - 1) // bs
    held = int(owned.sum())
    ids = torch.randperm(n_blocks, generator=g, device="cuda").int()
    c = torch.arange(cols, device="cuda")
    mine = c[None, :] < owned[:, None]
    table = torch.full((n, cols), -1, dtype=torch.int32, device="cuda")
    table[mine] = ids[:held]
    s["free"] = torch.full((n_blocks,), -1, dtype=torch.int32, device="cuda")
    s["free"][:case["free"]] = ids[held:held + case["free"]]
    s["n_free"] = _i32([case["free"]])
    s["table"], s["lens"], s["owned"] = table, lens, owned.int()
    s["new"] = _i32(new)
    s["tokens"] = _starts(new)[-1] + 5  # a step's buffers hold a few rows more than its tokens
    s["n_blocks"] = n_blocks


def _prepare_append(s, case, g):
    T, H, KV, D = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    act, kv, bs = DTYPE[case["act"]], DTYPE[case["kv"]], case["block"]
    # queries, keys and values are parts of one projection's row
    x = _normal(g, (T, case["before"] + (H + 2 * KV) * D), act, 1.7)[:, case["before"]:]
    s["q"] = x[:, :H * D].unflatten(1, (H, D))
    s["k"] = x[:, H * D:(H + KV) * D].unflatten(1, (KV, D))
    s["v"] = x[:, (H + KV) * D:].unflatten(1, (KV, D))
    blocks = -(-T // bs) + 2
    s["k_rows"] = _normal(g, (blocks, bs, KV, D), kv)
    s["v_rows"] = _normal(g, (blocks, bs, KV, D), kv)
    s["positions"] = torch.randint(0, case["far"], (T,), generator=g, device="cuda").int()
    # runs of a block's slots, blocks in a random order
    order = torch.randperm(blocks, generator=g, device="cuda")
    t = torch.arange(T, device="cuda")
    s["slots"] = order[t // bs] * bs + t % bs
    s["q_norm"] = s["k_norm"] = None
    if case["norm"]:
        s["q_norm"] = 1.0 + 0.1 * torch.randn(D, generator=g, device="cuda")
        s["k_norm"] = 1.0 + 0.1 * torch.randn(D, generator=g, device="cuda")


def _prepare_attend(s, case, g):
    new, hist = _lengths(case)
    P, bs = case["shared"], case["block"]
    lens = [P + h + x for h, x in zip(hist, new)]
    need = [-(-n // bs) - P // bs for n in lens]
    n_blocks = P // bs + sum(need) + 3
    order = torch.randperm(n_blocks, generator=g, device="cuda").int()
    table = torch.full((len(lens), P // bs + max(need)), -1, dtype=torch.int32, device="cuda")
    s["prefix"] = order[:P // bs].contiguous()
    table[:, :P // bs] = s["prefix"]
    c = torch.arange(max(need), device="cuda")
    mine = c[None, :] < _i32(need)[:, None]
    tail = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device="cuda")
    tail[mine] = order[P // bs:P // bs + sum(need)]
    table[:, P // bs:] = tail
    s["table"], s["lens"] = table, _i32(lens)
    s["starts"] = None if max(new) == 1 else _i32(_starts(new))
    s["tokens"], s["max_new"], s["max_len"], s["max_own"] = sum(new), max(new), max(lens), max(lens) - P
    shape = (n_blocks, bs, case["kv_heads"], case["dim"])
    s["k_rows"], s["v_rows"] = (_normal(g, shape, DTYPE[case["kv"]]) for _ in range(2))
    s["q"] = _normal(g, (s["tokens"], case["heads"], case["dim"]), DTYPE[case["act"]], 1.5)
    s["scale"] = case["dim"] ** -0.5


def _prepare_verify(s, case, g):
    """The step's tokens (a sequence's last one, then its drafts) and what target and draft give for the next."""
    new, _ = _lengths(case)
    V, T, n = case["vocab"], sum(new), case["seqs"]
    s["starts"] = _i32(_starts(new))
    s["tokens"] = torch.randint(0, V, (T,), generator=g, device="cuda").int()
    logits = torch.randn((T, V), generator=g, device="cuda") * 2.5
    s["target"] = torch.softmax(logits, 1)
    # the row before each drafted token
    first = torch.zeros(T, dtype=torch.bool, device="cuda")
    first[s["starts"][:-1].long()] = True
    at = (~first).nonzero()[:, 0]
    near = logits[at - 1] + case["near"] * torch.randn((T - n, V), generator=g, device="cuda")
    gumbel = -torch.log(-torch.log(torch.rand((T - n, V), generator=g, device="cuda").clamp(1e-20, 1 - 1e-7)))
    s["tokens"][at] = (near + gumbel).argmax(1).int()
    s["draft"] = torch.softmax(near, 1) if case["draft"] else None
    s["u"] = torch.rand(T - n, generator=g, device="cuda")
    s["u_last"] = torch.rand(n, generator=g, device="cuda")
    s["max_new"] = max(new)


# ------------------------------------------------------------------ the plain forms


def _plain_extend(s):
    bs, cols = s["case"]["block"], s["case"]["cols"]
    new, n = s["new"].long(), s["new"].numel()
    lens = s["lens"].long() - (0 if s["drop"] is None else s["drop"].long())
    owned = s["owned"].long()
    tokens = new.clamp(min=0)
    starts = torch.cat([tokens.new_zeros(1), tokens.cumsum(0)])
    # the blocks of the requests that end go onto the stack
    col = torch.arange(cols, device="cuda")
    gone = (new < 0)[:, None] & (col[None, :] < owned[:, None])
    place = s["n_free"].long() + gone.flatten().cumsum(0) - 1
    free = s["free"].clone()
    size = free.numel()
    free = torch.cat([free, free.new_zeros(1)])
    free[torch.where(gone.flatten(), place, size)] = s["table"].flatten()
    free = free[:size]
    top = s["n_free"].long() + gone.sum()
    # requests in order get what they need as long as the stack holds it
    need = torch.where(new > 0, (-(-(lens + tokens) // bs) - owned).clamp(min=0), 0)
    fits = lens + tokens <= cols * bs
    need = torch.where(fits, need, 0)
    taken = need.cumsum(0)
    granted = fits & ((need == 0) | (taken <= top))
    # (the sums are of what was asked for: behind a refused request all that need blocks are refused)
    got = torch.where(granted, need, 0)
    before = taken - need
    fresh = (col[None, :] >= owned[:, None]) & (col[None, :] < (owned + got)[:, None])
    index = (top - 1 - before[:, None] - (col[None, :] - owned[:, None])).clamp(0, size - 1)
    table = torch.where(fresh, free[index], s["table"])
    n_free = top - got.sum()
    ends = new < 0
    lens_out = torch.where(ends, 0, torch.where(granted, lens + tokens, lens))
    owned_out = torch.where(ends, 0, owned + got)
    # the tokens
    t = torch.arange(s["tokens"], device="cuda")
    seq = torch.bucketize(t, starts[1:], right=True).clamp(max=n - 1)
    live = (t < starts[-1]) & granted[seq]
    pos = torch.where(live, lens[seq] + t - starts[seq], -1)
    block = table[seq, (pos // bs).clamp(0, cols - 1)].long()
    slots = torch.where(live, block * bs + pos % bs, -1)
    s["table"].copy_(table)
    s["free"].copy_(free)
    return dict(table=s["table"], free=s["free"], lens=lens_out.int(), owned=owned_out.int(), n_free=n_free.int().reshape(1),
                starts=starts.int(), granted=granted.int(), positions=pos.int(), slots=slots)


def _turns(case):
    """Turns a position of each pair, in 64 bits, and what cosine and sine are multiplied with."""
    R, theta, factor, orig = case["rot"], case["theta"], case["factor"], case["original"]
    kind = case["scaling"]
    i = torch.arange(R // 2, dtype=torch.float64, device="cuda")
    if kind == "ntk":
        theta = theta * factor ** (R / (R - 2))
    f = theta ** (-2.0 * i / R)
    if kind == "linear":
        f = f / factor
    if kind == "yarn":
        # pairs that turn more than 32 times over the original length are kept, those below once stretched
        edge = [R * math.log(orig / (2 * math.pi * turns)) / (2 * math.log(theta)) for turns in (32.0, 1.0)]
        low, high = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), R - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        f = f / factor * ramp + f * (1 - ramp)
    if kind == "wavelength":
        ramp = ((orig * f / (2 * math.pi) - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        f = (1 - ramp) * f / factor + ramp * f
    return f / (2 * math.pi), 0.1 * math.log(factor) + 1.0 if kind == "yarn" else 1.0


def _plain_rotated(x, norm, case, positions):
    x, R = x.float(), case["rot"]
    if norm is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * norm
    f, m = _turns(case)
    angle = 2 * math.pi * torch.frac(positions.double()[:, None, None] * f)
    c, n = (angle.cos() * m).float(), (angle.sin() * m).float()
    if case["layout"] == "half":
        a, b = x[..., :R // 2], x[..., R // 2:R]
        return torch.cat([a * c - b * n, a * n + b * c, x[..., R:]], -1)
    a, b = x[..., 0:R:2], x[..., 1:R:2]
    return torch.cat([torch.stack([a * c - b * n, a * n + b * c], -1).flatten(-2), x[..., R:]], -1)


def _plain_append(s):
    case = s["case"]
    q = _plain_rotated(s["q"], s["q_norm"], case, s["positions"]).to(s["q"].dtype)
    k = _plain_rotated(s["k"], s["k_norm"], case, s["positions"])
    s["k_rows"].flatten(0, 1)[s["slots"]] = k.to(s["k_rows"].dtype)
    s["v_rows"].flatten(0, 1)[s["slots"]] = s["v"].to(s["v_rows"].dtype)
    return q, s["k_rows"], s["v_rows"]


def _places(s):
    """(sequence, place in it, position) of each token."""
    t = torch.arange(s["tokens"], device="cuda")
    lens = s["lens"].long()
    if s["starts"] is None:
        return t, torch.zeros_like(t), lens - 1
    starts = s["starts"].long()
    seq = torch.bucketize(t, starts[1:], right=True)
    place = t - starts[seq]
    return seq, place, lens[seq] - (starts[seq + 1] - starts[seq]) + place


def _plain_attend(s):
    case = s["case"]
    H, KV, D, P, bs = case["heads"], case["kv_heads"], case["dim"], case["shared"], case["block"]
    G, B, m, T = H // KV, case["seqs"], s["max_new"], s["tokens"]
    seq, place, pos = _places(s)
    q = s["q"].float().view(T, KV, G, D) * s["scale"]
    # the shared positions: one product for all tokens' rows, [KV][T G][P]
    kp, vp = (s[n][s["prefix"].long()].float().reshape(P, KV, D).transpose(0, 1).contiguous() for n in ("k_rows", "v_rows"))
    rows = q.transpose(0, 1).reshape(KV, T * G, D)
    sp = torch.bmm(rows, kp.transpose(1, 2).contiguous())
    # each sequence's own, gathered with zeros past its length, [B KV][m G][own]
    t = torch.arange(s["max_own"], device="cuda")
    live = t[None, :] < (s["lens"] - P)[:, None]
    block = s["table"].long().clamp(min=0)[:, (P + t) // bs]
    at = block * bs + (P + t) % bs
    ko, vo = (torch.where(live[:, :, None, None], s[n].flatten(0, 1)[at].float(), 0.0).transpose(1, 2)
              .reshape(B * KV, -1, D).contiguous() for n in ("k_rows", "v_rows"))
    qo = torch.zeros((B, m, KV, G, D), device="cuda")
    qo[seq, place] = q
    upto = torch.zeros((B, m), dtype=torch.long, device="cuda")  # a short sequence's spare places see its first own one
    upto[seq, place] = pos - P
    qo = qo.permute(0, 2, 1, 3, 4).reshape(B * KV, m * G, D)
    so = torch.bmm(qo, ko.transpose(1, 2).contiguous()).view(B, KV, m, G, -1)
    so = so.masked_fill_((t > upto[:, :, None])[:, None, :, None, :], -math.inf)
    # one softmax over both
    top = so.amax(-1).permute(0, 2, 1, 3)[seq, place]  # [T][KV][G]
    if P:
        top = torch.maximum(top, sp.amax(-1).view(KV, T, G).transpose(0, 1))
    sp = sp.sub_(top.transpose(0, 1).reshape(KV, T * G, 1)).exp_()
    padded = torch.zeros((B, m, KV, G), device="cuda")
    padded[seq, place] = top
    so = so.sub_(padded.permute(0, 2, 1, 3)[..., None]).exp_()
    total = sp.sum(-1).view(KV, T, G).transpose(0, 1) + so.sum(-1).permute(0, 2, 1, 3)[seq, place]
    out = torch.bmm(sp, vp).view(KV, T, G, D).transpose(0, 1)
    out = out + torch.bmm(so.view(B * KV, m * G, -1), vo).view(B, KV, m, G, D).permute(0, 2, 1, 3, 4)[seq, place]
    return (out / total[..., None]).reshape(T, H, D).to(s["q"].dtype)


def _plain_verify(s):
    """In 64 bits: products next to the border of a test, and running sums over a vocabulary."""
    T, n, V = s["tokens"].numel(), s["starts"].numel() - 1, s["case"]["vocab"]
    starts, tokens = s["starts"].long(), s["tokens"].long()
    t = torch.arange(T, device="cuda")
    seq = torch.bucketize(t, starts[1:], right=True)
    place = t - starts[seq]
    drafted = t - seq - 1  # the draft's row that a token comes from, for those not first in their sequence
    p = s["target"][(t - 1).clamp(min=0), tokens].double()
    if s["draft"] is not None and T > n:
        u = s["u"][drafted.clamp(min=0)].double()
        good = u * s["draft"][drafted.clamp(min=0), tokens].double() < p
    else:
        good = (s["u"][drafted.clamp(0, max(T - n - 1, 0))].double() < p) if T > n else torch.ones_like(p, dtype=torch.bool)
    bad = (~good & (place > 0)).long()
    # tokens of a sequence before its first refused one
    wrong = bad.cumsum(0)
    wrong = wrong - torch.cat([wrong.new_zeros(1), wrong])[starts[seq]]
    accepted = torch.zeros(n, dtype=torch.long, device="cuda").index_add_(0, seq, ((wrong == 0) & (place > 0)).long())
    last = starts[:-1] + accepted  # the row that the next token is drawn from
    refused = last + 1 < starts[1:]
    w = s["target"][last].double()
    if T > n:
        row = (last - torch.arange(n, device="cuda")).clamp(max=T - n - 1)
        if s["draft"] is not None:
            less = s["draft"][row].double()
        else:
            less = torch.zeros_like(w).scatter_(1, tokens[(last + 1).clamp(max=T - 1)][:, None], math.inf)
        left = (w - less).clamp(min=0)
        w = torch.where((refused & (left.sum(1) > 0))[:, None], left, w)
    run = w.cumsum(1)
    drawn = (run > (s["u_last"].double() * w.sum(1))[:, None]).int().argmax(1)
    out = torch.full((T,), -1, dtype=torch.long, device="cuda")
    keep = place < accepted[seq]
    out[keep] = tokens[(t + 1).clamp(max=T - 1)][keep]
    out[last] = drawn
    return out.int(), accepted.int()


# ------------------------------------------------------------------ the framework's calls


@functools.lru_cache(maxsize=None)
def _rope(rot, layout, scaling, theta, factor, original):
    """A model's rotation, made once from its configuration."""
    return _lib().Rope(rot, theta, layout=layout, scaling=scaling, factor=factor, original=original)


def _own_extend(s):
    J = _lib()
    n, dev = s["new"].numel(), s["new"].device
    pool = J.BlockPool(s["table"], s["lens"], s["owned"], s["free"], s["n_free"], s["n_blocks"], s["case"]["block"])
    # the step's results beside the state that it starts from
    into = torch.empty(4 * n + 2, dtype=torch.int32, device=dev)
    lens, owned, starts, granted, n_free = into.split([n, n, n + 1, n, 1])
    positions = torch.empty(s["tokens"], dtype=torch.int32, device=dev)
    slots = torch.empty(s["tokens"], dtype=torch.int64, device=dev)
    J.paged_extend(pool, s["new"], positions, slots, starts, drop=s["drop"], granted=granted, into=(lens, owned, n_free))
    return dict(table=s["table"], free=s["free"], lens=lens, owned=owned, n_free=n_free, starts=starts, granted=granted,
                positions=positions, slots=slots)


def _own_append(s):
    J, c = _lib(), s["case"]
    rope = _rope(c["rot"], c["layout"], c["scaling"], c["theta"], c["factor"], c["original"])
    q = torch.empty(s["q"].shape, dtype=s["q"].dtype, device=s["q"].device)
    J.paged_append(s["k_rows"], s["v_rows"], q, s["q"], s["k"], s["v"], s["positions"], s["slots"], rope, q_norm=s["q_norm"],
                   k_norm=s["k_norm"], eps=EPS)
    return q, s["k_rows"], s["v_rows"]


def _own_attend(s):
    J = _lib()
    cache = J.PagedCache(s["k_rows"], s["v_rows"], s["table"], s["lens"], starts=s["starts"], max_len=s["max_len"],
                         shared=s["prefix"])
    return J.paged_attention(torch.empty_like(s["q"]), s["q"], cache, s["scale"])


def _own_verify(s):
    J = _lib()
    n, T, dev = s["starts"].numel() - 1, s["tokens"].numel(), s["tokens"].device
    out = torch.empty(T, dtype=torch.int32, device=dev)
    accepted = torch.empty(n, dtype=torch.int32, device=dev)
    J.verify_drafts(out, accepted, s["target"], s["draft"], s["tokens"], s["starts"], s["u"], s["u_last"])
    return out, accepted


def run(state):
    kind = state["case"]["kind"]
    if own:
        return dict(extend=_own_extend, append=_own_append, attend=_own_attend, verify=_own_verify)[kind](state)
    return dict(extend=_plain_extend, append=_plain_append, attend=_plain_attend, verify=_plain_verify)[kind](state)


# ------------------------------------------------------------------ 64 bits


def _exact_append(s, case):
    """From complex numbers: a pair is multiplied by m exp(i angle)."""
    R, theta, factor, orig = case["rot"], case["theta"], case["factor"], case["original"]
    freq, m = [], 1.0
    for i in range(R // 2):
        base = theta * factor ** (R / (R - 2.0)) if case["scaling"] == "ntk" else theta
        f = math.exp(-2.0 * i / R * math.log(base))
        if case["scaling"] == "linear":
            f /= factor
        elif case["scaling"] == "yarn":
            m = 1.0 + 0.1 * math.log(factor)
            fast, slow = (R / 2 * (math.log(orig) - math.log(2 * math.pi * b)) / math.log(theta) for b in (32, 1))
            fast, slow = max(math.floor(fast), 0), min(math.ceil(slow), R - 1)
            share = min(max((i - fast) / max(slow - fast, 1e-3), 0.0), 1.0)
            f *= (1.0 - share) + share / factor
        elif case["scaling"] == "wavelength":
            wave = 2 * math.pi / f
            if wave > orig / 1.0:
                f /= factor
            elif wave >= orig / 4.0:
                kept = (orig / wave - 1.0) / 3.0
                f *= kept + (1.0 - kept) / factor
        freq.append(f)
    angle = s["positions"].double()[:, None, None] * torch.tensor(freq, dtype=torch.float64, device="cuda")
    z = torch.polar(torch.full_like(angle, m), angle)

    def turned(x, norm):
        x = x.double()
        if norm is not None:
            x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS) * norm.double()
        y = x.clone()
        one, two = (slice(0, R // 2), slice(R // 2, R)) if case["layout"] == "half" else (slice(0, R, 2), slice(1, R, 2))
        w = torch.complex(x[..., one].contiguous(), x[..., two].contiguous()) * z
        y[..., one], y[..., two] = w.real, w.imag
        return y

    k_rows, v_rows = s["k_rows"].double(), s["v_rows"].double()
    bs = case["block"]
    k_rows[s["slots"] // bs, s["slots"] % bs] = turned(s["k"], s["k_norm"])
    v_rows[s["slots"] // bs, s["slots"] % bs] = s["v"].double()
    return turned(s["q"], s["q_norm"]), k_rows, v_rows


def _exact_attend(s, case):
    """A sequence and a group of heads at a time, over its own table's blocks."""
    new, hist = _lengths(case)
    G, bs = case["heads"] // case["kv_heads"], case["block"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for i, (n, h) in enumerate(zip(new, hist)):
        L = case["shared"] + h + n
        blocks = s["table"][i, :-(-L // bs)].long()
        k, v = s["k_rows"][blocks].flatten(0, 1)[:L], s["v_rows"][blocks].flatten(0, 1)[:L]
        later = None
        if n > 1:
            later = torch.arange(L, device="cuda")[None, :] > torch.arange(L - n, L, device="cuda")[:, None]
            later = later.repeat_interleave(G, 0)
        for j in range(case["kv_heads"]):
            q = s["q"][at:at + n, j * G:(j + 1) * G].double().reshape(n * G, -1)
            a = q @ k[:, j].double().t().contiguous() * s["scale"]
            if later is not None:
                a.masked_fill_(later, -math.inf)
            out[at:at + n, j * G:(j + 1) * G] = (torch.softmax(a, 1) @ v[:, j].double()).view(n, G, -1)
        at += n
    return out


def exact(case, seed):
    """Whole numbers have none: the steps' plain forms are in whole numbers or 64 bits themselves."""
    if case["kind"] not in ("append", "attend"):
        return None
    s = prepare(case, seed)
    return _exact_append(s, case) if case["kind"] == "append" else _exact_attend(s, case)
