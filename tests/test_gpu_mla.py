"""Latent attention on the GPU: append, the absorbed and the expanded form against the 64-bit oracle.

Pool rows that no sequence owns, and those past a length, hold NaN unless a test says otherwise, so
a row read where it must not be shows in the output."""
import numpy as np
import pytest
import torch

import jero_hip as J
from mla_oracle import EPS, THETA, Problem, off

pytestmark = pytest.mark.gpu

TYPES = [("f32", "f16"), ("f16", "f16"), ("f32", "f32")]
BIG = dict(rank=512, rope=64, nope=128, v=128)
FORMS = ["absorbed", "expanded"]

# lens, new, heads, block, widths: each edge of the tiles (16, 32, 64 positions; 16, 32, 64, 128 query rows),
# pages that end inside one, sequences of one token and of none
CASES = [
    ([1], [1], 1, 16, {}),
    ([2], [2], 3, 1, dict(rank=8, rope=8, nope=8, v=8)),
    ([15, 16, 17], [1, 1, 1], 5, 4, {}),
    ([31, 32, 33, 34], [1, 3, 0, 2], 4, 16, dict(rank=72, rope=24, nope=40, v=56)),
    ([63, 64, 65], [1, 1, 1], 8, 64, dict(rank=128, rope=32, nope=64, v=64)),
    ([127, 128, 129, 1], [2, 1, 1, 1], 20, 32, dict(rank=128, rope=32, nope=64, v=64)),
    ([200, 5, 77], [1, 1, 1], 17, 16, BIG),
    ([1000], [1], 65, 64, BIG),
    ([515, 40], [1, 4], 128, 16, BIG),
    ([300], [2], 33, 256, dict(rank=328, rope=40, nope=104, v=88)),
    ([130, 131], [1, 1], 2, 8, dict(rank=512, rope=64, nope=256, v=256)),
    ([90, 64], [1, 1], 3, 16, dict(rank=256, rope=64, nope=192, v=192)),
]
PROMPTS = [
    ([130], [130], 2, 16, {}),
    ([64, 65, 129], [64, 65, 129], 3, 32, dict(rank=128, rope=32, nope=64, v=64)),
    ([300, 20, 257], [17, 20, 200], 2, 16, BIG),
    ([97, 256], [31, 128], 3, 4, dict(rank=72, rope=24, nope=40, v=56)),
    ([140], [140], 1, 64, dict(rank=256, rope=64, nope=192, v=256)),
]


def ids(case):
    return "-".join(str(x) for x in case[0]) + f"_h{case[2]}_b{case[3]}_r{case[4].get('rank', 64)}"


def problem(case, act="f32", kv="f16", **kw):
    lens, new, heads, block, dims = case
    return Problem(sum(lens) + heads, lens, new, heads=heads, block=block, act=act, kv=kv, **dims, **kw)


def one_each(p):
    return p.new == [1] * len(p.new)


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("case", CASES + PROMPTS, ids=ids)
@pytest.mark.parametrize("form", FORMS)
def test_against_the_oracle(dev, form, case, act, kv):
    print(f"mla {form} {act} {kv} {case}", flush=True)
    if form == "expanded" and case[4].get("nope", 0) + case[4].get("rope", 0) > 256:
        pytest.skip("refused: nope + rope above 256")
    p = problem(case, act, kv, pad_rows=2)
    p.device(dev)
    ref = p.attention()
    print("  off by", p.check(p.run(form), ref, form), flush=True)
    if form == "absorbed" and one_each(p):  # a decode step: no starts
        q = Problem(sum(case[0]) + case[2], *case[:2], heads=case[2], block=case[3], act=act, kv=kv, **case[4])
        q.device(dev, starts=False)
        q.check(q.run(form), what="without starts")


@pytest.mark.parametrize("form", FORMS)
def test_rows_that_attend_to_nothing_get_zeros(dev, form):
    """An empty sequence, a sequence with more tokens than positions, and a sequence without tokens."""
    p = Problem(5, [0, 3, 7, 40], [1, 5, 0, 2], heads=6, pad_rows=3).device(dev)
    out = p.run(form)
    p.check(out, what=form)
    assert (out[0] == 0).all() and (out[1:3] == 0).all() and (out[3] != 0).any()


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("form", FORMS)
def test_bad_blocks_are_masked(dev, form, act, kv):
    """Ids outside the pool are not followed: their positions are masked, all of them leave zeros."""
    p = Problem(6, [100, 64, 20], [1, 2, 1], heads=5, act=act, kv=kv)
    p.table[0, 2] = p.n_blocks
    p.table[0, 4] = -1
    p.table[1, 0] = 2 ** 31 - 1
    p.table[2, :] = -(2 ** 31)
    p.device(dev)
    out = p.run(form)
    p.check(out, what=form)
    assert (out[3] == 0).all()


@pytest.mark.parametrize("form", FORMS)
def test_positions_from_max_len_on_are_not_attended_to(dev, form):
    p = Problem(7, [100, 30, 64], [3, 1, 1], heads=3, max_len=64).device(dev)
    p.check(p.run(form), what=form)


@pytest.mark.parametrize("form", FORMS)
def test_masked_places_may_hold_anything(dev, form):
    """The rows past each length and the blocks of others hold infinities, or the type's lowest value."""
    for rest in (np.inf, -np.inf, np.finfo(np.float16).min):
        p = Problem(8, [50, 17, 129], [2, 1, 1], heads=4, rest=rest).device(dev)
        p.check(p.run(form), what=f"{form} {rest}")


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("form", FORMS)
def test_peaked_scores(dev, form, act, kv):
    """Queries 40 times as long: one position takes nearly all of a row, the rest underflow."""
    p = Problem(9, [70, 200], [2, 1], heads=4, act=act, kv=kv, gain=60.0).device(dev)
    p.check(p.run(form), what=form)


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("size", [2.0 ** -70, 1e-7, 1e7, 2.0 ** 70])
def test_f32_queries_of_any_size(dev, form, size, kv):
    """Far below and above f16's range, with the scale that brings the scores back."""
    p = Problem(38, [70, 33], [2, 1], heads=3, kv=kv)
    p.q = (p.q.astype(np.float64) * size).astype(np.float32)
    p.scale = float(np.float32(p.scale / size))
    p.device(dev)
    p.check(p.run(form), what=f"{form} {size}")


def test_long_queries_and_far_positions(dev):
    """Absorbed queries past f16's range (their scores are brought back by the scale), and the rotation at a
    position where 32-bit angles are off by 1e-3."""
    p = Problem(10, [40], [1], heads=4)
    p.q *= np.float32(3e4)
    p.scale = float(np.float32(p.scale / 3e4))
    p.device(dev)
    p.check(p.run("absorbed"), what="long queries")
    far = Problem(11, [20001], [1], heads=2, block=256, rank=64, rope=64, max_len=20001).device(dev)
    far.check(far.run("absorbed"), what="far position")
    far.check(far.run("expanded"), what="far position")


@pytest.mark.parametrize("form", FORMS)
def test_rotated_queries(dev, form):
    """rope_theta 0: the queries come rotated."""
    p = Problem(12, [33, 80], [2, 1], heads=3).device(dev)
    p.check(p.run(form, theta=0.0), p.attention(theta=0.0), form)
    p.check(p.run(form, theta=5e5), p.attention(theta=5e5), form)


@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("form", FORMS)
def test_strided_rows(dev, form, act):
    """q and out as columns of wider rows: the columns beside out stay as they were."""
    p = Problem(13, [33, 80], [5, 1], heads=3, act=act).device(dev)
    D, V = p.H * (p.N + p.P), p.H * p.V
    wide = torch.full((p.T, D + 24), float("nan"), dtype=p.d["q"].dtype, device=dev)
    wide[:, 16:16 + D] = p.d["q"].view(p.T, D)
    dst = torch.full((p.T, V + 16), 7.0, dtype=p.d["q"].dtype, device=dev)
    q = wide[:, 16:16 + D].unflatten(1, (p.H, p.N + p.P))
    out = p.run(form, out=dst[:, 8:8 + V].unflatten(1, (p.H, p.V)), q=q)
    p.check(out, what=form)
    assert (dst[:, :8] == 7).all() and (dst[:, 8 + V:] == 7).all()


@pytest.mark.parametrize("form", FORMS)
def test_workspaces(dev, form):
    """A caller's workspace, the library's own, and for the expanded form one that holds a single head's."""
    p = Problem(14, [70, 131], [6, 1], heads=5, rank=128, rope=32, nope=64, v=64).device(dev)
    ref = p.attention()
    want = p.run(form)
    p.check(want, ref, form)
    L = J.lib()
    if form == "absorbed":
        need = L.jero_hip_mla_absorbed_workspace_bytes(p.cache.ref, p.T, p.H)
    else:
        need = L.jero_hip_mla_prefill_workspace_bytes(p.cache.ref, J.F32, 2, p.N, p.V, p.total())
    ws = torch.full((need + 256,), 255, dtype=torch.uint8, device=dev)  # NaNs
    got = p.run(form, workspace=ws[:need])
    torch.cuda.synchronize()
    assert torch.equal(got, want) and (ws[need:] == 255).all()
    with pytest.raises(J.K3Error) as ei:
        p.run(form, workspace=ws[:256])
    assert ei.value.variant == "TensorBoundsError"
    out = torch.zeros_like(want)
    q, d = p.d["q"], p.d
    if form == "absorbed":
        J.check(L.jero_hip_mla_absorbed_attention(p.cache.ref, J.F32, q.data_ptr(), q.stride(0), p.T, p.H, p.N, p.V,
                                                  d["k_b"].data_ptr(), d["v_b"].data_ptr(), p.scale, THETA,
                                                  out.data_ptr(), out.stride(0), None, 0, J._stream()))
    else:
        J.check(L.jero_hip_mla_prefill_attention(p.cache.ref, J.F32, q.data_ptr(), q.stride(0), p.T, p.H, p.N, p.V,
                                                 d["kv_b"].data_ptr(), p.total(), p.scale, THETA, out.data_ptr(),
                                                 out.stride(0), None, 0, J._stream()))
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_sequences_past_total_len_are_empty(dev):
    p = Problem(15, [40, 100, 30], [2, 3, 1], heads=3).device(dev)
    out = p.run("expanded", total=75)  # the second does not fit behind the first, the third does
    want = p.run("expanded")
    torch.cuda.synchronize()
    assert torch.equal(out[:2], want[:2]) and (out[2:5] == 0).all() and torch.equal(out[5], want[5])


@pytest.mark.parametrize("form", FORMS)
def test_same_calls_give_the_same_bits(dev, form):
    p = Problem(16, [700, 90], [3, 1], heads=20, **BIG).device(dev)
    a, b = p.run(form), p.run(form)
    torch.cuda.synchronize()
    assert torch.equal(a, b)


@pytest.mark.parametrize("form", FORMS)
def test_a_captured_call_follows_lengths_and_tables(dev, form):
    """Replayed as the sequences grow and as a block moves, each replay against an eager call, with eager work
    in between."""
    p = Problem(17, [90, 33], [1, 1], heads=4, max_len=128, block=16)
    for s, n in enumerate(p.lens):  # blocks for what will be appended
        p.table[s, :8] = np.arange(8) + 8 * s
    g = np.random.default_rng(1)
    p.n_blocks = 17
    p.rows = g.standard_normal((17, 16, p.R + p.P)).astype(np.float16)
    p.device(dev)
    out = torch.zeros((p.T, p.H, p.V), device=dev)
    L = J.lib()
    need = max(L.jero_hip_mla_absorbed_workspace_bytes(p.cache.ref, p.T, p.H),
               L.jero_hip_mla_prefill_workspace_bytes(p.cache.ref, J.F32, p.H, p.N, p.V, 256))
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    kw = {} if form == "absorbed" else dict(total=256)
    s = torch.cuda.Stream(dev)
    with torch.cuda.stream(s):
        p.run(form, out=out, workspace=ws, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        J.mla_append(p.cache, p.d["x"], p.d["norm"], EPS, THETA)
        p.run(form, out=out, workspace=ws, **kw)
    for step in range(5):
        p.lens = [91 + step, 34 + 17 * step]
        p.d["lens"].copy_(torch.tensor(p.lens, dtype=torch.int32))
        if step == 3:  # the first sequence's block 2 moves to the spare one
            p.d["rows"][16] = p.d["rows"][int(p.table[0, 2])]
            p.table[0, 2] = 16
            p.d["table"].copy_(torch.from_numpy(p.table))
        p.d["x"].copy_(torch.from_numpy(g.standard_normal(p.x.shape).astype(np.float32)))
        p.q = g.standard_normal(p.q.shape).astype(np.float32)
        p.d["q"].copy_(torch.from_numpy(p.q))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        p.rows = p.d["rows"].cpu().numpy()
        p.check(out, what=f"{form} step {step}")
        eager = p.run(form, **kw)
        torch.cuda.synchronize()
        assert torch.equal(eager, out)


def test_two_graphs_by_turns(dev):
    """Both forms captured, each with the workspace it made for itself, replayed by turns with eager calls in
    between."""
    p = Problem(42, [700, 90, 33], [3, 1, 2], heads=6, rank=128, rope=32, nope=64, v=64, pad_rows=1).device(dev)
    ref = p.attention()
    outs, graphs = [], []
    side = torch.cuda.Stream(dev)
    for form in FORMS:
        out = torch.full((p.T, p.H, p.V), 7.0, device=dev)
        with torch.cuda.stream(side):
            p.run(form, out=out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            p.run(form, out=out)
        outs.append(out)
        graphs.append(graph)
    for turn in range(4):
        for out in outs:
            out[:-1].zero_()
        for graph in graphs if turn % 2 else graphs[::-1]:
            graph.replay()
        eager = [p.run(form) for form in FORMS]
        torch.cuda.synchronize()
        for form, out, e in zip(FORMS, outs, eager):
            p.check(out, ref, f"{form} turn {turn}")
            assert torch.equal(out, e)


@pytest.mark.parametrize("form", FORMS)
def test_two_streams_at_once(dev, form):
    """Two calls that overlap, each with a workspace of its own."""
    ps = [Problem(18 + i, [400 + 50 * i], [1 + i], heads=8, rank=128, rope=32, nope=64, v=64).device(dev) for i in range(2)]
    want = [p.run(form).clone() for p in ps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in ps]
    for _ in range(5):
        got = []
        for p, s in zip(ps, streams):
            with torch.cuda.stream(s):
                got.append(p.run(form))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    s = streams[0]
    out = ps[0].run(form, stream=s)
    s.synchronize()
    assert torch.equal(out, want[0])


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("form", FORMS)
def test_later_positions_may_hold_anything(dev, form, act, kv):
    """Rows and queries of NaN and infinities, of a call's own tokens: the tokens before them do not see them, those
    that attend to NaN are NaN."""
    for what, rank in ((np.nan, 64), (np.inf, 128), (-np.inf, 8)):
        p = Problem(32, [40, 150, 9], [6, 150 if form == "expanded" else 4, 1], heads=3, act=act, kv=kv, rank=rank)
        hit = []
        for t, s, pos in p.tokens():
            if (s, pos) in ((0, 37), (1, 148)):
                p.rows[p.table[s, pos // p.block], pos % p.block, -3 if s else rank - 1] = what
                p.q[t] = what
            if s == 0 and pos >= 37 or s == 1 and pos >= 148:
                hit.append(t)
        p.device(dev)
        out = p.run(form).float().cpu().numpy()
        if np.isnan(what):
            assert np.isnan(out[hit]).all()
        with np.errstate(all="ignore"):
            exact, far = p.attention()
        rest = [t for t, _, _ in p.tokens() if t not in hit]
        far_, rms = off(out[rest].astype(np.float64), exact[rest], far[rest])
        assert far_ <= 1 and rms <= 1, (what, far_, rms)


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("form", FORMS)
def test_infinite_latents_with_scores_of_minus_infinity(dev, form, act, kv):
    """A score of minus infinity weighs nothing, but the values beside it are not finite: NaN, as 0 * inf."""
    p = Problem(44, [60, 40], [3, 1], heads=2, nope=8, act=act, kv=kv)
    p.rows[p.table[0, 2], 32 % 16, 0] = np.inf
    first = range(3)
    for h in range(2):
        p.q[:3, h, :8] = -np.sign(p.wk[h, :, 0]) * np.abs(p.q[:3, h, :8])
    p.device(dev)
    out = p.run(form).float().cpu().numpy().astype(np.float64)
    with np.errstate(all="ignore"):
        exact, far = p.attention()
    assert np.isnan(out[list(first)]).all()
    assert off(out[3:4], exact[3:4], far[3:4])[0] <= 1


@pytest.mark.parametrize("scale", [-0.3, 0.0])
@pytest.mark.parametrize("form", FORMS)
def test_other_scales(dev, form, scale):
    """A negative scale, and 0: the mean of the values."""
    p = Problem(33, [70, 33], [2, 1], heads=4)
    p.scale = scale if scale == 0 else float(np.float32(scale))
    p.device(dev)
    p.check(p.run(form), what=form)


@pytest.mark.parametrize("form", FORMS)
def test_rows_before_the_first_start(dev, form):
    """The first sequence's rows begin at 3: those before it belong to none."""
    p = Problem(39, [50, 0, 21], [4, 0, 2], heads=3, pad_rows=3, rest=0.25)
    p.starts += 3
    p.device(dev)
    p.check(p.run(form), what=form)
    J.mla_append(p.cache, p.d["x"], p.d["norm"], EPS, THETA)
    check_rows(p, p.d["rows"], p.rows, *p.appended())


# more than 64 heads, which f16 activations take two 16s a wave: each padded width, part 16s, steps on both sides
# of the buffers' number
@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("heads,dims", [(66, {}), (81, dict(rank=72, rope=24)), (97, dict(rank=256, rope=64)),
                                        (130, dict(rank=200, rope=40)), (113, dict(rank=504, rope=64)), (257, {})],
                         ids=str)
def test_many_heads(dev, heads, dims, act, kv):
    print(f"mla absorbed {act} {kv} {heads} {dims}", flush=True)
    p = Problem(40, [1, 31, 32, 95, 97, 130, 161, 3], [1, 1, 2, 1, 1, 3, 1, 1], heads=heads, nope=16, v=24, act=act, kv=kv,
                pad_rows=1, **dims)
    p.table[4, 2] = -1
    p.device(dev)
    p.check(p.run("absorbed"), what="many heads")


# tokens of a sequence that read its rows together: few heads, sequences of more and of fewer tokens than an item,
# ends within a step, at its edges and past max_len, tokens below position 0, and rows that are not finite
SHARED = [(20, [3, 3, 3, 3], [32, 33, 34, 65], None), (8, [9, 1, 17, 0, 2], [40, 1, 100, 7, 64], None),
          (1, [70, 3, 5], [129, 40, 4], None), (32, [2, 2, 3], [31, 96, 200], 128), (13, [4, 4], [3, 5], None),
          (16, [1, 1, 1, 12], [50, 20, 70, 161], 150)]


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("dims", [{}, dict(rank=200, rope=40), dict(rank=512, rope=64)], ids=["128", "256", "512"])
@pytest.mark.parametrize("heads,new,lens,max_len", SHARED, ids=lambda x: str(x))
def test_tokens_that_share_rows(dev, heads, new, lens, max_len, dims, act, kv):
    print(f"mla absorbed {act} {kv} {heads} {new} {dims}", flush=True)
    p = Problem(41, lens, new, heads=heads, nope=16, v=24, act=act, kv=kv, max_len=max_len, block=8, pad_rows=1, **dims)
    p.table[0, 1 if lens[0] > 8 else 0] = -1 if max_len is None else p.table[0, 0]
    p.device(dev)
    ref = p.attention()
    p.check(p.run("absorbed"), ref, "shared")
    # the last token's own row of NaN: no other sees it
    s = int(np.argmax(p.new))
    t, pos = int(p.starts[s + 1]) - 1, p.lens[s] - 1
    if pos < p.max_len and p.table[s, pos // 8] >= 0:  # (a row of no block is not attended to)
        p.d["rows"][int(p.table[s, pos // 8]), pos % 8, 0] = float("nan")
        out = p.run("absorbed").float().cpu().numpy().astype(np.float64)
        rest = [i for i, _, _ in p.tokens() if i != t]
        assert np.isnan(out[t]).all() and off(out[rest], ref[0][rest], ref[1][rest])[0] <= 1


MANY = [(70, [8] * 70, 2), (600, [1] * 600, 16), (130, [i % 7 for i in range(130)], 4)]


@pytest.mark.parametrize("n,new,block", MANY, ids=lambda x: str(x) if isinstance(x, int) else "")
@pytest.mark.parametrize("form", FORMS)
def test_many_sequences(dev, form, n, new, block):
    """More sequences, and tokens, than a wave's lanes and than a workgroup's threads."""
    print(f"mla {form} {n} sequences", flush=True)
    lens = [(37 * i) % 41 for i in range(n)]
    p = Problem(34, lens, new, heads=2, block=block, nope=8, v=8, pad_rows=1).device(dev)
    ref = p.attention()
    p.check(p.run(form), ref, form)
    if one_each(p):
        q = Problem(34, lens, new, heads=2, block=block, nope=8, v=8).device(dev, starts=False)
        q.check(q.run(form), what="without starts")
    p.device(dev)
    J.mla_append(p.cache, p.d["x"], p.d["norm"], EPS, THETA)
    check_rows(p, p.d["rows"], p.rows, *p.appended())


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("block", [1, 2, 16])
def test_tables_of_many_blocks(dev, block, act, kv):
    """Long sequences of small blocks: the absorbed form reads their ids 64 at a time, and some are none."""
    p = Problem(35, [2500 if block == 16 else 333, 130], [1, 2], heads=3, block=block, act=act, kv=kv, rank=128, rope=32)
    p.table[0, 66:70] = -1
    p.table[0, 130] = p.n_blocks
    p.device(dev)
    ref = p.attention()
    for form in FORMS:
        print(f"mla {form} block {block}", flush=True)
        p.check(p.run(form), ref, form)


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("dims", [{}, dict(rank=72, rope=24), dict(rank=512, rope=64, nope=104, v=128),
                                  dict(rank=328, rope=64, nope=136, v=72), dict(rank=8, rope=8, nope=192, v=256)], ids=str)
def test_positions_of_many_heads(dev, dims, act, kv):
    """Enough heads for the expansion's large tiles: positions that end inside one, a block that is none, and a NaN
    row, which the tokens before it do not see."""
    print(f"mla expanded {act} {kv} {dims}", flush=True)
    p = Problem(43, [200, 0, 131, 1, 190], [3, 1, 0, 1, 2], heads=131, act=act, kv=kv, pad_rows=1, **dims)
    p.table[0, 3] = -1
    p.device(dev)
    ref = p.attention()
    p.check(p.run("expanded"), ref, "many heads")
    p.d["rows"][int(p.table[4, 189 // 16]), 189 % 16, 1] = float("nan")
    out = p.run("expanded").float().cpu().numpy().astype(np.float64)
    rest = [t for t, _, _ in p.tokens() if t != 6]
    assert np.isnan(out[6]).all() and off(out[rest], ref[0][rest], ref[1][rest])[0] <= 1


# lens, new, heads, widths: few blocks of 128 tokens over long sequences, which are cut into runs of 256 positions
# or more, each a partial row a token
LONG = [
    ([1500], [3], 4, {}), ([513], [1], 2, {}), ([257], [257], 2, {}), ([300, 20, 256], [40, 20, 1], 3, {}), ([1100, 700, 40], [2, 130, 1], 3, dict(rank=128, rope=32, nope=64, v=64)),
    ([1025, 0, 600], [1, 1, 40], 5, BIG), ([2049], [1], 2, dict(rank=72, rope=24, nope=192, v=200)),
]


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("case", LONG, ids=lambda c: "-".join(map(str, c[0])))
def test_prompts_cut_into_runs(dev, case, act, kv):
    """With room for the partial rows and without, and where a whole run's blocks are none."""
    print(f"mla expanded {act} {kv} {case}", flush=True)
    lens, new, heads, dims = case
    p = Problem(36, lens, new, heads=heads, block=64, act=act, kv=kv, pad_rows=2, **dims)
    for gone in (False, True):
        if gone:
            p.table[0, 0:8] = -1
            p.table[0, 17:25] = -1
        p.device(dev)
        ref = p.attention()
        p.check(p.run("expanded"), ref, "cut")
        L = J.lib()
        need = L.jero_hip_mla_prefill_workspace_bytes(p.cache.ref, J.F16 if act == "f16" else J.F32, 1, p.N, p.V, p.total())
        ws = torch.full((need + 256,), 255, dtype=torch.uint8, device=dev)
        p.check(p.run("expanded", workspace=ws[:need]), ref, "whole")
        assert (ws[need:] == 255).all()
    if gone:  # and nothing but what is masked
        p.table[0, :] = -1
        p.device(dev)
        out = p.run("expanded")
        p.check(out, what="masked")
        assert (out[:new[0]] == 0).all()


def test_a_captured_long_prompt_follows_its_length(dev):
    """One graph over lengths on both sides of a run's end."""
    p = Problem(37, [1400], [2], heads=4, block=64, pad_rows=1, rest=0.0).device(dev)
    out = torch.full((p.T, p.H, p.V), 7.0, device=dev)
    need = J.lib().jero_hip_mla_prefill_workspace_bytes(p.cache.ref, J.F32, p.H, p.N, p.V, p.total())
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    kw = dict(workspace=ws, total=1400)
    s = torch.cuda.Stream(dev)
    with torch.cuda.stream(s):
        p.run("expanded", out=out, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p.run("expanded", out=out, **kw)
    for n in (1400, 2, 511, 512, 514, 255, 256, 257, 1, 1025, 0, 1399):
        p.lens = [n]
        p.d["lens"].copy_(torch.tensor([n], dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        p.check(out, what=f"length {n}")
        eager = p.run("expanded", total=1400)
        torch.cuda.synchronize()
        assert torch.equal(eager, out)


# ---------------------------------------------------------------- append


def check_rows(p, rows, before, ref, hit):
    got = rows.float().cpu().numpy().astype(np.float64)
    old = before.astype(np.float64)
    assert np.array_equal(got[~hit], old[~hit], equal_nan=True), "rows of no token were written"
    half = 2.0 ** -11 if p.kv == "f16" else 2.0 ** -24
    # the stored value's half step; the f32 arithmetic before it: the mean of squares (rank sums), its root and
    # quotient and two products for the latent, two products and a sum of the pair's length for the key part
    slack = 2.0 ** -24 * (6 + np.sqrt(p.R))
    pair = np.abs(ref[hit])
    k = pair[:, p.R:].reshape(len(pair), -1, 2)
    pair[:, p.R:] = np.repeat(np.sqrt((k ** 2).sum(-1)), 2, -1)
    far = half * np.abs(ref[hit]) + slack * pair + (2.0 ** -25 if p.kv == "f16" else 0)
    assert (np.abs(got[hit] - ref[hit]) <= far).all()


APPENDS = [
    ([1], [1], 16, {}), ([5, 17, 64], [5, 1, 33], 16, {}), ([300, 2, 0], [300, 2, 0], 64, BIG),
    ([20, 3], [4, 3], 1, dict(rank=8, rope=8)), ([100, 50], [100, 7], 32, dict(rank=328, rope=24)),
    ([16, 33], [2, 5], 8, dict(rank=504, rope=56)),
]


@pytest.mark.parametrize("act,kv", TYPES + [("f16", "f32")])
@pytest.mark.parametrize("case", APPENDS, ids=lambda c: f"{c[0]}_{c[2]}")
def test_append(dev, case, act, kv):
    lens, new, block, dims = case
    print(f"mla_append {act} {kv} {case}", flush=True)
    p = Problem(21, lens, new, block=block, act=act, kv=kv, pad_rows=2, **dims).device(dev)
    J.mla_append(p.cache, p.d["x"], p.d["norm"], EPS, THETA)
    check_rows(p, p.d["rows"], p.rows, *p.appended())
    p.device(dev)
    J.mla_append(p.cache, p.d["x"], None, 0.0, 0.0)  # stored as they are
    check_rows(p, p.d["rows"], p.rows, *p.appended(theta=0, norm=False))


@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("before", [1, 3, 8])
def test_append_columns_of_wider_rows(dev, act, before):
    """x at any offset and stride of its elements."""
    p = Problem(22, [40, 9], [13, 9], act=act).device(dev)
    wide = torch.full((p.T, before + p.R + p.P + 5), float("nan"), dtype=p.d["x"].dtype, device=dev)
    wide[:, before:before + p.R + p.P] = p.d["x"]
    J.mla_append(p.cache, wide[:, before:before + p.R + p.P], p.d["norm"], EPS, THETA)
    check_rows(p, p.d["rows"], p.rows, *p.appended())


def test_append_leaves_out_what_has_no_slot(dev):
    """Positions below 0 and from max_len on, and blocks outside the pool."""
    p = Problem(23, [3, 70, 40], [6, 20, 40], max_len=60, rest=0.5)
    p.table[2, 1] = p.n_blocks + 5
    p.table[1, 3] = -1
    p.device(dev)
    J.mla_append(p.cache, p.d["x"], p.d["norm"], EPS, THETA)
    check_rows(p, p.d["rows"], p.rows, *p.appended())


def test_append_far_and_zero_rows(dev):
    """A row of zeros stays zeros (eps), and the rotation holds at the longest context."""
    p = Problem(24, [131072], [2], block=1 << 17, rank=16, rope=64, rest=0.0)
    p.x[0, :16] = 0
    p.device(dev)
    J.mla_append(p.cache, p.d["x"], p.d["norm"], EPS, THETA)
    check_rows(p, p.d["rows"], p.rows, *p.appended())


def test_slots_past_32_bits(dev):
    """A pool of more than 4 GiB: rows whose element and byte offsets do not fit 32 bits are written and read."""
    R, P, bs = 512, 64, 1 << 16
    n = 60  # 60 * 65536 * 576 = 2.26e9 elements, 4.5e9 bytes
    rows = torch.empty((n, bs, R + P), dtype=torch.float16, device=dev)
    table = torch.tensor([[n - 1]], dtype=torch.int32, device=dev)
    p = Problem(25, [80], [80], block=1 << 16, heads=2, **BIG)
    low = Problem(25, [80], [80], block=1 << 16, heads=2, **BIG).device(dev)
    p.d = dict(low.d, rows=rows, table=table)
    rows[n - 1, :80] = low.d["rows"][int(low.table[0, 0]), :80]
    p.cache = J.LatentCache(rows, table, low.d["lens"], R, starts=low.d["starts"], max_len=80)
    for form in FORMS:
        a, b = p.run(form), low.run(form)
        torch.cuda.synchronize()
        assert torch.equal(a, b)
    J.mla_append(p.cache, p.d["x"], p.d["norm"], EPS, THETA)
    J.mla_append(low.cache, low.d["x"], low.d["norm"], EPS, THETA)
    assert torch.equal(rows[n - 1, :80], low.d["rows"][int(low.table[0, 0]), :80])


# ---------------------------------------------------------------- together


@pytest.mark.parametrize("act,kv", TYPES)
def test_a_prompt_and_its_decode_steps(dev, act, kv):
    """As a model's layer runs them: prompts appended and attended to in the expanded form, then tokens one at
    a time in the absorbed form; every step against the oracle over the rows the cache then holds, and the last
    tokens' outputs against the expanded form of the same queries."""
    p = Problem(30, [37, 60], [37, 60], heads=6, act=act, kv=kv, rank=128, rope=32, nope=64, v=64, max_len=96)
    g = np.random.default_rng(2)
    p.table[:] = np.random.default_rng(3).permutation(12).reshape(2, 6)
    p.n_blocks = 12
    p.rows = np.full((12, 16, 160), np.nan, p.rows.dtype)
    p.device(dev)
    J.mla_append(p.cache, p.d["x"], p.d["norm"], EPS, THETA)
    ref, hit = p.appended()
    check_rows(p, p.d["rows"], p.rows, ref, hit)
    p.rows = p.d["rows"].cpu().numpy()
    p.check(p.run("expanded"), what="prompt")
    for step in range(3):
        p.lens = [n + 1 for n in p.lens]
        p.new, p.T = [1, 1], 2
        p.starts = np.array([0, 1, 2], np.int32)
        p.x = (g.standard_normal((2, 160)) * 1.7).astype(p.x.dtype)
        p.q = (g.standard_normal((2, 6, 96)) * 1.5).astype(p.q.dtype)
        p.device(dev, starts=False)
        J.mla_append(p.cache, p.d["x"], p.d["norm"], EPS, THETA)
        p.rows = p.d["rows"].cpu().numpy()
        a = p.run("absorbed")
        p.check(a, what=f"step {step}")
        p.cache = J.LatentCache(p.d["rows"], p.d["table"], p.d["lens"], p.R, starts=torch.from_numpy(p.starts).to(dev),
                                max_len=p.max_len)
        b = p.run("expanded")
        p.check(b, what=f"step {step}")
        exact, bounds = p.attention()
        assert off(a.double().cpu().numpy(), b.double().cpu().numpy(), 2 * bounds)[0] <= 1


def test_refusals_of_the_python_front_end(dev):
    p = Problem(31, [20], [2]).device(dev)
    d, c = p.d, p.cache
    out = torch.zeros((2, 4, 40), device=dev)

    def refused(variant, fn):
        with pytest.raises(J.K3Error) as ei:
            fn()
        assert ei.value.variant == variant

    A = lambda **k: J.mla_absorbed_attention(k.get("out", out), k.get("q", d["q"]), c, k.get("k_b", d["k_b"]),  # noqa: E731
                                             k.get("v_b", d["v_b"]), 0.1, k.get("theta", THETA))
    E = lambda **k: J.mla_prefill_attention(k.get("out", out), k.get("q", d["q"]), c, k.get("kv_b", d["kv_b"]),  # noqa: E731
                                            k.get("total", 20), 0.1, THETA)
    for call in (A, E):
        refused("InvalidArgument", lambda: call(out=out.half()))
        refused("InvalidArgument", lambda: call(q=d["q"].cpu()))
        refused("CapabilityMismatch", lambda: call(q=d["q"].double(), out=out.double()))
        refused("TensorBoundsError", lambda: call(out=out[:1]))
        refused("InvalidArgument", lambda: call(q=d["q"].transpose(1, 2).contiguous().transpose(1, 2)))
        refused("TensorBoundsError", lambda: call(q=d["q"][:0], out=out[:0]))
    refused("InvalidArgument", lambda: A(k_b=d["k_b"].float()))
    refused("TensorBoundsError", lambda: A(k_b=d["k_b"][:3]))
    refused("TensorBoundsError", lambda: A(v_b=d["v_b"][:, :, :56].contiguous()))
    refused("InvalidArgument", lambda: A(theta=-1.0))
    refused("TensorBoundsError", lambda: E(kv_b=d["kv_b"][:, :70].contiguous()))
    refused("TensorBoundsError", lambda: E(total=0))
    refused("TensorBoundsError", lambda: J.mla_append(c, d["x"][:, :79], d["norm"], EPS, THETA))
    refused("TensorBoundsError", lambda: J.mla_append(c, d["x"], d["norm"][:60], EPS, THETA))
    refused("InvalidArgument", lambda: J.mla_append(c, d["x"].cpu(), d["norm"], EPS, THETA))
    refused("InvalidArgument", lambda: J.mla_append(c, d["x"], d["norm"], -1.0, THETA))
    T = torch
    for kw, variant in ((dict(rows=d["rows"].double()), "CapabilityMismatch"), (dict(table=d["table"].long()), "InvalidArgument"),
                        (dict(lens=d["lens"].cpu()), "InvalidArgument"), (dict(rank=80), "TensorBoundsError"),
                        (dict(starts=T.zeros(3, dtype=T.int32, device=dev)), "TensorBoundsError"),
                        (dict(table=d["table"][:, :1].expand(-1, 4)), "InvalidArgument")):
        a = dict(rows=d["rows"], table=d["table"], lens=d["lens"], rank=64)
        a.update(kw)
        refused(variant, lambda: J.LatentCache(**a))
