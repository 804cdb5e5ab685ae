"""Latent attention on the GPU at the ends of f16's range: cached rows, expanded keys and values."""
import numpy as np
import pytest

from mla_oracle import Problem, off

pytestmark = pytest.mark.gpu

TYPES = [("f32", "f16"), ("f16", "f16"), ("f32", "f32")]
WIDTHS = [{}, dict(rank=128, rope=32, nope=64, v=128), dict(rank=72, rope=40, nope=192, v=200)]


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("dims", WIDTHS, ids=["64", "128", "256"])
def test_expanded_values_past_the_range(dev, dims, act, kv):
    """Finite latents whose expanded values (and some keys) pass 65504: not finite for the tokens that attend to them,
    and no other token sees them.  Late positions of a prompt, one that ends inside a tile, and its last."""
    p = Problem(70, [40, 150, 300, 9], [6, 150, 200, 1], heads=3, act=act, kv=kv, **dims)
    odd = {0: [37], 1: [31, 148], 2: [110, 299]}
    for s, places in odd.items():
        for pos in places:
            p.rows[p.table[s, pos // p.block], pos % p.block, :p.R] = 3e4 * np.sign(p.wv[s, 5].astype(np.float32))
    hit = [t for t, s, pos in p.tokens() if s in odd and pos >= min(odd[s])]
    rest = [t for t, _, _ in p.tokens() if t not in hit]
    # the latents themselves are within the range: the absorbed form attends to them as to any
    exact, far = p.attention()
    p.device(dev)
    print(f"mla expanded {act} {kv} {dims}: values past the range", flush=True)
    out = p.run("expanded").float().cpu().numpy().astype(np.float64)
    far_, rms = off(out[rest], exact[rest], far[rest])
    assert far_ <= 1 and rms <= 1, (far_, rms)
    for t, s, pos in p.tokens():
        if t in hit:
            assert not np.isfinite(out[t, s, 5]), (t, s, pos)
    if act == "f32":
        print(f"mla absorbed {act} {kv} {dims}: large latents", flush=True)
        out = p.run("absorbed").float().cpu().numpy().astype(np.float64)
        far_, rms = off(out[rest], exact[rest], far[rest])
        assert far_ <= 1 and rms <= 1 and np.isfinite(out[hit]).all(), (far_, rms)


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("size", [2.0 ** -6, 2.0 ** 4, 2.0 ** 9])
@pytest.mark.parametrize("form", ["absorbed", "expanded"])
def test_cached_rows_of_other_sizes(dev, form, size, act, kv):
    """Rows far from 1, with the scale that brings the scores back.  Where parts reach f16's last place, cached,
    expanded and merged values are off by up to 2^-25 more (deviation / sqrt 3): an output by that of a weight row's
    sum (its root of squares), and a score by that of its absorbed and plain queries', which moves an output by the
    spread of the values."""
    p = Problem(71, [90, 33, 130], [3, 1, 2], heads=4, act=act, kv=kv)
    p.rows = (p.rows.astype(np.float64) * size).astype(p.rows.dtype)
    p.scale = float(np.float32(p.scale / size))
    exact, far = p.attention()
    last, wv, wk, q = 2.0 ** -25, p.wv.astype(np.float64), p.wk.astype(np.float64), p.q.astype(np.float64)
    absorbed = np.einsum("thn,hnr->thr", q[..., :p.N], wk)
    both = np.concatenate([absorbed, q], -1)
    spread = max(np.ptp(p.visible(s, n - 1)[:, :p.R] @ wv.reshape(-1, p.R).T) for s, n in enumerate(p.lens))
    far[..., 0] += last * (np.abs(wv).sum(2).max() + 1 + p.scale * np.abs(both).sum(-1).max() * spread)
    far[..., 1] += last / np.sqrt(3) * (np.sqrt((wv ** 2).sum(2).max()) + 1 +
                                        p.scale * np.sqrt((both ** 2).sum(-1).max()) * spread)
    p.device(dev)
    print(f"mla {form} {act} {kv}: rows of {size}", flush=True)
    print("  off by", p.check(p.run(form), (exact, far), form), flush=True)
