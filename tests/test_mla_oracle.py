"""The latent-attention oracle: both forms of the definition agree, and its bounds tell mistakes."""
import numpy as np
import pytest

from mla_oracle import THETA, Problem, off as how_far, rotate


def small(act="f32", **kw):
    return Problem(3, [9, 33, 1], [2, 3, 1], heads=3, act=act, rest=0.0, **kw)


def test_the_absorbed_form_is_the_expanded_one():
    p = small()
    exact, _ = p.attention()
    for t, s, pos in p.tokens():
        c = p.visible(s, pos)
        for h in range(p.H):
            q = p.q[t, h].astype(np.float64)
            qa = np.concatenate([p.wk[h].astype(np.float64).T @ q[:p.N], rotate(q[p.N:], pos)])
            a = p.scale * (c @ qa)
            w = np.exp(a - a.max())
            o = (w / w.sum()) @ c[:, :p.R]
            assert np.allclose(p.wv[h].astype(np.float64) @ o, exact[t, h], rtol=1e-12, atol=1e-13)


def test_rotation_keeps_scores_of_equal_distance():
    g = np.random.default_rng(0)
    a, b = g.standard_normal((2, 32))
    assert abs(rotate(a, 7) @ rotate(b, 3) - rotate(a, 104) @ rotate(b, 100)) < 1e-12


def test_empty_rows_are_zero():
    p = Problem(1, [0, 2], [1, 3], rest=0.0)
    exact, _ = p.attention()
    assert (exact[0] == 0).all() and (exact[1] == 0).all() and (exact[2] != 0).any()


@pytest.mark.parametrize("act", ["f32", "f16"])
def test_bounds_tell_mistakes(act):
    """A computed row within the bounds passes; each planted mistake is outside them."""
    p = small(act)
    exact, far = p.attention()
    rows = [t for t, _, _ in p.tokens()]

    def off(y):
        return max(how_far(y[rows], exact[rows], far[rows])) > 1

    def with_(**kw):
        old = {k: getattr(p, k) for k in kw}
        for k, v in kw.items():
            setattr(p, k, v)
        y, _ = p.attention()
        for k, v in old.items():
            setattr(p, k, v)
        return y

    assert not off(exact)
    # the precision the bounds stand for: the factors rounded once
    if act == "f16":
        assert not off(with_(q=p.q.astype(np.float16)))
    else:
        assert off(with_(q=p.q.astype(np.float16)))  # f32 queries must not be rounded to f16
    assert off(with_(scale=p.scale * 1.02))
    assert off(p.attention(causal=False)[0])
    assert off(p.attention(turn=False)[0])
    assert off(p.attention(theta=THETA * 2)[0])
    assert off(with_(wv=np.roll(p.wv, 1, 0)))
    assert off(with_(wk=np.roll(p.wk, 1, 1)))
    assert off(with_(lens=[n - 1 for n in p.lens]))  # every token one position early
    assert off(with_(table=np.roll(p.table, 1, 0)))
