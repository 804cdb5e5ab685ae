"""Refusals of the paged serving entry points, without a GPU: every call here fails its checks before anything is
enqueued, and no pointer is followed.  Frequencies of the rotations, which are a host call."""
import ctypes as C

import numpy as np
import pytest

import jero_hip as J
import paged_oracle as P

FAKE = 0x10000  # aligned, never followed


def pool(**kw):
    d = dict(table_dev=FAKE, lens_dev=FAKE, owned_dev=FAKE, free_dev=FAKE, n_free_dev=FAKE, lens_out_dev=None,
             owned_out_dev=None, n_free_out_dev=None, n_seqs=4, table_stride=8, n_blocks=16, free_capacity=16,
             shared_blocks=0, block_size=16)
    d.update(kw)
    return J.HipBlockPool(**d)


def extend(p, new=FAKE, drop=None, tokens=8, starts=FAKE, granted=None, positions=FAKE, slots=FAKE, ws=None, n=0):
    return J.lib().jero_hip_paged_extend(C.byref(p) if p else None, new, drop, tokens, starts, granted, positions, slots, ws, n,
                                         None)


def test_bad_pools():
    assert extend(None) == 21
    for name in ("table_dev", "lens_dev", "owned_dev", "free_dev", "n_free_dev"):
        assert extend(pool(**{name: None})) == 21 and extend(pool(**{name: FAKE + 2})) == 21, name
    for name in ("lens_out_dev", "owned_out_dev", "n_free_out_dev"):
        assert extend(pool(**{name: FAKE + 1})) == 21, name
    for kw, status in [(dict(block_size=0), 10), (dict(block_size=24), 10), (dict(block_size=1 << 21), 10),
                       (dict(block_size=-16), 10), (dict(n_seqs=0), 14), (dict(n_seqs=(1 << 19) + 1), 14),
                       (dict(table_stride=0), 14), (dict(table_stride=1 << 30), 14), (dict(n_blocks=0), 14),
                       (dict(n_blocks=1 << 31), 14), (dict(free_capacity=0), 14), (dict(free_capacity=1 << 31), 14),
                       (dict(shared_blocks=-1), 14), (dict(shared_blocks=9), 14),
                       (dict(table_stride=1 << 12, block_size=1 << 20), 12)]:
        assert extend(pool(**kw)) == status, kw


def test_bad_extend():
    p = pool()
    for kw in (dict(new=None), dict(starts=None), dict(positions=None), dict(slots=None), dict(new=FAKE + 2), dict(drop=FAKE + 1),
               dict(granted=FAKE + 2), dict(positions=FAKE + 2), dict(slots=FAKE + 4)):
        assert extend(p, **kw) == 21, kw
    assert extend(p, tokens=0) == 14 and extend(p, tokens=-1) == 14 and extend(p, tokens=(1 << 24) + 1) == 14
    big = pool(n_seqs=2000)
    need = J.lib().jero_hip_paged_extend_workspace_bytes(2000)
    assert need >= 2000 * 16
    assert extend(big, ws=FAKE, n=need - 1) == 14 and extend(big, ws=FAKE + 8, n=need) == 21
    assert J.lib().jero_hip_paged_extend_workspace_bytes(0) == 0


def rope_init(rot=64, layout=0, theta=1e4, scaling=0, factor=1.0, original=4096.0, low=0.0, high=0.0, out=True):
    r = J.HipRope()
    return J.lib().jero_hip_rope_init(C.byref(r) if out else None, rot, layout, theta, scaling, factor, original, low, high)


def test_bad_ropes():
    nan, inf = float("nan"), float("inf")
    assert rope_init() == 0 and rope_init(out=False) == 21
    for kw in (dict(rot=0), dict(rot=-8), dict(rot=12), dict(rot=264), dict(layout=2), dict(layout=-1), dict(scaling=5),
               dict(scaling=-1)):
        assert rope_init(**kw) == 10, kw
    for theta in (0.0, 1.0, -1e4, nan, inf):
        assert rope_init(theta=theta) == 21
    for scaling in (1, 2, 3, 4):
        for factor in (0.0, 0.5, -2.0, nan, inf):
            assert rope_init(scaling=scaling, factor=factor) == 21
    for scaling in (3, 4):
        for kw in (dict(original=0.0), dict(original=nan), dict(original=inf), dict(low=-1.0), dict(low=8.0, high=4.0),
                   dict(low=2.0, high=2.0), dict(low=nan), dict(high=inf)):
            assert rope_init(scaling=scaling, factor=2.0, **kw) == 21, kw
    with pytest.raises(J.K3Error):
        J.Rope(64, 1e4, layout="pairs")
    with pytest.raises(J.K3Error):
        J.Rope(64, 1e4, scaling="other")


@pytest.mark.parametrize("scaling,factor,original", [("none", 1.0, 0), ("linear", 4.0, 0), ("ntk", 8.0, 0), ("yarn", 4.0, 32768),
                                                     ("yarn", 1.0, 2048), ("wavelength", 8.0, 8192), ("wavelength", 2.0, 64)])
@pytest.mark.parametrize("rot,theta", [(8, 1e4), (64, 1e4), (128, 1e6), (256, 5e5)])
def test_frequencies(rot, theta, scaling, factor, original):
    """64-bit powers and logarithms on both sides: a few units in the last place."""
    r = J.Rope(rot, theta, scaling=scaling, factor=factor, original=original)
    f, m = P.frequencies(rot, theta, scaling, factor, original)
    got = np.array(r.c.turns[:rot // 2]) * 2 * np.pi
    assert np.max(np.abs(got / f - 1)) < 1e-13
    assert r.c.magnitude == np.float32(m) and r.c.rot_dim == rot


def append(act=J.F32, q=FAKE, qs=256, k=FAKE, ks=128, v=FAKE, vs=128, tokens=3, heads=4, kv=2, dim=64, pos=FAKE, slots=FAKE,
           rope=True, qn=None, kn=None, eps=1e-6, qo=FAKE, qos=256, kr=FAKE, vr=FAKE, kd=J.KV_F16, n=64, rot=64):
    r = J.Rope(rot, 1e4) if rope else None
    return J.lib().jero_hip_paged_append(act, q, qs, k, ks, v, vs, tokens, heads, kv, dim, pos, slots, r.ref if r else None,
                                         qn, kn, eps, qo, qos, kr, vr, kd, n, None)


def test_bad_append():
    for kw in (dict(act=J.BF16), dict(kd=2), dict(heads=1025), dict(kv=1025), dict(dim=0), dict(dim=60), dict(dim=264)):
        assert append(**kw) == 10, kw
    for kw in (dict(q=None), dict(qo=None), dict(k=None), dict(v=None), dict(kr=None), dict(vr=None), dict(slots=None),
               dict(pos=None), dict(q=FAKE + 8), dict(qo=FAKE + 8), dict(k=FAKE + 4), dict(v=FAKE + 8), dict(kr=FAKE + 8),
               dict(vr=FAKE + 2), dict(pos=FAKE + 2), dict(slots=FAKE + 4), dict(qn=FAKE + 4), dict(kn=FAKE + 8),
               dict(qs=260), dict(qos=260), dict(ks=132), dict(vs=132)):
        assert append(**kw) == 21, kw
    for eps in (-1e-6, float("nan"), float("inf")):
        assert append(qn=FAKE, eps=eps) == 21 and append(kn=FAKE, eps=eps) == 21
    for kw in (dict(heads=0, kv=0), dict(heads=-1), dict(kv=-1), dict(tokens=0), dict(tokens=(1 << 24) + 1), dict(qs=248),
               dict(qos=248), dict(ks=120), dict(vs=120), dict(n=0), dict(rot=128)):
        assert append(**kw) == 14, kw


def test_append_tokens_that_a_launch_holds():
    """256 threads a token, and a launch has fewer than 2^32 threads."""
    for tokens in (1 << 24, (1 << 24) + 1):
        assert append(tokens=tokens) == 14


def test_append_in_place_at_another_stride():
    """A token's results would fall on another's queries."""
    for other in (dict(qos=512), dict(qs=512)):
        assert append(qo=FAKE, q=FAKE, **other) == 21
        assert "one stride" in J.lib().jero_hip_last_error().decode()


def verify(target=FAKE, ts=100000, draft=FAKE, ds=100000, tokens=FAKE, starts=FAKE, u=FAKE, ul=FAKE, n=2, T=6, N=4, V=100000, out=FAKE,
           acc=FAKE, dropped=None, ws=FAKE, size=1 << 20):
    return J.lib().jero_hip_verify_drafts(target, ts, draft, ds, tokens, starts, u, ul, n, T, N, V, out, acc, dropped, ws, size,
                                          None)


def test_bad_verify():
    for kw in (dict(target=None), dict(tokens=None), dict(starts=None), dict(u=None), dict(ul=None), dict(out=None),
               dict(acc=None), dict(target=FAKE + 2), dict(draft=FAKE + 1), dict(tokens=FAKE + 2), dict(starts=FAKE + 2),
               dict(u=FAKE + 2), dict(ul=FAKE + 2), dict(out=FAKE + 2), dict(acc=FAKE + 2), dict(dropped=FAKE + 2),
               dict(ws=FAKE + 8)):
        assert verify(**kw) == 21, kw
    for kw in (dict(n=0), dict(n=65536), dict(T=0), dict(T=(1 << 22) + 1), dict(N=-1), dict(N=6), dict(V=0),
               dict(V=(1 << 24) + 1), dict(ts=99999), dict(ds=99999), dict(size=31)):
        assert verify(**kw) == 14, kw
    size = J.lib().jero_hip_verify_drafts_workspace_bytes
    assert size(0, 100) == size(65536, 100) == size(2, 0) == size(2, (1 << 24) + 1) == 0
    need = size(2, 100000)
    assert size(2, 100) == 0 < need < size(2, 200000) and verify(size=need - 1) == 14


def cache(**kw):
    d = dict(k_dev=FAKE, v_dev=FAKE, table_dev=FAKE, lens_dev=FAKE, starts_dev=None, shared_dev=None, n_blocks=8,
             table_stride=4, n_seqs=2, max_len=64, shared_blocks=0, block_size=16, kv_dtype=J.KV_F16, n_heads_kv=2, head_dim=64)
    d.update(kw)
    return J.HipPagedCache(**d)


def attention(c, act=J.F32, q=FAKE, qs=256, tokens=2, heads=4, scale=0.1, out=FAKE, os_=256, ws=FAKE, n=1 << 30):
    return J.lib().jero_hip_paged_attention(C.byref(c) if c else None, act, q, qs, tokens, heads, scale, out, os_, ws, n, None)


BAD_CACHES = [
    (dict(k_dev=None), 21), (dict(v_dev=None), 21), (dict(table_dev=None), 21), (dict(lens_dev=None), 21),
    (dict(k_dev=FAKE + 8), 21), (dict(v_dev=FAKE + 4), 21), (dict(table_dev=FAKE + 2), 21), (dict(lens_dev=FAKE + 1), 21),
    (dict(starts_dev=FAKE + 2), 21), (dict(shared_dev=FAKE + 2), 21), (dict(kv_dtype=2), 10), (dict(head_dim=0), 10),
    (dict(head_dim=60), 10), (dict(head_dim=264), 10), (dict(block_size=0), 10), (dict(block_size=24), 10),
    (dict(block_size=1 << 21), 10), (dict(n_blocks=0), 14), (dict(n_blocks=1 << 31), 14), (dict(n_seqs=0), 14),
    (dict(n_seqs=1), 14), (dict(n_seqs=3), 14), (dict(n_heads_kv=0), 14), (dict(n_heads_kv=3), 14), (dict(max_len=0), 14),
    (dict(max_len=65), 14), (dict(table_stride=0), 14), (dict(shared_blocks=1), 14), (dict(shared_blocks=-1), 14),
    (dict(shared_blocks=5, shared_dev=FAKE), 14), (dict(max_len=4194305), 12),
]


def test_bad_attention():
    assert attention(None) == 21
    size = J.lib().jero_hip_paged_attention_workspace_bytes
    for kw, status in BAD_CACHES:
        assert attention(cache(**kw)) == status, kw
        assert size(C.byref(cache(**kw)), J.F32, 2, 4) == 0, kw
    c = cache()
    assert attention(c, act=J.BF16) == 10 and attention(cache(kv_dtype=J.KV_F32), act=J.F16) == 10
    for kw in (dict(q=None), dict(out=None), dict(q=FAKE + 8), dict(out=FAKE + 4), dict(qs=260), dict(os_=260),
               dict(scale=float("nan")), dict(scale=float("inf"))):
        assert attention(c, **kw) == 21, kw
    for kw in (dict(heads=0), dict(heads=3), dict(tokens=0), dict(tokens=1 << 23), dict(qs=248), dict(os_=248)):
        assert attention(c, **kw) == 14, kw
    assert attention(c, heads=1026) == 10
    many = cache(n_seqs=1 << 19, n_heads_kv=16, starts_dev=FAKE)
    assert attention(many, tokens=4, heads=16, qs=1024, os_=1024) == 10
    assert attention(cache(n_seqs=1 << 16, n_heads_kv=1), tokens=1 << 16, heads=1024, qs=65536, os_=65536) == 10
    # a call whose positions are cut wants room for its parts
    long = cache(table_stride=1 << 10, max_len=1 << 14)
    need = size(C.byref(long), J.F32, 2, 4)
    assert need > 0
    assert attention(long, n=need - 1) == 14 and attention(long, ws=FAKE + 16, n=need) == 21
    assert size(C.byref(cache()), J.F32, 2, 4) == 0
