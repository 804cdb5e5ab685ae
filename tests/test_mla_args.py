"""Refusals of the latent-attention entry points, without a GPU: every call here fails its checks before
anything is enqueued, and no pointer is followed."""
import ctypes as C

import pytest
import torch

import jero_hip as J

FAKE = 0x10000  # 16-byte and 256-byte aligned, never followed


def cache(**kw):
    d = dict(rows_dev=FAKE, table_dev=FAKE, lens_dev=FAKE, starts_dev=None, n_blocks=8, table_stride=4, n_seqs=2, max_len=64,
             block_size=16, kv_dtype=J.KV_F16, rank=64, rope_dim=16)
    d.update(kw)
    return J.HipLatentCache(**d)


def append(c, act=J.F32, x=FAKE, stride=80, tokens=2, norm=FAKE, eps=1e-6, theta=1e4):
    return J.lib().jero_hip_mla_append(C.byref(c) if c else None, act, x, stride, tokens, norm, eps, theta, None)


def absorbed(c, act=J.F32, q=FAKE, qs=96, tokens=2, heads=2, nope=32, v=40, kb=FAKE, vb=FAKE, scale=0.1, theta=1e4, out=FAKE,
             os_=80, ws=FAKE, n=1 << 30):
    return J.lib().jero_hip_mla_absorbed_attention(C.byref(c) if c else None, act, q, qs, tokens, heads, nope, v, kb, vb,
                                                   scale, theta, out, os_, ws, n, None)


def prefill(c, act=J.F32, q=FAKE, qs=96, tokens=2, heads=2, nope=32, v=40, w=FAKE, total=128, scale=0.1, theta=1e4, out=FAKE,
            os_=80, ws=FAKE, n=1 << 30):
    return J.lib().jero_hip_mla_prefill_attention(C.byref(c) if c else None, act, q, qs, tokens, heads, nope, v, w, total,
                                                  scale, theta, out, os_, ws, n, None)


BAD_CACHES = [
    (dict(rows_dev=None), 21), (dict(table_dev=None), 21), (dict(lens_dev=None), 21), (dict(rows_dev=FAKE + 8), 21),
    (dict(table_dev=FAKE + 2), 21), (dict(lens_dev=FAKE + 1), 21), (dict(starts_dev=FAKE + 2), 21),
    (dict(kv_dtype=2), 10), (dict(kv_dtype=-1), 10), (dict(rank=0), 10), (dict(rank=60), 10), (dict(rank=520), 10),
    (dict(rank=-8), 10), (dict(rope_dim=0), 10), (dict(rope_dim=12), 10), (dict(rope_dim=72), 10),
    (dict(block_size=0), 10), (dict(block_size=24), 10), (dict(block_size=1 << 21), 10), (dict(block_size=-16), 10),
    (dict(n_blocks=0), 14), (dict(n_blocks=1 << 31), 14), (dict(n_seqs=0), 14), (dict(n_seqs=-1), 14), (dict(max_len=0), 14),
    (dict(n_seqs=1), 14), (dict(n_seqs=3), 14),  # two tokens, no starts
    (dict(max_len=65), 14), (dict(table_stride=0), 14), (dict(table_stride=-4), 14),
    (dict(max_len=4194305), 12),
]


@pytest.mark.parametrize("call", [append, absorbed, prefill])
def test_bad_caches(call):
    assert call(None) == 21
    for kw, status in BAD_CACHES:
        assert call(cache(**kw)) == status, kw


def test_bad_append():
    c = cache()
    assert append(c, act=J.BF16) == 10 and append(c, act=-1) == 10
    assert append(c, x=None) == 21 and append(c, x=FAKE + 2) == 21 and append(c, act=J.F16, x=FAKE + 1) == 21
    assert append(c, norm=FAKE + 2) == 21
    assert append(c, stride=79) == 14 and append(c, tokens=0) == 14 and append(c, tokens=-1) == 14
    for eps in (-1e-6, float("nan"), float("inf")):
        assert append(c, eps=eps) == 21
    for theta in (-1e4, float("nan"), float("inf")):
        assert append(c, theta=theta) == 21


@pytest.mark.parametrize("call", [absorbed, prefill])
def test_bad_attention(call):
    c = cache()
    assert call(c, act=J.BF16) == 10
    assert call(cache(kv_dtype=J.KV_F32), act=J.F16) == 10  # f16 activations over an f32 cache
    assert call(c, q=None) == 21 and call(c, out=None) == 21 and call(c, q=FAKE + 8) == 21 and call(c, out=FAKE + 4) == 21
    assert call(c, heads=0) == 14 and call(c, heads=1025) == 10
    assert call(c, nope=0) == 10 and call(c, nope=36) == 10 and call(c, nope=264) == 10
    assert call(c, v=0) == 10 and call(c, v=20) == 10 and call(c, v=264) == 10
    assert call(c, qs=95) == 14 and call(c, os_=79) == 14 and call(c, qs=100) == 21 and call(c, os_=84) == 21
    assert call(c, tokens=0) == 14 and call(c, tokens=1 << 23) == 14
    for x in (float("nan"), float("inf")):
        assert call(c, scale=x) == 21 and call(c, theta=x) == 21
    assert call(c, theta=-1.0) == 21
    assert call(c, n=100) == 14 and call(c, ws=FAKE + 16) == 21


def test_bad_weights_and_totals():
    c = cache()
    assert absorbed(c, kb=None) == 21 and absorbed(c, vb=None) == 21 and absorbed(c, vb=FAKE + 8) == 21
    assert prefill(c, w=None) == 21 and prefill(c, w=FAKE + 2) == 21
    assert prefill(c, total=0) == 14 and prefill(c, total=1 << 31) == 14
    assert prefill(c, nope=248, qs=2 * 264) == 10  # nope + rope above 256


def test_largest_calls():
    """Tokens, sequences, expanded rows and tiles past what the kernels' 32-bit counts are made for."""
    c = cache(n_seqs=1 << 20, starts_dev=FAKE)
    for call in (append, absorbed, prefill):
        assert call(c) == 14
        assert call(cache(starts_dev=FAKE), tokens=(1 << 19) + 1) == 14
    assert prefill(cache(), total=(1 << 23) + 1) == 14
    wide = dict(tokens=1 << 19, heads=1024, qs=1024 * 48, os_=1024 * 40)
    assert prefill(cache(n_seqs=1 << 19), n=1 << 62, **wide) == 10  # 2^19 tiles of 1024 heads
    assert absorbed(cache(n_seqs=1 << 19), **wide) == 10  # 2^29 rows
    assert prefill(cache(n_seqs=4097, starts_dev=FAKE)) == 10
    long = dict(max_len=1 << 22, table_stride=1 << 18)
    assert absorbed(cache(n_seqs=4097, **long), tokens=4097, n=0) == 10
    assert absorbed(cache(n_seqs=4096, **long), tokens=4096, n=0) == 14  # its workspace


def test_workspace_sizes():
    L, c = J.lib(), cache()
    assert L.jero_hip_mla_absorbed_workspace_bytes(None, 1, 1) == 0
    assert L.jero_hip_mla_absorbed_workspace_bytes(C.byref(c), 0, 1) == 0
    a, b = (L.jero_hip_mla_absorbed_workspace_bytes(C.byref(c), t, 4) for t in (1, 9))
    assert 0 < a < b
    one, two = (L.jero_hip_mla_prefill_workspace_bytes(C.byref(c), J.F32, h, 32, 40, 100) for h in (1, 2))
    assert 0 < one < two
    # all heads at once up to 1 GiB, and one head's whatever its size
    big = L.jero_hip_mla_prefill_workspace_bytes(C.byref(c), J.F16, 128, 128, 128, 1 << 20)
    assert big <= 1 << 30 and big >= L.jero_hip_mla_prefill_workspace_bytes(C.byref(c), J.F16, 1, 128, 128, 1 << 20)
    huge = (1 << 31) - 1
    assert L.jero_hip_mla_prefill_workspace_bytes(C.byref(c), J.F32, 128, 128, 128, huge) == \
        L.jero_hip_mla_prefill_workspace_bytes(C.byref(c), J.F32, 1, 128, 128, huge)


def test_host_tensors_are_refused():
    rows = torch.zeros(2, 16, 80, dtype=torch.float16)
    with pytest.raises(J.K3Error) as ei:
        J.LatentCache(rows, torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 64)
    assert ei.value.variant == "InvalidArgument"
