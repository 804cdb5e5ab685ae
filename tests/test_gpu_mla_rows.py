"""Token rows of latent attention that belong to no sequence, on the GPU: not read, not written."""
import numpy as np
import pytest
import torch

import jero_hip as J
from mla_oracle import EPS, THETA, Problem

pytestmark = pytest.mark.gpu

MIB = 1 << 20


def at_the_end(dev, a):
    """a's values as the last bytes of an allocation of their own."""
    whole = torch.zeros(32 * MIB, dtype=torch.uint8, device=dev)
    raw = torch.from_numpy(a).view(torch.uint8).flatten().to(dev)
    whole[whole.numel() - raw.numel():] = raw
    return whole, whole.data_ptr() + whole.numel() - raw.numel()


@pytest.mark.parametrize("first", [0, 3, 17])
@pytest.mark.parametrize("new,heads,tokens", [([1, 1, 1], 3, 64), ([4, 2, 3], 5, 40), ([1, 0, 2], 65, 21), ([0, 0, 0], 2, 9)],
                         ids=str)
@pytest.mark.parametrize("act", ["f32", "f16"])
def test_a_call_of_more_rows_than_there_are(dev, act, new, heads, tokens, first):
    """A call padded to `tokens` rows, as a captured one is, whose x and q end with the last sequence's rows: those
    behind them (and the outputs of all that belong to none) are left alone."""
    print(f"mla padded {act} {new} {heads} heads, {tokens} tokens from {first} on", flush=True)
    p = Problem(60, [40, 33, 70], new, heads=heads, act=act, rest=0.25)
    live = sum(new)
    p.starts += first
    head = lambda a: np.concatenate([np.full((first,) + a.shape[1:], np.nan, a.dtype), a[:live]])  # noqa: E731
    p.q, p.x, p.T = head(p.q), head(p.x), tokens + first
    p.device(dev)
    A = J.F16 if act == "f16" else J.F32
    qs, os_ = heads * (p.N + p.P), heads * p.V
    keep, q = at_the_end(dev, p.q) if len(p.q) else (None, p.d["norm"].data_ptr())
    kept, x = at_the_end(dev, p.x) if len(p.x) else (None, p.d["norm"].data_ptr())
    ref = p.attention()
    L, d = J.lib(), p.d
    for form in ("absorbed", "expanded"):
        out = torch.full((p.T, heads, p.V), 7.0, dtype=d["q"].dtype, device=dev)
        if form == "absorbed":
            need = L.jero_hip_mla_absorbed_workspace_bytes(p.cache.ref, p.T, heads)
            ws = torch.full((need,), 255, dtype=torch.uint8, device=dev)
            J.check(L.jero_hip_mla_absorbed_attention(p.cache.ref, A, q, qs, p.T, heads, p.N, p.V, d["k_b"].data_ptr(),
                                                      d["v_b"].data_ptr(), p.scale, THETA, out.data_ptr(), os_,
                                                      ws.data_ptr(), need, J._stream()))
        else:
            need = L.jero_hip_mla_prefill_workspace_bytes(p.cache.ref, A, heads, p.N, p.V, p.total())
            ws = torch.full((need,), 255, dtype=torch.uint8, device=dev)
            J.check(L.jero_hip_mla_prefill_attention(p.cache.ref, A, q, qs, p.T, heads, p.N, p.V, d["kv_b"].data_ptr(),
                                                     p.total(), p.scale, THETA, out.data_ptr(), os_, ws.data_ptr(), need,
                                                     J._stream()))
        torch.cuda.synchronize()
        if live:
            p.check(out, ref, form)
        else:
            assert (out == 7).all()
    J.check(L.jero_hip_mla_append(p.cache.ref, A, x, p.R + p.P, p.T, d["norm"].data_ptr(), EPS, THETA, J._stream()))
    torch.cuda.synchronize()
    rows, hit = p.appended()
    got = d["rows"].double().cpu().numpy()
    assert np.array_equal(got[~hit], p.rows[~hit].astype(np.float64))
    # half a step of f16 and of the f32 arithmetic before it (at most 16 roundings of values up to 8)
    assert (np.abs(got[hit] - rows[hit]) <= 2.0 ** -11 * np.abs(rows[hit]) + 2.0 ** -17).all()


@pytest.mark.parametrize("one", [True, False], ids=["no starts", "starts"])
def test_lengths_far_below_zero(dev, one):
    """A length at the end of 32 bits: the sequence's tokens are at positions below 0, stored nowhere, zeros out."""
    p = Problem(61, [50, 60, 40, 64], [1] * 4 if one else [1, 3, 2, 2], heads=3, rest=0.25)
    p.lens[1], p.lens[2] = -(2 ** 31), -(2 ** 31) + 1
    p.device(dev, starts=not one)
    for form in ("absorbed", "expanded"):
        print(f"mla {form}, lengths far below 0", flush=True)
        out = p.run(form)
        p.check(out, what=form)
        assert (out[1:2 if one else 6] == 0).all()
    J.mla_append(p.cache, p.d["x"], p.d["norm"], EPS, THETA)
    _, hit = p.appended()
    got = p.d["rows"].double().cpu().numpy()
    assert np.array_equal(got[~hit], p.rows[~hit].astype(np.float64)) and hit.sum() == (2 if one else 3)
