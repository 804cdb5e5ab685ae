"""paged_append of queries alone and of keys and values alone: tensors without heads."""
import pytest
import torch

import jero_hip as J

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 5])
@pytest.mark.parametrize("kv_type", [torch.float32, torch.float16])
def test_no_heads(dev, T, kv_type):
    g = torch.Generator(device=dev).manual_seed(T)
    H, KV, D, n = 4, 2, 64, 16
    q, k, v = (torch.randn((T, h, D), generator=g, device=dev) for h in (H, KV, KV))
    pos, slots = torch.arange(T, dtype=torch.int32, device=dev) + 3, torch.arange(T, device=dev) * 2
    rope = J.Rope(D, 1e4)
    pools = [torch.zeros((n, KV, D), dtype=kv_type, device=dev) for _ in range(2)]
    out = torch.zeros_like(q)
    J.paged_append(*pools, out, q, k, v, pos, slots, rope)
    # queries alone
    none, empty = torch.zeros((T, 0, D), device=dev), torch.zeros((n, 0, D), dtype=kv_type, device=dev)
    alone = torch.zeros_like(q)
    J.paged_append(empty, empty, alone, q, none, none, pos, slots, rope)
    # keys and values alone
    more = [torch.zeros_like(p) for p in pools]
    J.paged_append(*more, none.clone(), none, k, v, pos, slots, rope)
    torch.cuda.synchronize()
    assert torch.equal(alone, out) and torch.equal(more[0], pools[0]) and torch.equal(more[1], pools[1])
    with pytest.raises(J.K3Error):
        J.paged_append(empty, empty, none.clone(), none, none, none, pos, slots, rope)
