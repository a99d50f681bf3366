"""Queries, keys and values as slices of other tensors: the results are those of contiguous ones, bit for bit."""
import pytest
import torch

from recsdk_b200.ops import _lib
from recsdk_b200.ops import softmax_attention as SA

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _off(lens):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=DEV)


def _cache(keys, page, Hkv, D, g):
    n = [(x + page - 1) // page for x in keys]
    cache = torch.randn(sum(n) + 1, 2, page, Hkv, D, generator=g, device=DEV).bfloat16()
    return cache, torch.randperm(sum(n) + 1, generator=g, device=DEV)[: sum(n)].int(), _off(n)


@pytest.mark.parametrize("dist", [256, 260, 1537, 8, 1])
def test_a_single_token_has_no_stride(dist):
    g = torch.Generator(device=DEV).manual_seed(dist)
    cache, ids, ptr = _cache([40], 16, 2, 64, g)
    base = torch.randn(6000, generator=g, device=DEV).bfloat16()
    q, k, v = (base[a:].as_strided((1, h, 64), (dist, 64, 1)) for a, h in ((0, 4), (2048, 2), (4096, 2)))
    kw = dict(q_offsets=_off([1]), k_offsets=_off([40]), page_ids=ids, page_indptr=ptr, page_size=16)
    assert torch.equal(SA.softmax_attention_paged(q, cache, **kw), SA.softmax_attention_paged(q.clone(), cache, **kw))
    zero, table = torch.zeros(1, dtype=torch.int32, device=DEV), SA.rotary_table(64, 64, device=DEV)
    c1, c2 = cache.clone(), cache.clone()
    out = torch.zeros(3000, dtype=torch.bfloat16, device=DEV).as_strided((1, 4, 64), (dist, 64, 1))
    got = SA.append_kv_rotary(q, k, v, c1, zero, zero + 33, ids, ptr, 16, table, out=out)
    want = SA.append_kv_rotary(q.clone(), k.clone(), v.clone(), c2, zero, zero + 33, ids, ptr, 16, table)
    assert got is out and torch.equal(got, want) and torch.equal(c1, c2) and not torch.equal(c1, cache)
    _lib.check_status()
