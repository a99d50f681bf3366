"""The serving operators on CPU tensors: what is refused, and when."""
import pytest
import torch

from recsdk_b200.inference import KVCacheConfig, KVCacheManager
from recsdk_b200.ops import sampling as S
from recsdk_b200.ops import softmax_attention as SA


def test_recommend_refuses_before_the_cache_is_touched():
    from recsdk_b200.models.hstu import HSTU, HSTUConfig
    from recsdk_b200.models.hstu_inference import HSTURanker

    torch.manual_seed(0)
    cfg = HSTUConfig(num_layers=1, d_model=128, num_heads=2, head_dim=64, max_seq_len=256, num_time_buckets=16)
    model = HSTU(cfg, torch.nn.Identity(), "cpu", torch.float32).eval()
    ranker = HSTURanker(model, KVCacheManager.from_config(KVCacheConfig(
        num_layers=1, num_heads=2, head_dim=64, page_size=16, offload_chunksize=64, num_primary_cache_pages=32, num_buffer_pages=8,
        host_capacity_per_layer=1 << 20, max_batch_size=4, max_seq_len=256, dtype=torch.float32, device="cpu")))
    users, hist, cands = torch.tensor([1, 2, 3]), torch.tensor([10, 20, 5]), torch.tensor([6, 0, 4])
    x, u = torch.randn(45, 128) * 0.5, torch.tensor([0.3, 0.5, 0.9])
    for uniform, kw in ((u, dict(top_p=0.0)), (u, dict(temperature=-1.0)), (u, dict(top_k=torch.tensor([1, 2]))), (u, dict(min_p=2.0)),
                        (u[:2], {}), (u.double(), {})):
        with pytest.raises(ValueError):
            ranker.recommend(users, hist, cands, x, uniform, **kw)
        assert ranker.plan(users, hist).tolist() == [0, 0, 0] and not ranker.kv.gpu.cache.any()
    ids, _ = ranker.recommend(users, hist, cands, x, u)
    assert ids[1] == -1 and ids[0] >= 0 and ranker.plan(users, hist).tolist() == [10, 20, 5]


def test_parameters_are_checked_without_scores():
    u = torch.rand(3)
    S.check_parameters(3, u.device, u, 0.5, torch.tensor([1, 2, 3]), 0.9, 0.1)
    for a, kw in (((2, u.device, u), {}), ((3, torch.device("meta"), u), {}), ((3, u.device, u), dict(top_p=0.0)),
                  ((3, u.device, u), dict(top_k=torch.rand(3)))):
        with pytest.raises(ValueError):
            S.check_parameters(*a, **kw)


def test_append_refuses_what_does_not_exist():
    """Two requests of two pages each; a token past its request's pages must not land in the neighbour's."""
    g = torch.Generator().manual_seed(1)
    cache = torch.randn(5, 2, 16, 2, 64, generator=g)
    ids, ptr, table = torch.tensor([3, 0, 4, 1]), torch.tensor([0, 2, 4]), SA.rotary_table(64, 64)
    q, k, v = torch.randn(2, 4, 64, generator=g), torch.randn(2, 2, 64, generator=g), torch.randn(2, 2, 64, generator=g)
    add = lambda b, pos, ids=ids, **kw: SA.append_kv_rotary(q, k, v, cache, torch.tensor(b), torch.tensor(pos), ids, ptr, 16, table, **kw)  # noqa: E731
    before = cache.clone()
    for args, kw in ((([0, 0], [0, 32]), {}), (([1, 0], [31, 32]), {}), (([0, 1], [0, 64]), {}), (([0, 1], [-1, 0]), {}), (([0, 2], [0, 0]), {}),
                     (([0, -1], [0, 0]), {}), (([0, 0], [0, 16], torch.tensor([3, -1, 4, 1])), {}), (([0, 1], [0, 16], torch.tensor([3, 0, 4, 5])), {}),
                     (([0, 1], [0, 16], torch.tensor([3, 0, 4])), {}), (([0, 0], [0, 1]), dict(slots=torch.tensor([0, 40]))),
                     (([0, 0], [0, 1]), dict(slots=torch.tensor([0, -1])))):
        with pytest.raises(IndexError):
            add(*args, **kw)
        assert torch.equal(cache, before)
    # padding is not looked at
    out = torch.full_like(q, 7.0)
    add([0, 9], [3, 999], num_tokens=torch.tensor([1], dtype=torch.int32), out=out)
    assert (out[1] == 7.0).all() and torch.equal(cache[3, 1, 3], v[0])
    cache.copy_(before)
    for n in (0, -1):
        add([0, 0], [0, 1], num_tokens=torch.tensor([n], dtype=torch.int32), out=out)
        assert torch.equal(cache, before)


def test_attention_refuses_missing_pages_that_are_seen():
    g = torch.Generator().manual_seed(2)
    cache, off = torch.randn(6, 2, 16, 2, 64, generator=g), torch.tensor
    q = torch.randn(2, 4, 64, generator=g)
    ids, ptr = off([4, 1, 3, 0, 5]), off([0, 4, 5])
    attend = lambda ids, ptr=ptr, k=off([0, 60, 70]), **kw: SA.softmax_attention_paged(q, cache, off([0, 1, 2]), k, ids, ptr, 16, **kw)  # noqa: E731
    want = attend(ids)
    for bad in (-1, 6, 10 ** 9):
        for at in range(5):
            hurt = ids.clone()
            hurt[at] = bad
            with pytest.raises(IndexError):
                attend(hurt)
    with pytest.raises(IndexError):                                    # fewer pages than keys
        attend(ids, ptr=off([0, 3, 5]))
    with pytest.raises(IndexError):
        SA.softmax_attention_shared_prefix(q, cache, off([0, 1, 2]), off([0, 0, 10]), ids[4:], off([0, 0, 1]), off([0, 32]), off([4, -1]),
                                           off([0, 2]), 16)
    # what lies before the window and behind the sinks may be gone, and there may be no page for it
    window = attend(ids, window=12, num_sinks=2)
    for bad in (-1, 6, 10 ** 9):
        hurt = ids.clone()
        hurt[1] = hurt[2] = bad
        assert torch.equal(attend(hurt, window=12, num_sinks=2), window)
    assert torch.equal(attend(torch.cat([ids, off([-3])]), ptr=off([0, 4, 6])), want)       # more pages than keys


def test_manager_wants_all_new_tokens():
    m = KVCacheManager.from_config(KVCacheConfig(
        num_layers=1, num_heads=2, head_dim=64, page_size=16, offload_chunksize=64, num_primary_cache_pages=32, num_buffer_pages=8,
        host_capacity_per_layer=1 << 20, max_batch_size=4, max_seq_len=512, dtype=torch.float32, device="cpu"))
    md = m.gpu.allocate(torch.tensor([3, 9]), torch.tensor([20, 33], dtype=torch.int32), torch.zeros(2, dtype=torch.int32))
    q, k, table = torch.randn(53, 4, 64), torch.randn(53, 2, 64), SA.rotary_table(512, 64)
    for n in (0, 20, 52):
        with pytest.raises(ValueError, match="all 53 new tokens"):
            m.gpu.append_kvcache_rotary(0, q[:n], k[:n], k[:n], md, table)
    assert not m.gpu.cache.any()
    m.gpu.append_kvcache_rotary(0, q, k, k, md, table)


def test_offsets_past_32_bits():
    g = torch.Generator().manual_seed(3)
    cache, off = torch.randn(4, 2, 16, 2, 64, generator=g), torch.tensor
    q = torch.randn(2, 4, 64, generator=g)
    for k in (off([0, 30, 62]), off([0, 30, 62]) + (1 << 31) - 40, off([0, 30, 62]) + (1 << 40)):
        o = SA.softmax_attention_paged(q, cache, off([0, 1, 2]), k, off([3, 1, 2, 0]), off([0, 2, 4]), 16)
        want = o if k[0] == 0 else want
        assert torch.equal(o, want)
    q, k = torch.randn(1, 4, 64), torch.randn(1, 2, 64)
    with pytest.raises(IndexError):
        SA.append_kv_rotary(q, k, k, cache, off([0]), off([(1 << 32) + 3]), off([3, 1]), off([0, 2]), 16, SA.rotary_table(32, 64))
