"""The serving operators on CPU tensors: what is refused, and when."""
import pytest
import torch

from recsdk_b200.inference import KVCacheConfig, KVCacheManager
from recsdk_b200.ops import sampling as S


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
