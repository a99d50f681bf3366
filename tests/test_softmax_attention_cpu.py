"""The serving operators on CPU tensors: definitions against independent ones, refusals, the manager's and the ranker's calls."""
import math

import pytest
import torch

from recsdk_b200.inference import KVCacheConfig, KVCacheManager
from recsdk_b200.ops import sampling as S
from recsdk_b200.ops import softmax_attention as SA


def _paged(lens, page, Hkv, D, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = [(x + page - 1) // page for x in lens]
    cache = torch.randn(sum(n) + 1, 2, page, Hkv, D, generator=g)
    ids = torch.randperm(sum(n) + 1, generator=g)[: sum(n)].int()
    ptr = torch.tensor([0] + torch.tensor(n).cumsum(0).tolist(), dtype=torch.int32)
    return cache, ids, ptr, g


def _off(lens):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32)


def test_attention_is_torch_softmax_attention():
    cache, ids, ptr, g = _paged([40, 23], 16, 2, 64)
    q = torch.randn(10, 4, 64, generator=g)
    for window, sinks in ((0, 0), (7, 2)):
        o, lse = SA.softmax_attention_paged(q, cache, _off([6, 4]), _off([40, 23]), ids, ptr, 16, window=window, num_sinks=sinks, return_lse=True)
        t = 0
        for b, (n, m) in enumerate(((6, 40), (4, 23))):
            c = cache[ids[ptr[b]:ptr[b + 1]].long()]
            k, v = (c[:, i].reshape(-1, 2, 64)[:m].repeat_interleave(2, dim=1).transpose(0, 1) for i in (0, 1))
            i, j = torch.arange(m - n, m)[:, None], torch.arange(m)[None, :]
            sees = (j <= i) & ((j > i - window) | (j < sinks) if window else torch.ones_like(j, dtype=torch.bool))
            want = torch.nn.functional.scaled_dot_product_attention(q[t:t + n].transpose(0, 1), k, v, attn_mask=sees)
            assert torch.allclose(o[t:t + n], want.transpose(0, 1), atol=1e-5)
            s = (q[t:t + n].transpose(0, 1) @ k.transpose(1, 2) / 8).masked_fill(~sees, -math.inf)
            assert torch.allclose(lse[t:t + n], torch.logsumexp(s, -1).t(), atol=1e-5)
            t += n


def test_shared_prefix_is_one_attention_over_both():
    own, prefix, page = [3, 5, 1], [32, 16], 16
    cache, ids, ptr, g = _paged(own + prefix, page, 2, 64)
    q = torch.randn(3, 2, 64, generator=g)
    oi, op, pi, pp = ids[:3], ptr[:4], ids[3:], ptr[3:] - ptr[3]
    o = SA.softmax_attention_shared_prefix(q, cache, _off([1] * 3), _off(own), oi, op, _off(prefix), pi, pp, page,
                                           group_offsets=torch.tensor([0, 2, 3]))
    # prefixes that end with their pages can simply stand in front of the own pages
    both = torch.cat([pi[:2], oi[:1], pi[:2], oi[1:2], pi[2:], oi[2:]])
    want = SA.softmax_attention_paged(q, cache, _off([1] * 3), _off([35, 37, 17]), both, torch.tensor([0, 3, 6, 8]), page)
    assert torch.allclose(o, want, atol=1e-5)


def test_rotation_is_by_relative_position():
    """Scores of turned queries and keys depend on the distance of their positions alone."""
    table = SA.rotary_table(5000, 64)
    assert torch.equal(table[0], torch.cat([torch.ones(32), torch.zeros(32)]))
    g = torch.Generator().manual_seed(1)
    q, k = torch.randn(1, 1, 64, generator=g), torch.randn(1, 1, 64, generator=g)
    for inter in (False, True):
        def turned(x, pos):
            cos, sin = table[torch.tensor([pos])][:, None].chunk(2, dim=-1)
            return SA._rotate_ref(x, cos, sin, inter)
        a = (turned(q, 17) * turned(k, 3)).sum()
        assert torch.allclose(a, (turned(q, 4014) * turned(k, 4000)).sum(), atol=1e-3)
        assert torch.allclose(turned(q, 4321).norm(), q.norm(), atol=1e-4)


def test_refusals_of_the_cache_operators():
    cache, ids, ptr, g = _paged([20], 16, 2, 64)
    q, k, v = torch.randn(1, 4, 64), torch.randn(1, 2, 64), torch.randn(1, 2, 64)
    one, z, table = _off([1]), torch.zeros(1, dtype=torch.int32), SA.rotary_table(32, 64)
    attn = lambda **kw: SA.softmax_attention_paged(**{**dict(q=q, kv_cache=cache, q_offsets=one, k_offsets=_off([20]), page_ids=ids,  # noqa: E731
                                                             page_indptr=ptr, page_size=16), **kw})
    add = lambda **kw: SA.append_kv_rotary(**{**dict(q=q, k=k, v=v, kv_cache=cache, batch_indices=z, positions=z, page_ids=ids,  # noqa: E731
                                                     page_indptr=ptr, page_size=16, table=table), **kw})
    attn()
    add()
    for kw in (dict(page_size=8), dict(kv_cache=cache.transpose(2, 3)), dict(kv_cache=cache[0]), dict(q=q[0]), dict(q=q[..., :32]),
               dict(q=torch.randn(1, 3, 64)), dict(q=q.half()), dict(q=torch.randn(1, 4, 64, requires_grad=True)), dict(window=-1),
               dict(num_sinks=-1), dict(scale=math.nan), dict(k_offsets=_off([20, 1])), dict(page_ids=ids.float()),
               dict(page_indptr=ptr[:1]), dict(q_offsets=one[None])):
        with pytest.raises(ValueError):
            attn(**kw)
    for kw in (dict(table=table.double()), dict(table=table[:, :24]), dict(table=SA.rotary_table(32, 80)), dict(k=torch.randn(1, 4, 64)),
               dict(v=torch.randn(2, 2, 64)), dict(positions=torch.zeros(2, dtype=torch.int32)), dict(batch_indices=z.float()),
               dict(out=torch.empty(1, 4, 32)), dict(num_tokens=torch.zeros(2, dtype=torch.int32)), dict(page_size=32)):
        with pytest.raises(ValueError):
            add(**kw)
    with pytest.raises(ValueError):
        SA.rotary_table(10, 24)
    pre = dict(prefix_offsets=_off([16, 4]), prefix_page_ids=ids, prefix_page_indptr=torch.tensor([0, 1, 2]), page_size=16)
    with pytest.raises(ValueError):                               # two groups, but nobody says whose
        SA.softmax_attention_shared_prefix(q, cache, one, _off([0]), ids, torch.tensor([0, 0]), **pre)
    with pytest.raises(ValueError):
        SA.softmax_attention_shared_prefix(q, cache, one, _off([0]), ids, torch.tensor([0, 0]), group_offsets=torch.tensor([0, 1]), **pre)


def test_sampling_against_plain_filters():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(40, 60, generator=g)
    u = torch.rand(40, generator=g)
    ids, lp = S.sample_scores(x, u, temperature=0.5, top_k=12, top_p=0.75, min_p=0.1)
    for r in range(40):
        p = torch.softmax(x[r].double() / 0.5, 0)
        keep = torch.zeros(60, dtype=torch.bool)
        order = p.argsort(descending=True)[:12]
        share = p[order] / p[order].sum()
        n = int((share.cumsum(0) < 0.75).sum()) + 1
        keep[order[:n]] = True
        keep &= p >= 0.1 * p.max()
        p = p * keep
        c = (p / p.sum()).cumsum(0)
        assert int(ids[r]) == int((c <= float(u[r])).sum())
        assert abs(float(lp[r]) - math.log(p[ids[r]] / p.sum())) < 1e-5
    assert S.sample_scores(torch.full((2, 3), -math.inf), u[:2])[0].tolist() == [-1, -1]
    assert S.sample_scores(torch.tensor([[1.0, 3, 3]]), u[:1], temperature=0.0)[0].tolist() == [1]
    assert S.sample_scores(x.reshape(-1), torch.rand(3), torch.tensor([0, 5, 5, 2400]))[0][1] == -1


def test_refusals_of_sampling():
    x, u = torch.randn(3, 5), torch.rand(3)
    S.sample_scores(x, u)
    for a, kw in (((x[0], u), {}), ((x, u), dict(offsets=torch.tensor([0, 5]))), ((x[0], u[:1]), dict(offsets=torch.tensor([0.0, 5.0]))),
                  ((x, u[:2]), {}), ((x, u.double()), {}), ((x.double(), u), {}), ((x, u), dict(temperature=-1.0)),
                  ((x, u), dict(temperature=math.inf)), ((x, u), dict(top_k=-1)), ((x, u), dict(top_p=0.0)), ((x, u), dict(top_p=1.5)),
                  ((x, u), dict(min_p=-0.1)), ((x, u), dict(min_p=math.nan)), ((x, u), dict(top_p=torch.rand(2))),
                  ((x, u), dict(top_k=torch.rand(3)))):
        with pytest.raises(ValueError):
            S.sample_scores(*a, **kw)


def test_manager_appends_turned_keys():
    m = KVCacheManager.from_config(KVCacheConfig(
        num_layers=2, num_heads=2, head_dim=64, page_size=16, offload_chunksize=64, num_primary_cache_pages=32, num_buffer_pages=8,
        host_capacity_per_layer=1 << 20, max_batch_size=4, max_seq_len=512, dtype=torch.float32, device="cpu"))
    users, lens = torch.tensor([3, 9]), torch.tensor([20, 33], dtype=torch.int32)
    md = m.gpu.allocate(users, lens, torch.zeros(2, dtype=torch.int32))
    g = torch.Generator().manual_seed(3)
    q, k, v = torch.randn(53, 4, 64, generator=g), torch.randn(53, 2, 64, generator=g), torch.randn(53, 2, 64, generator=g)
    table = SA.rotary_table(512, 64)
    got = m.gpu.append_kvcache_rotary(1, q, k, v, md, table)
    cos, sin = table[md.position.long()][:, None].chunk(2, dim=-1)
    assert torch.equal(got, SA._rotate_ref(q, cos, sin, False))
    kk, vv = m.gpu.get(md.kv_indices[md.kv_indptr[1]:md.kv_indptr[2]], md.kv_last_page_len[1], 1)
    assert torch.equal(kk, SA._rotate_ref(k, cos, sin, False)[20:]) and torch.equal(vv, v[20:])
    # the prompt's attention from the pages it was just written to
    o = SA.softmax_attention_paged(got, m.gpu.cache[1], md.new_history_offsets, md.total_history_offsets, md.kv_indices, md.kv_indptr, 16)
    want = torch.nn.functional.scaled_dot_product_attention(
        got[20:].transpose(0, 1), kk.repeat_interleave(2, 1).transpose(0, 1), vv.repeat_interleave(2, 1).transpose(0, 1), is_causal=True)
    assert torch.allclose(o[20:], want.transpose(0, 1), atol=1e-5)


def test_ranker_recommends_from_its_scores():
    from recsdk_b200.models.hstu import HSTU, HSTUConfig
    from recsdk_b200.models.hstu_inference import HSTURanker

    torch.manual_seed(0)
    cfg = HSTUConfig(num_layers=1, d_model=128, num_heads=2, head_dim=64, max_seq_len=256, num_time_buckets=16)
    model = HSTU(cfg, torch.nn.Identity(), "cpu", torch.float32).eval()
    make = lambda: HSTURanker(model, KVCacheManager.from_config(KVCacheConfig(  # noqa: E731
        num_layers=1, num_heads=2, head_dim=64, page_size=16, offload_chunksize=64, num_primary_cache_pages=32, num_buffer_pages=8,
        host_capacity_per_layer=1 << 20, max_batch_size=4, max_seq_len=256, dtype=torch.float32, device="cpu")))
    users, hist, cands = torch.tensor([1, 2, 3]), torch.tensor([10, 20, 5]), torch.tensor([6, 0, 4])
    x, u = torch.randn(45, 128) * 0.5, torch.tensor([0.3, 0.5, 0.9])
    scores = make().rank(users, hist, cands, x)
    ids, lp = make().recommend(users, hist, cands, x, u, temperature=0.5, top_p=0.9)
    want, want_lp = S.sample_scores(scores, u, torch.tensor([0, 6, 6, 10]), temperature=0.5, top_p=0.9)
    assert torch.equal(ids, want) and torch.equal(lp, want_lp) and ids[1] == -1


def test_slots_are_where_keys_go():
    cache, ids, ptr, g = _paged([20], 16, 2, 64)
    q, k, v = torch.randn(2, 4, 64, generator=g), torch.randn(2, 2, 64, generator=g), torch.randn(2, 2, 64, generator=g)
    table = SA.rotary_table(64, 64)
    z, pos = torch.zeros(2, dtype=torch.int32), torch.tensor([40, 41], dtype=torch.int32)
    SA.append_kv_rotary(q, k, v, cache, z, pos, ids, ptr, 16, table, slots=torch.tensor([15, 16]))
    cos, sin = table[pos.long()][:, None].chunk(2, dim=-1)
    turned = SA._rotate_ref(k, cos, sin, False)
    assert torch.equal(cache[ids[0].long(), 0, 15], turned[0]) and torch.equal(cache[ids[1].long(), 0, 0], turned[1])
    assert torch.equal(cache[ids[0].long(), 1, 15], v[0])
    with pytest.raises(ValueError):
        SA.append_kv_rotary(q, k, v, cache, z, pos, ids, ptr, 16, table, slots=torch.tensor([15]))


def test_sampling_refuses_what_wants_a_gradient():
    x, u = torch.randn(3, 5, requires_grad=True), torch.rand(3)
    with pytest.raises(ValueError, match="gradient"):
        S.sample_scores(x, u)
    with torch.no_grad():
        S.sample_scores(x, u)


def test_min_p_of_one_keeps_the_largest_only():
    x = torch.tensor([[0.0, -1e-30, 0.0, -1e-17, -1.0]])
    ids = {int(S.sample_scores(x, torch.tensor([v]), min_p=1.0)[0]) for v in (0.0, 0.3, 0.49, 0.51, 0.7, 0.99)}
    assert ids == {0, 2}
