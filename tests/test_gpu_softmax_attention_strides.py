"""Queries, keys and values as slices of other tensors, and numbers past 32 bits: the results are those of contiguous tensors and of
the same lengths, bit for bit."""
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


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [48, 128])
@pytest.mark.parametrize("new,keys", [([1, 1, 1], [70, 300, 9]), ([150, 1, 300], [150, 700, 333])])
def test_slices_of_many_tokens(new, keys, page, D):
    """A projection's slice, rows with padding behind them, every other token, one token for all, heads that are not adjacent."""
    g = torch.Generator(device=DEV).manual_seed(page + D)
    H, Hkv, T = 4, 2, sum(new)
    cache, ids, ptr = _cache(keys, page, Hkv, D, g)
    kw = dict(q_offsets=_off(new), k_offsets=_off(keys), page_ids=ids, page_indptr=ptr, page_size=page, window=200, num_sinks=3)
    base = torch.randn(2 * T, (H + 2 * Hkv) * D + 8, generator=g, device=DEV).bfloat16()
    slices = [base[:T, : (H + 2 * Hkv) * D].contiguous()[:, 2 * D:(2 + H) * D].unflatten(1, (H, D)),      # stride 8 D, a head's offset
              base[:T, : H * D].unflatten(1, (H, D)), base[::2, : H * D].unflatten(1, (H, D)),            # odd multiples of 16 bytes
              base[:1, : H * D].unflatten(1, (H, D)).expand(T, H, D),
              base.flatten()[: (T + H) * D].as_strided((T, H, D), (D, D, 1)),                             # tokens overlap
              base[:T, : 2 * H * D].unflatten(1, (H, 2 * D))[..., :D], base[:T, 1:1 + H * D].unflatten(1, (H, D))]
    for q in slices:
        want, want_lse = SA.softmax_attention_paged(q.clone(memory_format=torch.contiguous_format), cache, return_lse=True, **kw)
        got, lse = SA.softmax_attention_paged(q, cache, return_lse=True, **kw)
        assert torch.equal(got, want) and torch.equal(lse, want_lse)
        ref, _ = SA.softmax_attention_ref(q, cache, kw["q_offsets"], kw["k_offsets"], ids, ptr, page, window=200, num_sinks=3, dtype=torch.float64)
        mag = cache.clone()
        mag[:, 1] = mag[:, 1].abs()
        avg, _ = SA.softmax_attention_ref(q, mag, kw["q_offsets"], kw["k_offsets"], ids, ptr, page, window=200, num_sinks=3, dtype=torch.float64)
        # half a step of the weights and of the result, 2^-12 for scores that are fp32 sums of sum |q_i k_i| * scale <= 8 in 128 terms
        assert ((got.double() - ref).abs() <= 2.0 ** -8 * (avg + ref.abs()) + 2.0 ** -12 * avg).all()
    _lib.check_status()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,Hkv,D,R", [(1, 4, 2, 64, 64), (3001, 32, 8, 128, 64), (777, 5, 1, 64, 16)])
def test_queries_turned_in_place(T, H, Hkv, D, R, interleaved):
    """The result goes where the queries are, a slice of the projection that keys and values are slices of, too."""
    g = torch.Generator(device=DEV).manual_seed(T)
    cache, ids, ptr = _cache([T], 16, Hkv, D, g)
    qkv = torch.randn(T, (H + 2 * Hkv) * D, generator=g, device=DEV).bfloat16()
    q, k, v = (x.unflatten(1, (-1, D)) for x in qkv.split([H * D, Hkv * D, Hkv * D], dim=1))
    rest = qkv[:, H * D:].clone()
    zero, pos = torch.zeros(T, dtype=torch.int32, device=DEV), torch.arange(T, dtype=torch.int32, device=DEV)
    table = SA.rotary_table(T, R, device=DEV)
    c1, c2 = cache.clone(), cache.clone()
    want = SA.append_kv_rotary(q, k, v, c1, zero, pos, ids, ptr, 16, table, interleaved=interleaved)
    got = SA.append_kv_rotary(q, k, v, c2, zero, pos, ids, ptr, 16, table, interleaved=interleaved, out=q)
    assert got is q and torch.equal(q, want) and torch.equal(c1, c2) and torch.equal(qkv[:, H * D:], rest)
    _lib.check_status()


def test_the_launch_counter_counts_every_kernel():
    """Against the nodes of a captured graph, which are the call's kernels."""
    import ctypes

    rt = ctypes.CDLL("libcudart.so.12")
    g = torch.Generator(device=DEV).manual_seed(1)
    cache, ids, ptr = _cache([100, 100], 16, 2, 64, g)
    two = (_off([100, 100]), ids, ptr)

    def count(call):
        call()
        graph = torch.cuda.CUDAGraph(keep_graph=True)
        with torch.cuda.graph(graph):
            before = _lib.launch_count
            call()
            counted = _lib.launch_count - before
        n = ctypes.c_size_t(0)
        assert rt.cudaGraphGetNodes(ctypes.c_void_p(graph.raw_cuda_graph()), None, ctypes.byref(n)) == 0
        assert counted == n.value
        return counted

    seen = set()
    for new in (1, 12, 90):                                            # by rows; prefix by tiles and own keys by rows; all by tiles
        q = torch.randn(2 * new, 4, 64, generator=g, device=DEV).bfloat16()
        qo, one, go = _off([new, new]), _off([100]), _off([2])
        p_ids, p_ptr = ids[:7].contiguous(), _off([7])
        seen.add(count(lambda: SA.softmax_attention_paged(q, cache, qo, *two, 16)))
        seen.add(count(lambda: SA.softmax_attention_shared_prefix(q, cache, qo, *two, one, p_ids, p_ptr, 16, group_offsets=go)))
    assert seen == {2, 3, 4}


@pytest.mark.parametrize("new", [1, 100])
def test_page_lists_that_begin_nowhere(new):
    """Page tables whose ends are out of range: the pages are missing, reported and read as zeros, as the tokens are left out."""
    g = torch.Generator(device=DEV).manual_seed(3)
    cache, ids, ptr = _cache([300, 300], 16, 2, 64, g)
    q = torch.randn(2 * new, 4, 64, generator=g, device=DEV).bfloat16()
    k = torch.randn(2 * new, 2, 64, generator=g, device=DEV).bfloat16()
    want = SA.softmax_attention_paged(q, cache, _off([new, new]), _off([300, 300]), ids, ptr, 16)
    b = torch.arange(2, device=DEV).repeat_interleave(new)
    pos, table = torch.arange(300 - new, 300, device=DEV).repeat(2), SA.rotary_table(300, 64, device=DEV)
    for begin in ((1 << 31) - 1, ids.numel(), ids.numel() + 1):
        hurt = torch.stack([ptr[0], ptr[1], torch.tensor(begin, dtype=torch.int32, device=DEV)])       # request 1 ends nowhere: all there
        assert torch.equal(SA.softmax_attention_paged(q, cache, _off([new, new]), _off([300, 300]), ids, hurt, 16), want)
        hurt = torch.stack([torch.tensor(begin, dtype=torch.int32, device=DEV), ptr[1], ptr[2]])       # request 0 begins nowhere
        got = SA.softmax_attention_paged(q, cache, _off([new, new]), _off([300, 300]), ids, hurt, 16)
        with pytest.raises(_lib.KernelStatusError, match="bounds"):
            _lib.check_status()
        assert (got[:new] == 0).all() and torch.equal(got[new:], want[new:])
        c = cache.clone()
        SA.append_kv_rotary(q, k, k, c, b, pos, ids, hurt, 16, table)
        with pytest.raises(_lib.KernelStatusError, match="bounds"):
            _lib.check_status()
        assert torch.equal(c[ids[:19].long()], cache[ids[:19].long()]) and not torch.equal(c, cache)


@pytest.mark.parametrize("new", [1, 100])
def test_offsets_past_32_bits(new):
    """Many requests that share pages have more keys together than 32 bits count; lengths are differences."""
    g = torch.Generator(device=DEV).manual_seed(new)
    keys = [300, 150, 200]
    cache, ids, ptr = _cache(keys, 16, 2, 64, g)
    q = torch.randn(3 * new, 4, 64, generator=g, device=DEV).bfloat16()
    qo, ko = _off([new] * 3), _off(keys).long()
    want = SA.softmax_attention_paged(q, cache, qo, ko, ids, ptr, 16)
    for base in ((1 << 31) - 310, (1 << 32) - 400, 1 << 40):
        assert torch.equal(SA.softmax_attention_paged(q, cache, qo, ko + base, ids, ptr, 16), want)
    pre = (ids[:7].contiguous(), _off([7]), 16)
    want = SA.softmax_attention_shared_prefix(q, cache, qo, ko, ids, ptr, _off([100]).long(), *pre)
    assert torch.equal(SA.softmax_attention_shared_prefix(q, cache, qo, ko, ids, ptr, _off([100]).long() + (1 << 31) - 50, *pre), want)
    _lib.check_status()


@pytest.mark.parametrize("far", [(1 << 32) + 3, -(1 << 32) + 3, (1 << 31) + 3, 1 << 40])
def test_indices_past_32_bits_do_not_exist(far):
    """They are reported like any other that does not exist, not taken for what their low bits say."""
    g = torch.Generator(device=DEV).manual_seed(2)
    cache, ids, ptr = _cache([40, 40], 16, 2, 64, g)
    q, k, v = (torch.randn(2, h, 64, generator=g, device=DEV).bfloat16() for h in (4, 2, 2))
    b, pos, table = torch.tensor([0, 1], device=DEV), torch.tensor([5, 6], device=DEV), SA.rotary_table(64, 64, device=DEV)
    kw = dict(batch_indices=b, positions=pos, page_ids=ids.long(), page_indptr=ptr.long(), slots=pos)
    for name in kw:
        if name == "page_indptr":
            continue
        hurt = dict(kw)
        hurt[name] = kw[name].clone()
        hurt[name][0] = far
        c = cache.clone()
        SA.append_kv_rotary(q, k, v, c, page_size=16, table=table, **hurt)
        with pytest.raises(_lib.KernelStatusError, match="bounds"):
            _lib.check_status()
        assert torch.equal(c[ids[0].long()], cache[ids[0].long()]) and not torch.equal(c, cache)
    hurt = ids.long()
    hurt[1] = far
    SA.softmax_attention_paged(q, cache, _off([1, 1]), _off([40, 40]), hurt, ptr, 16)
    with pytest.raises(_lib.KernelStatusError, match="bounds"):
        _lib.check_status()
