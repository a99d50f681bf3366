"""Rotary append and softmax attention over the paged cache against their statements in 64 bits.

Bounds.  ``h = eps / 2`` is the largest relative error of one rounding to the inputs' type.  A weight is rounded once for
its product with V: ``h * A`` with ``A`` the attention's own average of ``|v|``; the result once: ``h * |o|``.  A score is
an fp32 sum of ``D <= 128`` exact products, each addition off by at most 2^-23 of the partial sum (truncation): with
``sum |q_i k_i| * scale <= 8`` for the inputs here that is 128 * 2^-23 * 8 = 2^-13, in the weights' numerator and their sum
together ``2^-12 * A``; the same 2^-12 bounds the lse (fp32 log and exp2.approx, 2^-22, stay far below)."""
import math

import pytest
import torch

from recsdk_b200.ops import _lib
from recsdk_b200.ops import softmax_attention as SA

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _cache(lens, page, Hkv, D, dtype, g, stale=None):
    """A cache that holds sequences of ``lens`` keys in shuffled pages; the slots in between hold ``stale``."""
    n = [(x + page - 1) // page for x in lens]
    pages = sum(n) + 2
    c = torch.randn(pages, 2, page, Hkv, D, generator=g, device=DEV)
    perm = torch.randperm(pages, generator=g, device=DEV).int()
    ids = perm[: sum(n)].contiguous()
    ptr = torch.tensor([0] + torch.tensor(n).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
    if stale is not None:
        c[perm[sum(n):].long()] = stale
        at = 0
        for x, k in zip(lens, n):
            if x % page:
                c[int(ids[at + k - 1]), :, x % page:] = stale
            at += k
    return c.to(dtype), ids, ptr


def _off(lens):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=DEV)


def _check(got, lse, ref, ref_lse, avg, dtype):
    h = torch.finfo(dtype).eps / 2
    assert torch.isfinite(got).all()
    tol = h * avg + h * ref.abs() + 2.0 ** -12 * avg
    err = (got.double() - ref).abs()
    assert (err <= tol).all(), "worst %g at %s" % ((err - tol).max().item(), (err - tol).argmax().item())
    none = ref_lse == -math.inf
    assert torch.equal(lse == -math.inf, none)
    assert (got[none] == 0).all()
    assert ((lse.double() - ref_lse)[~none].abs() <= 2.0 ** -12 + 2.0 ** -22 * ref_lse[~none].abs()).all()


def _run(new, keys, H, Hkv, D, page, dtype, window=0, sinks=0, seed=0, stale=math.nan, scale=None):
    g = torch.Generator(device=DEV).manual_seed(seed)
    cache, ids, ptr = _cache(keys, page, Hkv, D, dtype, g, stale)
    q = torch.randn(sum(new), H, D, generator=g, device=DEV).to(dtype)
    qo, ko = _off(new), _off(keys)
    got, lse = SA.softmax_attention_paged(q, cache, qo, ko, ids, ptr, page, scale=scale, window=window, num_sinks=sinks, return_lse=True)
    kw = dict(scale=scale, window=window, num_sinks=sinks, dtype=torch.float64)
    ref, ref_lse = SA.softmax_attention_ref(q, cache, qo, ko, ids, ptr, page, **kw)
    mag = cache.clone()
    mag[:, 1] = mag[:, 1].abs()
    avg, _ = SA.softmax_attention_ref(q, mag, qo, ko, ids, ptr, page, **kw)
    torch.cuda.synchronize()
    _lib.check_status()
    _check(got, lse, ref, ref_lse, avg, dtype)


@pytest.mark.parametrize("H,Hkv,D", [(8, 8, 64), (8, 2, 128), (7, 1, 64), (3, 3, 128), (40, 2, 64), (12, 4, 128)])
@pytest.mark.parametrize("page", [16, 48, 64, 128])
def test_single_tokens(H, Hkv, D, page):
    _run([1] * 7, [1, 2, 31, 33, 257, 1000, 130], H, Hkv, D, page, torch.bfloat16, seed=H + page)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 3), (33, 0), (64, 4), (100, 65), (5000, 7), (200, 5000)])
@pytest.mark.parametrize("new,keys", [([1, 1, 1], [700, 5, 130]), ([3, 0, 17, 5], [3, 9, 400, 505]), ([130, 300], [130, 777])])
def test_window_and_sinks(dtype, window, sinks, new, keys):
    _run(new, keys, 4, 2, 64, 32, dtype, window, sinks, seed=window)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hkv", [(4, 4), (8, 2), (7, 1), (16, 1)])
def test_prompts(D, H, Hkv):
    _run([257, 1, 64, 511], [257, 900, 64, 600], H, Hkv, D, 64, torch.bfloat16, seed=D + H)
    _run([257, 1, 64, 511], [257, 900, 64, 600], H, Hkv, D, 16, torch.float16, 100, 5, seed=D + H)


def test_long_history_one_request():
    """One request, every CTA holds a piece of it."""
    for D, H, Hkv in ((128, 8, 1), (64, 2, 2)):
        _run([1], [70001], H, Hkv, D, 64, torch.bfloat16, seed=3)
        _run([2], [70001], H, Hkv, D, 64, torch.bfloat16, 30000, 1000, seed=4)
        _run([300], [9001], H, Hkv, D, 64, torch.bfloat16, seed=5)


def test_rows_that_see_nothing_and_empty_requests():
    # more queries than keys: the first ones stand before the first key
    _run([5, 0, 3, 1], [2, 7, 0, 0], 4, 2, 64, 16, torch.bfloat16)
    _run([200, 0, 150, 1], [2, 7, 0, 300], 4, 2, 128, 16, torch.float16, 3, 1)


@pytest.mark.parametrize("scale", [0.0, -0.3, 0.01])
def test_other_scales(scale):
    _run([1, 140], [50, 300], 4, 2, 64, 32, torch.bfloat16, seed=9, scale=scale)


def test_strided_queries_and_gone_pages():
    """q is a slice of a projection; the pages before the window are no longer the request's."""
    g = torch.Generator(device=DEV).manual_seed(2)
    H, D, page = 4, 64, 16
    cache, ids, ptr = _cache([500, 333], page, H, D, torch.bfloat16, g)
    qkv = torch.randn(2, 3 * H * D, generator=g, device=DEV).bfloat16()
    q = qkv[:, H * D:2 * H * D].unflatten(1, (H, D))
    args = (_off([1, 1]), _off([500, 333]))
    want = SA.softmax_attention_paged(q.contiguous(), cache, *args, ids, ptr, page, window=40, num_sinks=2)
    gone = ids.clone()
    gone[2:28] = -7
    hurt = cache.clone()
    hurt[ids[2:28].long()] = math.nan
    got = SA.softmax_attention_paged(q, hurt, *args, gone, ptr, page, window=40, num_sinks=2)
    torch.cuda.synchronize()
    _lib.check_status()
    assert torch.equal(got, want)


def test_missing_page_is_reported():
    g = torch.Generator(device=DEV).manual_seed(2)
    cache, ids, ptr = _cache([100], 16, 2, 64, torch.bfloat16, g)
    q = torch.randn(1, 2, 64, generator=g, device=DEV).bfloat16()
    for bad in (-1, cache.shape[0]):
        ids2 = ids.clone()
        ids2[3] = bad
        out = SA.softmax_attention_paged(q, cache, _off([1]), _off([100]), ids2, ptr, 16)
        with pytest.raises(_lib.KernelStatusError):
            _lib.check_status()
        assert torch.isfinite(out).all()
    _lib.check_status()


def _run_prefix(new, own, prefix, groups, H, Hkv, D, page, dtype, seed=0, one=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    cache, ids, ptr = _cache(own + prefix, page, Hkv, D, dtype, g, math.nan)
    nb = len(own)
    oi, op = ids[: int(ptr[nb])].contiguous(), ptr[: nb + 1].contiguous()
    pi, pp = ids[int(ptr[nb]):].contiguous(), (ptr[nb:] - ptr[nb]).contiguous()
    q = torch.randn(sum(new), H, D, generator=g, device=DEV).to(dtype)
    qo, ko, po = _off(new), _off(own), _off(prefix)
    go = None if one else torch.tensor(groups, dtype=torch.int32, device=DEV)
    got, lse = SA.softmax_attention_shared_prefix(q, cache, qo, ko, oi, op, po, pi, pp, page, group_offsets=go, return_lse=True)
    kw = dict(prefix_offsets=po, prefix_page_ids=pi, prefix_page_indptr=pp, group_offsets=go, dtype=torch.float64)
    ref, ref_lse = SA.softmax_attention_ref(q, cache, qo, ko, oi, op, page, **kw)
    mag = cache.clone()
    mag[:, 1] = mag[:, 1].abs()
    avg, _ = SA.softmax_attention_ref(q, mag, qo, ko, oi, op, page, **kw)
    torch.cuda.synchronize()
    _lib.check_status()
    _check(got, lse, ref, ref_lse, avg, dtype)


@pytest.mark.parametrize("H,Hkv,D,dtype", [(8, 8, 64, torch.bfloat16), (8, 2, 128, torch.float16), (7, 1, 128, torch.bfloat16)])
def test_shared_prefix(H, Hkv, D, dtype):
    _run_prefix([1] * 6, [1, 5, 40, 1, 2, 300], [777, 64], [0, 4, 6], H, Hkv, D, 32, dtype)
    _run_prefix([1] * 40, [3] * 40, [3001], [0, 40], H, Hkv, D, 64, dtype, one=True)
    _run_prefix([4, 1, 0, 9] * 8, [4, 0, 3, 20] * 8, [129, 0, 1000], [0, 9, 9, 32], H, Hkv, D, 16, dtype)
    # the first two requests and the last one are in no group
    _run_prefix([2, 3, 1, 1, 30], [2, 3, 1, 0, 70], [100, 33], [2, 3, 4], H, Hkv, D, 16, dtype)
    _run_prefix([150, 200], [150, 250], [500], [0, 2], H, Hkv, D, 64, dtype)


def test_results_do_not_depend_on_the_run():
    g = torch.Generator(device=DEV).manual_seed(4)
    cache, ids, ptr = _cache([9000, 40, 3000], 64, 2, 128, torch.bfloat16, g)
    q = torch.randn(3, 8, 128, generator=g, device=DEV).bfloat16()
    outs = [SA.softmax_attention_paged(q, cache, _off([1, 1, 1]), _off([9000, 40, 3000]), ids, ptr, 64) for _ in range(5)]
    assert all(torch.equal(outs[0], o) for o in outs[1:])


# ----------------------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("H,Hkv,D,R,page", [(8, 8, 64, 64, 32), (32, 8, 128, 64, 64), (5, 1, 128, 128, 16), (3, 3, 64, 16, 7), (2, 1, 256, 96, 1)])
def test_append(dtype, interleaved, H, Hkv, D, R, page):
    g = torch.Generator(device=DEV).manual_seed(D + R)
    keys, new = [70, 1, 200, 33], [3, 1, 150, 0]
    cache, ids, ptr = _cache(keys, page, Hkv, D, dtype, g)
    qkv = torch.randn(sum(new), (H + 2 * Hkv) * D, generator=g, device=DEV).to(dtype)
    q, k, v = (x.unflatten(1, (-1, D)) for x in qkv.split([H * D, Hkv * D, Hkv * D], dim=1))
    b = torch.repeat_interleave(torch.arange(4), torch.tensor(new)).int().to(DEV)
    pos = torch.cat([torch.arange(n - m, n) for n, m in zip(keys, new)]).int().to(DEV)
    table = SA.rotary_table(201, R, device=DEV)
    before = cache.clone()
    got = SA.append_kv_rotary(q, k, v, cache, b, pos, ids, ptr, page, table, interleaved=interleaved)
    torch.cuda.synchronize()
    _lib.check_status()
    cos, sin = (x[:, None, :] for x in table.double()[pos.long()].chunk(2, dim=1))
    h = torch.finfo(dtype).eps / 2

    def near(x, y, src):
        # one rounding to 16 bits of an fp32 sum of two products (3 roundings of 2^-24 of their magnitudes, at most 2 max|x|)
        tiny = torch.finfo(dtype).tiny * h
        assert ((x.double() - y).abs() <= h * y.abs() + 2.0 ** -21 * src.double().abs().amax() + tiny).all()

    near(got, SA._rotate_ref(q.double(), cos, sin, interleaved), q)
    at = ids.long()[ptr.long()[b.long()] + pos.long() // page]
    near(cache[at, 0, pos.long() % page], SA._rotate_ref(k.double(), cos, sin, interleaved), k)
    assert torch.equal(cache[at, 1, pos.long() % page], v)
    cache[at, :, pos.long() % page] = before[at, :, pos.long() % page]
    assert torch.equal(cache, before)                                 # nothing else was written


def test_append_padding_in_place_and_far_positions():
    g = torch.Generator(device=DEV).manual_seed(1)
    cache, ids, ptr = _cache([40], 16, 2, 64, torch.bfloat16, g)
    q, k, v = (torch.randn(6, 2, 64, generator=g, device=DEV).bfloat16() for _ in range(3))
    pos = torch.tensor([30, 31, 32, 0, 0, 0], dtype=torch.int32, device=DEV)
    b = torch.zeros(6, dtype=torch.int32, device=DEV)
    table = SA.rotary_table(64, 64, device=DEV)
    full = SA.append_kv_rotary(q[:3], k[:3], v[:3], cache.clone(), b[:3], pos[:3], ids, ptr, 16, table)
    c1, q1 = cache.clone(), q.clone()
    n = torch.tensor([3], dtype=torch.int32, device=DEV)
    out = SA.append_kv_rotary(q1, k, v, c1, b, pos, ids, ptr, 16, table, num_tokens=n, out=q1)
    assert out is q1 and torch.equal(q1[:3], full) and torch.equal(q1[3:], q[3:])
    assert torch.equal(c1[ids[0].long()], cache[ids[0].long()])      # position 0 was not touched by the padding
    _lib.check_status()
    # a position beyond the table or the pages is left out and reported; the others are done
    for bad in (64, -1, 63):
        p2 = pos.clone()
        p2[1] = bad
        c2 = cache.clone()
        got = SA.append_kv_rotary(q[:3], k[:3], v[:3], c2, b[:3], p2[:3], ids, ptr, 16, table)
        with pytest.raises(_lib.KernelStatusError):
            _lib.check_status()
        assert torch.equal(got[0], full[0]) and torch.equal(got[2], full[2])


def test_one_step_in_a_graph():
    """Append, attend: captured once, replayed for other lengths, against the same calls made one by one."""
    g = torch.Generator(device=DEV).manual_seed(8)
    H, Hkv, D, page = 8, 2, 64, 16
    cache, ids, ptr = _cache([300, 200], page, Hkv, D, torch.bfloat16, g)
    q = torch.randn(2, H, D, generator=g, device=DEV).bfloat16()
    k, v = (torch.randn(2, Hkv, D, generator=g, device=DEV).bfloat16() for _ in range(2))
    table = SA.rotary_table(300, D, device=DEV)
    b = torch.arange(2, dtype=torch.int32, device=DEV)
    lens = torch.tensor([100, 17], dtype=torch.int32, device=DEV)
    qo = _off([1, 1])
    pos, ko = torch.zeros(2, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)

    def step():
        qr = SA.append_kv_rotary(q, k, v, cache, b, pos, ids, ptr, page, table)
        return SA.softmax_attention_paged(qr, cache, qo, ko, ids, ptr, page, window=64, num_sinks=4)

    def lengths(x):
        pos.copy_(x - 1)
        ko.copy_(torch.cat([torch.zeros_like(x[:1]), x.cumsum(0).int()]))

    lengths(lens)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for x in ([100, 17], [300, 1], [1, 200]):
        lengths(torch.tensor(x, dtype=torch.int32, device=DEV))
        graph.replay()
        got = out.clone()
        assert torch.equal(got, step())
    _lib.check_status()


def test_many_requests_and_wide_groups():
    g = torch.Generator().manual_seed(6)
    # more requests than threads that count them, some without tokens, some without keys
    new = torch.randint(0, 3, (3000,), generator=g).tolist()
    keys = [n + k for n, k in zip(new, torch.randint(0, 40, (3000,), generator=g).tolist())]
    _run(new, keys, 4, 2, 64, 16, torch.bfloat16, seed=6)
    new = torch.randint(0, 90, (700,), generator=g).tolist()
    keys = [n + k for n, k in zip(new, torch.randint(0, 100, (700,), generator=g).tolist())]
    _run(new, keys, 2, 2, 64, 32, torch.float16, 50, 3, seed=7)
    # 160 and 64 query heads on one key head
    _run([1, 3], [70, 500], 160, 1, 64, 16, torch.bfloat16, seed=8)
    _run([5, 33], [70, 300], 64, 1, 128, 16, torch.bfloat16, seed=9)


def test_long_offsets_and_uneven_lengths():
    """One very long request among short ones; the other offset type."""
    _run([1] * 9, [40001, 1, 2, 3, 64, 65, 100, 7, 9], 8, 2, 128, 64, torch.float16, seed=1)
    _run([150] + [1] * 5, [9000, 3, 2, 700, 1, 65], 4, 1, 64, 64, torch.bfloat16, 0, 0, seed=2)
    g = torch.Generator(device=DEV).manual_seed(2)
    cache, ids, ptr = _cache([100, 70], 16, 2, 64, torch.bfloat16, g)
    q = torch.randn(2, 4, 64, generator=g, device=DEV).bfloat16()
    a = SA.softmax_attention_paged(q, cache, _off([1, 1]), _off([100, 70]), ids, ptr, 16)
    b = SA.softmax_attention_paged(q, cache, _off([1, 1]).long(), _off([100, 70]).long(), ids.long(), ptr.long(), 16)
    assert torch.equal(a, b)


@pytest.mark.parametrize("new", [1, 200])
def test_a_broken_query_stays_alone(new):
    g = torch.Generator(device=DEV).manual_seed(3)
    cache, ids, ptr = _cache([300, 400], 16, 2, 64, torch.bfloat16, g)
    q = torch.randn(2 * new, 4, 64, generator=g, device=DEV).bfloat16()
    args = (cache, _off([new, new]), _off([300, 400]), ids, ptr, 16)
    want = SA.softmax_attention_paged(q, *args)
    q[0, 1] = math.nan
    got = SA.softmax_attention_paged(q, *args)
    assert torch.isnan(got[0, 1]).all()
    got[0, 1] = want[0, 1]
    assert torch.equal(got, want)


def test_calls_on_two_streams():
    g = torch.Generator(device=DEV).manual_seed(5)
    cache, ids, ptr = _cache([5000, 60, 900], 64, 2, 128, torch.bfloat16, g)
    few, many = torch.randn(3, 8, 128, generator=g, device=DEV).bfloat16(), torch.randn(300, 8, 128, generator=g, device=DEV).bfloat16()
    calls = [lambda: SA.softmax_attention_paged(few, cache, _off([1, 1, 1]), _off([5000, 60, 900]), ids, ptr, 64),
             lambda: SA.softmax_attention_paged(many, cache, _off([200, 50, 50]), _off([5000, 60, 900]), ids, ptr, 64, window=700)]
    want = [c() for c in calls]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(calls[i]())
    torch.cuda.synchronize()
    assert all(torch.equal(want[i], o) for i in (0, 1) for o in got[i])


def test_refusals_on_the_gpu():
    g = torch.Generator(device=DEV).manual_seed(2)
    cache, ids, ptr = _cache([20], 16, 2, 64, torch.bfloat16, g)
    q = torch.randn(1, 4, 64, generator=g, device=DEV).bfloat16()
    ok = dict(q=q, kv_cache=cache, q_offsets=_off([1]), k_offsets=_off([20]), page_ids=ids, page_indptr=ptr, page_size=16)
    SA.softmax_attention_paged(**ok)
    c32 = torch.zeros(3, 2, 16, 2, 32, dtype=torch.bfloat16, device=DEV)
    c24 = torch.zeros(3, 2, 24, 2, 64, dtype=torch.bfloat16, device=DEV)
    for kw in (dict(kv_cache=cache.float(), q=q.float()), dict(kv_cache=c32, q=q[..., :32]), dict(kv_cache=c24, page_size=24),
               dict(q_offsets=_off([1]).cpu()), dict(page_ids=ids.cpu()), dict(kv_cache=cache[:0]), dict(q=q.half())):
        with pytest.raises(ValueError):
            SA.softmax_attention_paged(**{**ok, **kw})


def test_decoding_with_beams():
    """Two users, three beams each: the prompt goes into shared pages, every step appends to the beams' own pages, attends
    behind the shared prefix and draws the next item; each call against its own statement on the same inputs."""
    from recsdk_b200.ops import sampling

    g = torch.Generator(device=DEV).manual_seed(12)
    H, Hkv, D, page, V, steps = 8, 2, 64, 16, 211, 20
    prompt, beams = [45, 30], 3
    emb = torch.randn(V, (H + 2 * Hkv) * D, generator=g, device=DEV).bfloat16()
    head = (torch.randn(V, H * D, generator=g, device=DEV) / 8).bfloat16()
    table = SA.rotary_table(100, D, device=DEV)
    cache = torch.full((20, 2, page, Hkv, D), math.nan, dtype=torch.bfloat16, device=DEV)
    split = lambda x: (t.unflatten(1, (-1, D)) for t in x.split([H * D, Hkv * D, Hkv * D], dim=1))  # noqa: E731
    # the prompts
    items = torch.randint(0, V, (75,), generator=g, device=DEV)
    b = torch.tensor([0] * 45 + [1] * 30, dtype=torch.int32, device=DEV)
    pos = torch.cat([torch.arange(45), torch.arange(30)]).int().to(DEV)
    p_ids, p_ptr = torch.tensor([7, 3, 11, 0, 9], dtype=torch.int32, device=DEV), torch.tensor([0, 3, 5], dtype=torch.int32, device=DEV)
    q, k, v = split(emb[items])
    q = SA.append_kv_rotary(q, k, v, cache, b, pos, p_ids, p_ptr, page, table)
    o = SA.softmax_attention_paged(q, cache, _off(prompt), _off(prompt), p_ids, p_ptr, page, window=32, num_sinks=4)
    want, _ = SA.softmax_attention_ref(q, cache, _off(prompt), _off(prompt), p_ids, p_ptr, page, window=32, num_sinks=4, dtype=torch.float64)
    assert (o.double() - want).abs().max() < 0.05
    # the beams
    n = 2 * beams
    own_ids = torch.tensor([1, 2, 4, 5, 6, 8, 10, 12, 13, 14, 15, 16], dtype=torch.int32, device=DEV)
    own_ptr, bi = torch.arange(0, 13, 2, dtype=torch.int32, device=DEV), torch.arange(n, dtype=torch.int32, device=DEV)
    groups = torch.tensor([0, beams, n], dtype=torch.int32, device=DEV)
    start = torch.tensor(prompt, dtype=torch.int32, device=DEV).repeat_interleave(beams)
    items = torch.randint(0, V, (n,), generator=g, device=DEV)
    for step in range(steps):
        q, k, v = split(emb[items])
        # positions count from the prompt, slots from the beam's own pages
        slots = torch.full_like(bi, step)
        before = k.clone()
        q0, q = q, SA.append_kv_rotary(q, k, v, cache, bi, start + step, own_ids, own_ptr, page, table, slots=slots)
        cos, sin = table[(start + step).long()][:, None].chunk(2, dim=-1)
        assert (q.double() - SA._rotate_ref(q0.double(), cos.double(), sin.double(), False)).abs().max() < 0.02
        at = own_ids.long()[own_ptr[:-1].long() + step // page]
        turned = SA._rotate_ref(before.double(), cos.double(), sin.double(), False)
        assert (cache[at, 0, step % page].double() - turned).abs().max() < 0.02 and torch.equal(cache[at, 1, step % page], v)
        kw = dict(group_offsets=groups)
        args = (q, cache, _off([1] * n), _off([step + 1] * n), own_ids, own_ptr)
        pre = (_off(prompt), p_ids, p_ptr)
        o = SA.softmax_attention_shared_prefix(*args, *pre, page, **kw)
        want, _ = SA.softmax_attention_ref(*args, page, prefix_offsets=pre[0], prefix_page_ids=p_ids, prefix_page_indptr=p_ptr,
                                           dtype=torch.float64, **kw)
        assert torch.isfinite(o).all() and (o.double() - want).abs().max() < 0.05
        scores = o.flatten(1).float() @ head.float().t()
        u = torch.rand(n, generator=g, device=DEV)
        items, lp = sampling.sample_scores(scores, u, temperature=0.9, top_k=40, top_p=0.9, min_p=0.01)
        ref, _ = sampling.sample_scores_ref(scores, u, temperature=0.9, top_k=40, top_p=0.9, min_p=0.01)
        assert torch.equal(items, ref) and (lp <= 0).all()
    _lib.check_status()
