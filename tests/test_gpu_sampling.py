"""``sample_scores`` on the GPU against its row-by-row statement in 64 bits: the items are the same, always."""
import math

import pytest
import torch

from recsdk_b200.ops import sampling as S

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _same(scores, u, offsets=None, **kw):
    ids, lp = S.sample_scores(scores, u, offsets, **kw)
    want, want_lp = S.sample_scores_ref(scores, u, offsets, **kw)
    assert ids.dtype == torch.int64 and lp.dtype == torch.float32
    assert torch.equal(ids, want), (ids - want).nonzero().flatten().tolist()
    some = want >= 0
    assert (lp[~some] == -math.inf).all()
    # both are fp32 roundings (half a step, 2^-24) of 64-bit values that agree to far more digits
    assert ((lp - want_lp)[some].abs() <= 2.0 ** -23 * want_lp[some].abs() + 1e-11).all()


FILTERS = [dict(), dict(top_k=1), dict(top_k=7), dict(top_k=10 ** 6), dict(top_p=0.3), dict(top_p=0.95), dict(min_p=0.05), dict(min_p=1.0),
           dict(temperature=0.0), dict(temperature=0.3, top_k=50, top_p=0.9), dict(temperature=2.5, top_k=300, top_p=0.5, min_p=0.01),
           dict(top_p=1e-6)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("width", [1, 2, 31, 33, 511, 4099, 50021])
def test_dense(dtype, width):
    g = torch.Generator(device=DEV).manual_seed(width)
    rows = 24 if width < 10000 else 6
    x = (torch.randn(rows, width, generator=g, device=DEV) * 2.5).to(dtype)
    for kw in FILTERS:
        _same(x, torch.rand(rows, generator=g, device=DEV), **kw)


@pytest.mark.parametrize("off", [torch.int32, torch.int64])
def test_jagged(off):
    g = torch.Generator(device=DEV).manual_seed(3)
    lens = [0, 1, 5, 0, 1000, 33, 4096, 2, 0]
    x = torch.randn(sum(lens), generator=g, device=DEV)
    o = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=off, device=DEV)
    for kw in FILTERS:
        _same(x, torch.rand(len(lens), generator=g, device=DEV), o, **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ties(dtype):
    """Many equal scores: the cut goes through them by index."""
    g = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randint(-3, 3, (16, 777), generator=g, device=DEV).to(dtype) * 0.5
    x[1] = 1.0
    x[2] = -0.0
    x[2, ::2] = 0.0
    for kw in FILTERS + [dict(top_k=100, top_p=0.5), dict(top_p=0.5)]:
        _same(x, torch.rand(16, generator=g, device=DEV), **kw)


def test_infinities_and_nan():
    inf = math.inf
    rows = [[-inf] * 5, [math.nan] * 5, [inf, 1.0, inf, -inf, math.nan], [-inf, math.nan, 2.0, -inf, -inf], [3e38, -3e38, 3e38, 0, 0],
            [-3.4e38, -inf, -3.4e38, math.nan, -3.4e38], [0.0, -0.0, 0.0, -0.0, -inf]]
    x = torch.tensor(rows, device=DEV)
    for uv in (0.0, 0.4, 0.999999):
        for kw in (dict(), dict(top_k=2), dict(top_p=0.4), dict(min_p=0.5), dict(temperature=0.0), dict(temperature=1e-30)):
            _same(x, torch.full((len(rows),), uv, device=DEV), **kw)
    _same(x.half(), torch.full((len(rows),), 0.7, device=DEV))


def test_border_uniforms_and_equal_weights():
    x = torch.zeros(8, 1000, device=DEV)
    u = torch.tensor([0.0, 0.001, 0.5, 0.25, 0.75, 1.0 - 2.0 ** -24, 1.0, 0.125], device=DEV)
    for kw in (dict(), dict(top_k=8), dict(top_k=512, top_p=0.5), dict(top_p=0.25)):
        _same(x, u, **kw)
    ids, lp = S.sample_scores(x, u, top_k=8)
    assert ids.tolist() == [0, 0, 4, 2, 6, 7, 7, 1] and torch.allclose(lp, torch.full_like(lp, -math.log(8)))


def test_parameters_per_row():
    g = torch.Generator(device=DEV).manual_seed(6)
    x = torch.randn(12, 3001, generator=g, device=DEV)
    u = torch.rand(12, generator=g, device=DEV)
    t = torch.tensor([0.0, 1, 0.5, 2, -1, 1, 1, 1, 0.2, 1, 3, 1], device=DEV)
    k = torch.tensor([0, 1, 5, 0, 3, -4, 10 ** 6, 100, 7, 0, 2, 3000], device=DEV)
    p = torch.tensor([1, 0.5, 2, 0.9, 0.1, 0.99, 0.7, 1, 0.0, -1, 0.5, 0.3], device=DEV)
    m = torch.tensor([0, 0, 0, 0.1, 0, 0.5, 0, 1, 2, 0, 0, 0.01], device=DEV)
    _same(x, u, temperature=t, top_k=k, top_p=p, min_p=m)
    _same(x, u, temperature=0.7, top_k=k.int(), top_p=0.8, min_p=m)


def test_strides_streams_and_graph():
    g = torch.Generator(device=DEV).manual_seed(7)
    big = torch.randn(10, 4000, generator=g, device=DEV)
    u = torch.rand(10, generator=g, device=DEV)
    for x in (big[:, 3:2000], big[::2, :777], big.t()[:10, ::3][:, :3]):
        _same(x, u[: x.shape[0]], top_k=20, top_p=0.9)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ids, _ = S.sample_scores(big, u, top_p=0.9)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gids, glp = S.sample_scores(big, u, top_p=0.9)
    graph.replay()
    assert torch.equal(gids, ids)
    u.copy_(torch.rand(10, generator=g, device=DEV))
    graph.replay()
    assert torch.equal(gids, S.sample_scores(big, u, top_p=0.9)[0])


def test_the_draws_follow_the_distribution():
    """Evenly spaced uniforms: every item comes exactly as often as its share says, to within one draw at each border."""
    x = torch.randn(300, generator=torch.Generator().manual_seed(8))
    n = 20000
    u = ((torch.arange(n) + 0.5) / n).to(DEV)
    ids, _ = S.sample_scores(x.to(DEV).expand(n, 300), u, temperature=0.8)
    want = torch.softmax(x.double() / torch.tensor(0.8, dtype=torch.float32).double(), 0) * n
    assert ((torch.bincount(ids.cpu(), minlength=300) - want).abs() <= 1.01).all()


def test_more_rows_than_blocks_and_long_jagged_rows():
    g = torch.Generator(device=DEV).manual_seed(9)
    x = torch.randn(70001, 6, generator=g, device=DEV)
    u = torch.rand(70001, generator=g, device=DEV)
    ids, _ = S.sample_scores(x, u, top_k=3)
    pick = torch.tensor([0, 1, 65535, 65536, 69999, 70000])
    assert torch.equal(ids[pick], S.sample_scores_ref(x[pick], u[pick], top_k=3)[0])
    # a row far longer than the average, beyond what shared memory holds
    lens = [700001, 3, 100, 2000]
    x = torch.randn(sum(lens), generator=g, device=DEV).half()
    o = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), device=DEV)
    for kw in (dict(top_p=0.9), dict(top_k=5000, top_p=0.99), dict(min_p=0.01), dict(temperature=0.0)):
        _same(x, torch.rand(4, generator=g, device=DEV), o, **kw)


def test_the_ranker_draws_from_its_scores():
    from recsdk_b200.inference import KVCacheConfig, KVCacheManager
    from recsdk_b200.models.hstu import HSTU, HSTUConfig
    from recsdk_b200.models.hstu_inference import HSTURanker

    torch.manual_seed(0)
    cfg = HSTUConfig(num_layers=2, d_model=128, num_heads=2, head_dim=64, max_seq_len=1024, num_time_buckets=16)
    model = HSTU(cfg, torch.nn.Identity(), DEV, torch.bfloat16).eval()
    make = lambda: HSTURanker(model, KVCacheManager.from_config(KVCacheConfig(  # noqa: E731
        num_layers=2, num_heads=2, head_dim=64, page_size=32, offload_chunksize=64, num_primary_cache_pages=64, num_buffer_pages=16,
        host_capacity_per_layer=1 << 22, max_batch_size=4, max_seq_len=1024, dtype=torch.bfloat16, device=DEV)))
    users, hist, cands = torch.tensor([3, 5, 8]), torch.tensor([100, 60, 30]), torch.tensor([20, 0, 300])
    x = (torch.randn(510, 128, device=DEV) * 0.5).bfloat16()
    u = torch.tensor([0.3, 0.1, 0.95], device=DEV)
    scores = make().rank(users, hist, cands, x)
    ids, lp = make().recommend(users, hist, cands, x, u, temperature=0.5, top_p=0.9)
    want, want_lp = S.sample_scores_ref(scores, u, torch.tensor([0, 20, 20, 320]), temperature=0.5, top_p=0.9)
    assert torch.equal(ids, want) and ids[1] == -1 and torch.allclose(lp[[0, 2]], want_lp[[0, 2]], rtol=1e-6)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("width", [1025, 5003, 65536, 131071])
def test_patterns_of_16_bits(dtype, width):
    """Rows whose values are few, all, or more often the same than 16 bits count; zeros of both signs, infinities, NaN."""
    g = torch.Generator(device=DEV).manual_seed(width)
    n = (12, width + 3)
    x = (torch.randn(*n, generator=g, device=DEV) * 2.0).to(dtype)[:, 3:]     # 16-byte borders fall anywhere
    x[1] = -1.5
    x[2] = 0.0
    x[2, ::2] = -0.0
    x[3] = torch.where(torch.rand(width, generator=g, device=DEV) < 0.9, 0.0, -0.0).to(dtype)
    x[3, 5] = 1e-3
    x[4] = torch.randint(-32768, 32768, (width,), generator=g, device=DEV).to(torch.int16).view(dtype)        # every pattern
    x[5] = torch.where(x[4].isfinite(), x[4], torch.zeros_like(x[4]))
    x[6, ::3] = -math.inf
    x[6, 1::3] = math.nan
    x[7] = -math.inf
    x[7, 1::2] = -math.nan
    x[8] = x[0].abs() * -1e-4
    x[9, width // 2] = math.inf
    x[10] = -x[5].abs()
    x[11] = -math.inf
    x[11, width - 1] = -3.0
    filters = FILTERS + [dict(top_k=513), dict(top_k=900, top_p=0.9), dict(top_k=width - 1, top_p=0.999), dict(top_p=0.9, min_p=0.002),
                         dict(temperature=3e4), dict(temperature=3e4, top_p=0.9, min_p=0.3), dict(temperature=1e-3, top_p=0.99)]
    for kw in filters:
        _same(x, torch.rand(12, generator=g, device=DEV), **kw)
    per_row = dict(top_k=torch.tensor([0, 1, 600, 0, 512, 513, 1024, 0, 5000, 0, 77, 0], dtype=torch.int32, device=DEV),
                   temperature=torch.tensor([0.0, 1.0, 2.0, 0.5] * 3, device=DEV))
    _same(x, torch.rand(12, generator=g, device=DEV), **per_row)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 9, 10, 33, 75])
def test_few_long_rows(dtype, rows):
    """One to eight CTAs a row."""
    g = torch.Generator(device=DEV).manual_seed(rows)
    x = torch.randn(rows, 300007 if rows < 20 else 70001, generator=g, device=DEV).to(dtype)
    for kw in (dict(), dict(top_p=0.9, min_p=0.002), dict(top_k=40), dict(top_k=5000, top_p=0.8), dict(temperature=0.0)):
        _same(x, torch.rand(rows, generator=g, device=DEV), **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_min_p_keeps_down_to_zero(dtype):
    """The lowest kept score is 0, whose neighbour below is -0."""
    x = -torch.rand(4, 3001, device=DEV).to(dtype) - 0.5
    x[:, 5::7] = 0.0
    x[1, 5::14] = -0.0
    x[2, 100] = 0.25
    for kw in (dict(min_p=1.0), dict(min_p=0.7), dict(min_p=0.7, top_p=0.99), dict(min_p=0.65, top_k=2000)):
        _same(x, torch.rand(4, device=DEV), **kw)


def test_more_long_rows_than_blocks():
    """Rows of patterns that a CTA works through one after another."""
    g = torch.Generator(device=DEV).manual_seed(11)
    x = torch.randn(66001, 1100, generator=g, device=DEV).bfloat16()
    u = torch.rand(66001, generator=g, device=DEV)
    pick = torch.tensor([0, 1, 464, 465, 65535, 65536, 66000])
    for kw in (dict(top_p=0.9), dict(top_k=600, top_p=0.9, min_p=0.01)):
        ids, _ = S.sample_scores(x, u, **kw)
        assert torch.equal(ids[pick], S.sample_scores_ref(x[pick], u[pick], **kw)[0])


def test_counts_past_32_bits():
    x = torch.randn(4, 2000, device=DEV)
    k = torch.tensor([1 << 40, (1 << 32) + 1, -(1 << 32) + 3, 2], device=DEV)
    _same(x, torch.rand(4, device=DEV), top_k=k, temperature=2.0)
