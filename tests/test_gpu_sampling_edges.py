"""``sample_scores`` at the ends of its ranges, against its row-by-row statement in 64 bits or what must come out."""
import math

import numpy as np
import pytest
import torch

from recsdk_b200.ops import sampling as S

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _same(scores, u, offsets=None, **kw):
    ids, lp = S.sample_scores(scores, u, offsets, **kw)
    want, want_lp = S.sample_scores_ref(scores, u, offsets, **kw)
    assert torch.equal(ids, want), (ids - want).nonzero().flatten().tolist()
    some = want >= 0
    assert (lp[~some] == -math.inf).all()
    # both are fp32 roundings (half a step, 2^-24) of 64-bit values that agree to far more digits
    assert ((lp - want_lp)[some].abs() <= 2.0 ** -23 * want_lp[some].abs() + 1e-11).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("width", [1, 500, 5000, 60000])
def test_parameters_that_are_nan(dtype, width):
    """As a comparison with NaN has it: no top-p, no temperature, and of min-p the largest scores only."""
    g = torch.Generator(device=DEV).manual_seed(width)
    x = torch.randn(5, width, generator=g, device=DEV).to(dtype)
    x[3, ::7] = 5.0
    u = torch.tensor([0.9, 0.5, 0.7, 0.6, 0.99], device=DEV)
    nan = torch.tensor([math.nan, 0.0, math.nan, math.nan, 0.5], device=DEV)
    for kw in (dict(), dict(top_k=3000), dict(top_k=7), dict(top_p=0.9)):
        _same(x, u, min_p=nan, **kw)
    _same(x, u, top_p=nan)
    _same(x, u, temperature=nan)
    if width > 1:
        top = S.sample_scores(x, u, min_p=nan)[0]
        assert top[[0, 2]].tolist() == [int(x[r].float().argmax()) for r in (0, 2)] and top[3] % 7 == 0


def _exact(x, u, top_k, top_p):
    """The item of one row with sums of 64 binary digits: an item weighs down to 2^-42 of the row here, and a running sum of millions
    of items in 53 digits can be off by as much."""
    x = x.double().cpu().numpy()
    order = np.argsort(-x, kind="stable")
    w = np.exp((x[order] - x.max()).astype(np.longdouble))
    if top_k:
        order, w = order[:top_k], w[:top_k]
    run = np.cumsum(w)
    n = 1 + int((run[:-1] < np.longdouble(np.float32(top_p)) * run[-1]).sum())
    back = np.argsort(order[:n])
    order, w = order[back], w[back]
    run = np.cumsum(w)
    i = int(np.argmax(run > np.longdouble(np.float32(u)) * run[-1]))
    return int(order[i]), float(np.log(w[i] / run[-1]))


def _check_exact(x, top_k=0, top_p=1.0):
    u = 1.0 - 2.0 ** -24
    ids, lp = S.sample_scores(x, torch.full((x.shape[0],), u, device=DEV), top_k=top_k, top_p=top_p)
    for r in range(x.shape[0]):
        want, want_lp = _exact(x[r], u, top_k, top_p)
        assert int(ids[r]) == want and abs(float(lp[r]) - want_lp) <= 2.0 ** -23 * abs(want_lp)


@pytest.mark.parametrize("rows", [1, 80])
def test_many_weights_next_to_nothing(rows):
    """One score far above millions of others, which together are kept all the same: with u next to 1 the item is one of them, and
    which one tells how many are."""
    g = torch.Generator(device=DEV).manual_seed(rows)
    x = torch.randn(1, 1 << 22, generator=g, device=DEV) * 0.1 - 28.4
    x[:, 77] = 0.0
    for kw in (dict(top_p=1 - 2.0 ** -21), dict(top_p=1 - 2.0 ** -20), dict(top_k=1 << 21, top_p=1 - 2.0 ** -21)):
        _check_exact(x, **kw)
        if rows > 1:                                                  # a CTA per row instead of several
            some = S.sample_scores(x.expand(rows, x.shape[1]), torch.full((rows,), 1 - 2.0 ** -24, device=DEV), **kw)[0]
            assert (some == some[0]).all() and int(some[0]) == _exact(x[0], 1 - 2.0 ** -24, kw.get("top_k", 0), kw["top_p"])[0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_patterns_next_to_nothing(dtype):
    g = torch.Generator(device=DEV).manual_seed(2)
    x = (torch.rand(2, 1 << 20, generator=g, device=DEV) * 4 - 31).to(dtype)
    x[:, 77] = 0.0
    for p in (1 - 2.0 ** -23, 1 - 2.0 ** -22):
        _check_exact(x, top_p=p)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_weights_past_the_short_rows_units(dtype):
    """Sums from one item's to all items', at temperatures that make every weight 1 or next to none another one."""
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(2, 700001, generator=g, device=DEV).to(dtype)
    for t in (1e-3, 0.05, 1.0, 100.0, 3e4, 1e30, 1e-38):
        for kw in (dict(top_p=0.9), dict(top_k=400000, top_p=0.5), dict(top_p=1e-6), dict(top_p=1 - 2.0 ** -24)):
            _same(x, torch.rand(2, generator=g, device=DEV), temperature=t, **kw)
    _same(x, torch.rand(2, generator=g, device=DEV), temperature=torch.tensor([math.inf, 2.0], device=DEV), top_p=0.7)
    x[:, ::2] = -math.inf
    x[0, 5] = math.inf
    x[1, 7::5] = math.nan
    _same(x, torch.rand(2, generator=g, device=DEV), top_p=0.9)
    # one infinite score, divided by an infinite temperature: whatever else there is has no weight
    ids, lp = S.sample_scores(x, torch.rand(2, generator=g, device=DEV), temperature=torch.tensor([math.inf, 1.0], device=DEV), top_p=0.9)
    assert int(ids[0]) == 5 and float(lp[0]) == 0.0


def test_a_row_of_almost_two_to_the_31():
    """As long as a row may be, among many empty ones (one CTA a row): its last item is the only one that can be drawn."""
    n = (1 << 31) - 65
    x = torch.full((n,), -math.inf, device=DEV)
    x[n - 1] = -2.0
    off = torch.zeros(101, dtype=torch.int64, device=DEV)
    off[43:] = n
    u = torch.full((100,), 0.5, device=DEV)
    for kw in (dict(), dict(top_p=0.9)):
        ids, lp = S.sample_scores(x, u, off, **kw)
        assert int(ids[42]) == n - 1 and float(lp[42]) == 0.0
        ids[42] = -1
        assert (ids == -1).all()
    del x
    torch.cuda.empty_cache()
    with pytest.raises(ValueError, match="2\\^31"):
        S.sample_scores(torch.empty(1, device=DEV).expand(1, (1 << 31) - 64), u[:1])


@pytest.mark.parametrize("lens", [[1, 700, 0, 300000], [1024, 1025, 33, 0, 1, 200001], [1000, 3, 90000]])
def test_short_rows_shared_by_several_ctas(lens):
    """Jagged rows that one CTA could sort, in clusters that the longest row is given."""
    g = torch.Generator(device=DEV).manual_seed(sum(lens))
    x = torch.randn(sum(lens), generator=g, device=DEV)
    o = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
    for kw in (dict(), dict(top_k=1), dict(top_k=7), dict(top_k=10 ** 6), dict(top_p=0.3), dict(top_p=0.95), dict(min_p=0.05), dict(min_p=1.0),
               dict(temperature=0.0), dict(temperature=0.3, top_k=50, top_p=0.9), dict(temperature=2.5, top_k=300, top_p=0.5, min_p=0.01)):
        for _ in range(3):
            _same(x, torch.rand(len(lens), generator=g, device=DEV), o, **kw)
