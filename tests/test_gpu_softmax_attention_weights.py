"""fp16 weights of keys far below the largest score: many of them together carry weight that none of them has alone.

Bounds.  With ``h = 2^-11`` a weight in fp16's normal range is off by ``h`` of itself and the result by ``h`` of itself, so
``h * A + h * |o|`` with ``A`` the attention's own average of ``|v|``.  A weight below that range is off by at most half of its
smallest step, 2^-25.  The kernels hold the largest weight at 2^15 (few rows) or between 2^11 and 2^15 (many rows), so that is
2^-36 of the largest weight, of which the sum holds at least one: ``n * 2^-36 * max |v|`` for n keys.  A score is an fp32 sum of
D <= 128 exact products with ``sum |q_i k_i| * scale <= 24`` here, off by 128 * 2^-23 * 24 = 24 * 2^-16, which the numerator and
the sum of weights each take once: ``48 * 2^-16 * A``; the lse takes it once."""
import math

import pytest
import torch

from recsdk_b200.ops import _lib
from recsdk_b200.ops import softmax_attention as SA

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _off(lens):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=DEV)


def _inputs(new, keys, D, gap, at, g, page=64, Hkv=2, H=4):
    """Every request's key ``at`` (from the end if negative) scores ``gap`` above its others and has a value next to nothing."""
    n = [(x + page - 1) // page for x in keys]
    cache = torch.randn(sum(n), 2, page, Hkv, D, generator=g, device=DEV)
    cache[:, 0] *= 0.05
    cache[:, 1] = 1.0 + 0.1 * cache[:, 1]
    ids = torch.randperm(sum(n), generator=g, device=DEV).int()
    ptr = _off(n)
    for b, m in enumerate(keys):
        if at is None:
            # the scores climb all the way, by less than the gap in all
            up = torch.linspace(0.0, 1.25, n[b] * page, device=DEV).view(n[b], page, 1, 1)
            cache[ids[int(ptr[b]):int(ptr[b + 1])].long(), 0] += up
        else:
            j = at % (m - new[b] + 1)                                  # one that all of the request's queries see
            row = cache[int(ids[int(ptr[b]) + j // page])]
            row[0, j % page], row[1, j % page] = 1.25, 0.01
    q = 1.75 + 0.01 * torch.randn(sum(new), H, D, generator=g, device=DEV)
    return q.half(), cache.half(), _off(new), _off(keys), ids, ptr, page, dict(scale=gap / (1.75 * 1.25 * D))


@pytest.mark.parametrize("gap", [10.0, 14.0, 17.5])
@pytest.mark.parametrize("at", [0, -1, 20000, None])
@pytest.mark.parametrize("new,keys", [([1, 1], [40000, 30001]), ([1] * 160, [700] * 159 + [50000]), ([200], [40000]), ([130, 300], [30001, 45000])])
@pytest.mark.parametrize("D", [64, 128])
def test_weights_far_below_the_largest(D, new, keys, at, gap):
    g = torch.Generator(device=DEV).manual_seed(D + len(new))
    *args, kw = _inputs(new, keys, D, gap, at, g)
    got, lse = SA.softmax_attention_paged(*args, return_lse=True, **kw)
    ref, ref_lse = SA.softmax_attention_ref(*args, dtype=torch.float64, **kw)     # (all values are positive: their average is ref)
    assert (ref > 0).all()
    _lib.check_status()
    h = 2.0 ** -11
    tol = 2 * h * ref + max(keys) * 2.0 ** -36 * 1.6 + 48 * 2.0 ** -16 * ref
    err = (got.double() - ref).abs()
    assert (err <= tol).all(), "worst %g of %g" % ((err - tol).max().item(), ref.flatten()[(err - tol).argmax()].item())
    assert ((lse.double() - ref_lse).abs() <= 24 * 2.0 ** -16 + 2.0 ** -22 * ref_lse.abs()).all()


@pytest.mark.parametrize("at", [0, 20000, None])
@pytest.mark.parametrize("D", [64, 128])
def test_as_many_requests_as_warps(D, at):
    """Enough single tokens for every warp to go through all the keys of some (here all have the same ones)."""
    g = torch.Generator(device=DEV).manual_seed(D)
    q, cache, _, _, ids, ptr, page, kw = _inputs([1], [33000], D, 17.5, at, g)
    n = 1200
    args = (q.expand(n, 4, D).contiguous(), cache, _off([1] * n), _off([33000] * n), ids.repeat(n), _off([ids.numel()] * n), page)
    got = SA.softmax_attention_paged(*args, **kw)
    ref, _ = SA.softmax_attention_ref(q, cache, _off([1]), _off([33000]), ids, ptr, page, dtype=torch.float64, **kw)
    _lib.check_status()
    tol = 2 * 2.0 ** -11 * ref + 33000 * 2.0 ** -36 * 1.6 + 48 * 2.0 ** -16 * ref
    err = (got.double() - ref).abs()
    assert (err <= tol).all(), "worst %g of %g" % (err.max().item(), ref.max().item())


@pytest.mark.parametrize("new", [1, 90])
def test_behind_a_shared_prefix(new):
    """The large weight is in the prefix, the many small ones in the request's own keys, and the other way round."""
    g = torch.Generator(device=DEV).manual_seed(4)
    for at in (0, 41000):
        q, cache, qo, ko, ids, ptr, page, kw = _inputs([new, new], [40000, 40000], 64, 17.5, at, g)
        own = SA.softmax_attention_ref(q[:new], cache, qo[:2], _off([40000]), ids[:625], ptr[:2], page, dtype=torch.float64, **kw)[0]
        # the first 16000 keys of request 0 as the prefix of a group of one
        got = SA.softmax_attention_shared_prefix(q[:new], cache, qo[:2], _off([24000]), ids[250:625].contiguous(), _off([375]), _off([16000]),
                                                 ids[:250].contiguous(), _off([250]), page, **kw)
        tol = 2 * 2.0 ** -11 * own + 40000 * 2.0 ** -36 * 1.6 + 48 * 2.0 ** -16 * own
        assert ((got.double() - own).abs() <= tol).all()
    _lib.check_status()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new", [1, 140])
def test_very_large_scores(dtype, new):
    """One key stands out by more than any weight can show, at sizes where fp32 has no digits behind the point: the result is that
    key's value, to within the rounding of its weight and of the result (half a step each); or the score is reported."""
    g = torch.Generator(device=DEV).manual_seed(5)
    D, page = 64, 16
    cache = torch.randn(25, 2, page, 2, D, generator=g, device=DEV)
    cache[:, 0] *= 0.01
    cache[3, 0, 5] = 30000.0
    cache = cache.to(dtype)
    q = torch.full((new, 4, D), 3000.0, device=DEV).to(dtype)
    want = cache[3, 1, 5].repeat_interleave(2, 0).double()
    for scale in (1e-4, 1e-3, 1.9e-3, 1.0, 30.0):                   # scores of 5.76e9 times that
        got = SA.softmax_attention_paged(q, cache, _off([new]), _off([400]), torch.arange(25, device=DEV), _off([25]), page, scale=scale)
        if new > 1 and scale > 1e-3:
            with pytest.raises(_lib.KernelStatusError, match="too large"):
                _lib.check_status()
            continue
        _lib.check_status()
        assert ((got.double() - want).abs() <= 1.01 * torch.finfo(dtype).eps * want.abs()).all()
    if new > 1:                                                       # nothing but scores far below 0
        low = cache.clone()
        low[:, 0] = -30000.0
        SA.softmax_attention_paged(q, low, _off([new]), _off([400]), torch.arange(25, device=DEV), _off([25]), page, scale=1.0)
        with pytest.raises(_lib.KernelStatusError, match="too large"):
            _lib.check_status()
    q[0, 1, 3] = math.inf                                             # infinities are not sizes
    got = SA.softmax_attention_paged(q, cache, _off([new]), _off([400]), torch.arange(25, device=DEV), _off([25]), page, scale=1e-3)
    assert torch.isnan(got[0, 1]).all() and torch.isfinite(got[:, 2:]).all()
    _lib.check_status()
