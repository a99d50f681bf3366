"""``sample_scores`` at the ends of its ranges, against its row-by-row statement in 64 bits or what must come out."""
import math

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
