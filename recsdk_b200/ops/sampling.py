"""Drawing one item per row from its scores on ``csrc/cuda/sampling.cu``: temperature, top-k, top-p and min-p, from given
uniform numbers.  Rows are dense ``[B, V]`` or jagged (the scores of every user's own candidates, as
``HSTURanker.rank`` returns them).  ``sample_scores_ref`` states the same in 64-bit PyTorch for CPU tensors and the tests."""
from __future__ import annotations

import math
import struct
from typing import Optional, Tuple, Union

import torch

from . import _lib

Param = Union[float, int, torch.Tensor]

_SAMPLE_CALL = struct.Struct("@12q5i3f")                # SampleCall of sampling.cu
_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_BIG = torch.finfo(torch.float32).max


def _param(name: str, value: Param, rows: int, dtype: torch.dtype, device: torch.device, lo: float, hi: float, open_lo: bool = False):
    """-> (per-row tensor or None, scalar).  Scalars are checked; what tensors hold is taken as it is."""
    if isinstance(value, torch.Tensor):
        if value.shape != (rows,) or value.device != device:
            raise ValueError("%s must be a scalar or a [%d] tensor on %s, got %s on %s"
                             % (name, rows, device, tuple(value.shape), value.device))
        if dtype is torch.int32 and value.dtype not in (torch.int32, torch.int64):
            raise ValueError("%s must hold integers, got %s" % (name, value.dtype))
        if value.dtype is torch.int64 and dtype is torch.int32:
            value = value.clamp(-1, (1 << 31) - 1)
        return value.to(dtype).contiguous(), 0
    if not (value >= lo and value <= hi) or (open_lo and value == lo):
        raise ValueError("%s = %r is outside %s%g, %g]" % (name, value, "(" if open_lo else "[", lo, hi))
    return None, value


def check_parameters(rows: int, device: torch.device, uniform: torch.Tensor, temperature: Param = 1.0, top_k: Param = 0,
                     top_p: Param = 1.0, min_p: Param = 0.0):
    """Refuses what :func:`sample_scores` refuses of its parameters for ``rows`` rows on ``device``, for callers that have work to
    do before they have scores.  -> (per-row tensor or None, scalar) of temperature, top_k, top_p, min_p."""
    if uniform.shape != (rows,) or uniform.dtype is not torch.float32 or uniform.device != device:
        raise ValueError("uniform must be [%d] fp32 on %s" % (rows, device))
    return (_param("temperature", temperature, rows, torch.float32, device, 0.0, _BIG),
            _param("top_k", top_k, rows, torch.int32, device, 0, (1 << 31) - 1),
            _param("top_p", top_p, rows, torch.float32, device, 0.0, 1.0, open_lo=True),
            _param("min_p", min_p, rows, torch.float32, device, 0.0, 1.0))


def sample_scores(scores: torch.Tensor, uniform: torch.Tensor, offsets: Optional[torch.Tensor] = None, temperature: Param = 1.0,
                  top_k: Param = 0, top_p: Param = 1.0, min_p: Param = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """One item per row -> ``(ids [B] int64, logprobs [B] fp32)``.

    ``scores``: fp32 / fp16 / bf16, ``[B, V]`` (any row stride) or, with ``offsets [B + 1]`` (int32 / int64), the rows one
    after another ``[T]``.  ``uniform [B]`` fp32: numbers in ``[0, 1)``.  In the order (score descending, index ascending)
    the filters keep the first ``top_k`` items (0: all); of those, up to and with the one at which the running sum of
    ``exp(score / temperature)`` reaches ``top_p`` of their sum; of those, the ones with at least ``min_p`` times the
    largest weight (``min_p = 1``: the largest scores only).  The item drawn is the first one, in index order, whose running
    sum over the kept items exceeds ``uniform`` times their sum.  ``temperature = 0`` takes the largest score (the first
    of equals).  Every parameter is a number or a ``[B]`` tensor on the scores' device; in a tensor ``top_k <= 0`` and
    ``top_p >= 1`` are off and ``temperature <= 0`` takes the largest score (NaN: ``top_p`` is off, ``temperature`` takes the
    largest score, ``min_p`` keeps the largest scores only).

    ``ids`` count within the row; ``logprobs`` is the log of the drawn item's share of what was kept (0 for
    ``temperature = 0``) - the propensity to log.  NaN and ``-inf`` are never drawn; a row with nothing else, or with
    nothing at all, gives ``-1`` and ``-inf``.

    Weights carry 1.4e-13 of themselves; what ``top_p`` compares is summed in units of 2^-44 of the largest weight (rows of up to
    2^18 items, longer ones 2^-61 of their sum), the draw's sums in 64 bits.  A border that close to ``top_p`` or ``uniform`` can
    fall on either side, and on another one where the row's alignment or the number of rows has its parts summed in another
    order; the same call always gives the same."""
    if offsets is None:
        if scores.dim() != 2:
            raise ValueError("scores must be [B, V], or [T] with offsets; got %s" % (tuple(scores.shape),))
        rows, width = scores.shape
    else:
        if scores.dim() != 1 or offsets.dim() != 1 or offsets.numel() < 1:
            raise ValueError("jagged scores must be [T] with offsets [B + 1]; got %s and %s"
                             % (tuple(scores.shape), tuple(offsets.shape)))
        if offsets.dtype not in (torch.int32, torch.int64) or offsets.get_device() != scores.get_device():
            raise ValueError("offsets must be int32 or int64 on the scores' device")
        rows, width = offsets.numel() - 1, scores.shape[0]
    index = scores.get_device()                                         # (-1: CPU)
    code = _CODES.get(scores.dtype)
    if code is None:
        raise ValueError("scores must be fp32, fp16 or bf16, got %s" % (scores.dtype,))
    if scores.requires_grad and torch.is_grad_enabled():
        raise ValueError("scores require a gradient, which this operator does not have (use torch.no_grad())")
    if width > (1 << 31) - 65:
        raise ValueError("2^31 - 64 and more scores in a row (or in all jagged rows) are not supported")
    (t_t, t_v), (k_t, k_v), (p_t, p_v), (m_t, m_v) = check_parameters(rows, scores.device, uniform, temperature, top_k, top_p, min_p)
    if not scores.is_cuda:
        return sample_scores_ref(scores, uniform, offsets, temperature, top_k, top_p, min_p)
    if not _lib.is_current(index):
        with torch.cuda.device(index):
            return sample_scores(scores, uniform, offsets, temperature, top_k, top_p, min_p)
    if width > 1 and scores.stride(-1) != 1:
        scores = scores.contiguous()
    uniform = uniform.contiguous()
    ld = off_ptr = off_64 = 0
    if offsets is None:
        ld = scores.stride(0)
    else:
        offsets = offsets.contiguous()
        off_ptr, off_64 = offsets.data_ptr(), offsets.dtype is torch.int64
    ids, logprobs = uniform.new_empty(rows, dtype=torch.int64), torch.empty_like(uniform)
    lib, sms, _ = _lib.launch_env(index)
    rc = lib.rb_sample_scores(_SAMPLE_CALL.pack(
        scores.data_ptr(), ld, off_ptr, width, uniform.data_ptr(), 0 if t_t is None else t_t.data_ptr(), 0 if k_t is None else k_t.data_ptr(),
        0 if p_t is None else p_t.data_ptr(), 0 if m_t is None else m_t.data_ptr(), ids.data_ptr(), logprobs.data_ptr(),
        _lib.raw_stream(index), off_64, rows, int(k_v), code, sms, t_v, p_v, m_v))
    _lib.check(rc, "rb_sample_scores")
    return ids, logprobs


def sample_scores_ref(scores, uniform, offsets=None, temperature: Param = 1.0, top_k: Param = 0, top_p: Param = 1.0,
                      min_p: Param = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """The definition of :func:`sample_scores`, row by row in 64 bits (parameters are taken as their fp32 values)."""
    rows = scores.shape[0] if offsets is None else offsets.numel() - 1
    off = None if offsets is None else offsets.tolist()
    at = lambda v, r: float(torch.as_tensor(v[r] if isinstance(v, torch.Tensor) else v, dtype=torch.float32))  # noqa: E731
    ids = torch.full((rows,), -1, dtype=torch.int64)
    logprobs = torch.full((rows,), -math.inf, dtype=torch.float64)
    for r in range(rows):
        x = (scores[r] if off is None else scores[off[r]:off[r + 1]]).double().cpu()
        x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
        if x.numel() == 0 or float(x.max()) == -math.inf:
            continue
        order = torch.sort(x, descending=True, stable=True)[1]
        order = order[x[order] > -math.inf]
        t = at(temperature, r)
        if not t > 0:
            ids[r], logprobs[r] = order[0], 0.0
            continue
        top = x[order[0]]
        w = torch.where(x[order] == top, torch.ones((), dtype=torch.float64), torch.exp((x[order] - top) / t))
        k = int(top_k[r] if isinstance(top_k, torch.Tensor) else top_k)
        if k > 0:
            order, w = order[:k], w[:k]
        if at(top_p, r) < 1.0:
            run = torch.cumsum(w, 0)
            n = 1 + int((run[:-1] < at(top_p, r) * run[-1]).sum())
            order, w = order[:n], w[:n]
        # (next to the largest score a weight rounds to 1, but is less)
        keep = w >= at(min_p, r) if at(min_p, r) < 1.0 else x[order] == top
        keep[0] = True
        order, w = order[keep], w[keep]
        order, back = torch.sort(order)
        run = torch.cumsum(w[back], 0)
        u = float(uniform[r])
        over = (run > max(u if u == u else 0.0, 0.0) * run[-1]) & (w[back] > 0)
        i = int(over.nonzero()[0]) if bool(over.any()) else int((w[back] > 0).nonzero()[-1])
        ids[r], logprobs[r] = order[i], math.log(float(w[back][i] / run[-1]))
    return ids.to(scores.device), logprobs.float().to(scores.device)
