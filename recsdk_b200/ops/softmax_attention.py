"""Softmax attention over the paged KV cache, for serving: the counterparts of ``append_kvcache`` and
``hstu_attention_paged`` for models with rotary positions and ordinary attention.

* ``append_kv_rotary`` writes the new tokens' keys (turned by their positions) and values into their pages and returns the
  turned queries (``csrc/cuda/kv_rotary.cu``),
* ``softmax_attention_paged`` attends from the new tokens to the cache: causal, optionally only to a sliding window and
  the first few tokens; grouped query heads (``csrc/cuda/softmax_attention.cu``),
* ``softmax_attention_shared_prefix`` does so for groups of requests - one user's candidates or beams - whose histories
  begin with the same tokens: those are read and multiplied once per group.

The cache is the manager's ``[pages, 2, page_size, kv_heads, head_dim]`` of one layer; offsets, page ids and positions are
those of :class:`~recsdk_b200.inference.KVCacheMetadata`.  There is no gradient.  CPU tensors take the fp32 statements
(``*_ref``), which are also what the tests compare with."""
from __future__ import annotations

import functools
import math
import struct
from typing import Optional

import torch

from . import _lib

_HEAD_DIMS = (64, 128)
_INT32, _INT64 = torch.int32, torch.int64
# the launchers' argument records (KvAppendCall, SoftmaxAttnCall): 8-byte fields, ints, floats
_APPEND_CALL = struct.Struct("@19q12i")
_ATTEND_CALL = struct.Struct("@20q12if")


def rotary_table(max_positions: int, rotary_dim: int, base: float = 10000.0, device=None) -> torch.Tensor:
    """fp32 ``[max_positions, rotary_dim]``: ``rotary_dim / 2`` cosines, then as many sines of ``position * base^(-2i /
    rotary_dim)``, computed in 64 bits (a far position times a frequency has no correct digit of its angle left in 32)."""
    if rotary_dim <= 0 or rotary_dim % 16 or max_positions <= 0:
        raise ValueError("rotary_dim must be a positive multiple of 16 and max_positions positive")
    half = rotary_dim // 2
    freq = torch.pow(torch.tensor(base, dtype=torch.float64), -torch.arange(half, dtype=torch.float64) / half)
    ang = torch.arange(max_positions, dtype=torch.float64)[:, None] * freq[None, :]
    return torch.cat([ang.cos(), ang.sin()], dim=1).float().to(device if device is not None else "cpu")


# ----------------------------------------------------------------------------- checks
def _rows(name: str, x: torch.Tensor, heads: Optional[int], dim: int, like: torch.Tensor) -> torch.Tensor:
    """[T, heads, dim] with adjacent heads and 16-byte aligned rows (others are copied; a single row has no stride to mind)."""
    shape = x.shape
    if len(shape) != 3 or shape[2] != dim or (heads is not None and shape[1] != heads):
        raise ValueError("%s must be [tokens, %s, %d], got %s" % (name, "heads" if heads is None else heads, dim, tuple(shape)))
    if x.dtype is not like.dtype or x.get_device() != like.get_device():
        raise ValueError("%s must be %s on %s like the cache, got %s on %s" % (name, like.dtype, like.device, x.dtype, x.device))
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError("%s requires a gradient, which this operator does not have (use torch.no_grad())" % name)
    if x.is_cuda:
        st = x.stride()
        if shape[0] == 1 and st[0] != shape[1] * dim:
            x = x.as_strided(shape, (shape[1] * dim,) + st[1:])
            st = x.stride()
        if (st[2] != 1 or st[1] != dim or st[0] & 7 or st[0] < 0 or x.data_ptr() & 15) and x.numel():
            x = x.contiguous()
            if x.data_ptr() & 15:
                x = x.clone()
    return x


def _ints(name: str, x: torch.Tensor, index: int, n: Optional[int] = None, differences: bool = False) -> torch.Tensor:
    """A vector of int32 on device ``index`` (-1: CPU); int64 is converted: to numbers that do not exist either where it has more
    than 32 bits, or, ``differences``, so that they stay."""
    shape = x.shape
    if len(shape) != 1 or (n is not None and shape[0] != n):
        raise ValueError("%s must be a vector%s, got %s" % (name, "" if n is None else " of %d" % n, tuple(shape)))
    dtype = x.dtype
    if x.get_device() != index or (dtype is not _INT32 and dtype is not _INT64):
        raise ValueError("%s must be int32 or int64 on the cache's device, got %s on %s" % (name, dtype, x.device))
    if dtype is _INT32:
        return x if x.is_contiguous() else x.contiguous()
    return x if index < 0 else (x if differences else x.clamp(-1, (1 << 31) - 1)).to(_INT32).contiguous()


def _cache(kv_cache: torch.Tensor, page_size: int, dims=None) -> torch.Tensor:
    shape = kv_cache.shape
    if len(shape) != 5 or shape[1] != 2 or shape[2] != page_size or not kv_cache.is_contiguous():
        raise ValueError("kv_cache must be a contiguous [pages, 2, %d, kv_heads, head_dim], got %s" % (page_size, tuple(shape)))
    if kv_cache.is_cuda:
        if kv_cache.dtype is not torch.bfloat16 and kv_cache.dtype is not torch.float16:
            raise ValueError("kv_cache must be bf16 or fp16, got %s" % (kv_cache.dtype,))
        if dims is not None and shape[4] not in dims:
            raise ValueError("head_dim must be one of %s, got %d" % (dims, shape[4]))
        if kv_cache.data_ptr() & 15:
            raise ValueError("kv_cache must be 16-byte aligned")
    return kv_cache


# ----------------------------------------------------------------------------- append
def _rotate_ref(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool) -> torch.Tensor:
    half = cos.shape[-1]
    y = x.to(torch.float64 if x.dtype == torch.float64 else torch.float32).clone()
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = y[..., first].clone(), y[..., second].clone()
    y[..., first], y[..., second] = a * cos - b * sin, b * cos + a * sin
    return y.to(x.dtype)


def _pages_of(b, to, page_ids, page_indptr, page_size: int, pages: int) -> torch.Tensor:
    """The page of every token (place ``to`` of request ``b``), -1 where it does not exist."""
    known = (b >= 0) & (b < page_indptr.shape[0] - 1) & (to >= 0)
    b = torch.where(known, b, 0)
    if page_indptr.shape[0] < 2 or page_ids.shape[0] == 0:
        return torch.full_like(to, -1)
    at = page_indptr[b] + to // page_size
    known = known & (at >= 0) & (at < page_indptr[b + 1]) & (at < page_ids.shape[0])
    page = page_ids[torch.where(known, at, 0)]
    return torch.where(known & (page >= 0) & (page < pages), page, -1)


def append_kv_rotary(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kv_cache: torch.Tensor, batch_indices: torch.Tensor,
                     positions: torch.Tensor, page_ids: torch.Tensor, page_indptr: torch.Tensor, page_size: int,
                     table: torch.Tensor, interleaved: bool = False, num_tokens: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Turn the new tokens' queries and keys by their positions, write keys and values into their pages, return the queries.

    ``q [n, heads, head_dim]``, ``k`` / ``v [n, kv_heads, head_dim]`` (token stride free, e.g. slices of one projection);
    token ``i`` is token ``positions[i]`` of request ``batch_indices[i]``, whose pages are
    ``page_ids[page_indptr[b]:page_indptr[b + 1]]``.  ``table`` is :func:`rotary_table`'s ``[max_positions, rotary_dim]``
    (or any cosines and sines); the first ``rotary_dim`` elements of a head turn, element ``i`` with ``i + rotary_dim / 2``
    or, ``interleaved``, ``2i`` with ``2i + 1``.  ``slots``: where a token goes among its request's keys if not at its
    position - behind a shared prefix, whose tokens the request's pages do not hold.  No two tokens of a call may go to the same
    place.

    ``num_tokens``: optional device int32 ``[1]`` (``new_history_nnz_npu``): only that many tokens are there, the rows
    behind them are neither appended nor written to the result - for static buffers under a captured graph.  ``out``: where the
    queries go (may be ``q``).  A token whose position or page does not exist is left out and reported by
    ``_lib.check_status``; on CPU tensors it is refused, before anything is written."""
    cache = _cache(kv_cache, page_size)
    pages, _, _, Hkv, D = cache.shape
    index = cache.get_device()
    if D % 16:
        raise ValueError("head_dim must be a multiple of 16, got %d" % D)
    q, k, v = _rows("q", q, None, D, cache), _rows("k", k, Hkv, D, cache), _rows("v", v, Hkv, D, cache)
    n, H, _ = q.shape
    if k.shape[0] != n or v.shape[0] != n:
        raise ValueError("q, k and v must hold the same tokens, got %d, %d and %d" % (n, k.shape[0], v.shape[0]))
    if table.dim() != 2 or table.dtype is not torch.float32 or table.get_device() != cache.get_device() or not table.is_contiguous() \
            or table.shape[1] % 16 or not 0 < table.shape[1] <= D or (table.is_cuda and table.data_ptr() & 15):
        raise ValueError("table must be a contiguous fp32 [max_positions, rotary_dim] on %s with rotary_dim a multiple of 16 and "
                         "at most %d, got %s %s on %s" % (cache.device, D, table.dtype, tuple(table.shape), table.device))
    batch_indices, positions = _ints("batch_indices", batch_indices, index, n), _ints("positions", positions, index, n)
    page_ids, page_indptr = _ints("page_ids", page_ids, index), _ints("page_indptr", page_indptr, index)
    if num_tokens is not None:
        num_tokens = _ints("num_tokens", num_tokens, index, 1)
    if slots is not None:
        slots = _ints("slots", slots, index, n)
    if page_indptr.shape[0] < 1:
        raise ValueError("page_indptr must be [requests + 1]")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != cache.device or (out.numel() and (
            out.stride(2) != 1 or (H > 1 and out.stride(1) != D) or (n > 1 and (out.stride(0) % 8 or out.stride(0) < H * D))
            or out.data_ptr() % 16)):
        raise ValueError("out must be %s %s on %s with adjacent heads and 16-byte aligned rows" % (tuple(q.shape), q.dtype, cache.device))
    if n == 0:
        return out
    if not cache.is_cuda:
        m = n if num_tokens is None else max(0, min(n, int(num_tokens)))
        pos, b = positions[:m].long(), batch_indices[:m].long()
        to = pos if slots is None else slots[:m].long()
        at = _pages_of(b, to, page_ids.long(), page_indptr.long(), page_size, pages)
        if ((pos < 0) | (pos >= table.shape[0]) | (at < 0)).any():
            raise IndexError("a token's position is not in the table, or its page does not exist")
        cos, sin = table[pos][:, None, :].chunk(2, dim=-1)
        out[:m] = _rotate_ref(q[:m], cos, sin, interleaved)
        cache[at, 0, to % page_size] = _rotate_ref(k[:m], cos, sin, interleaved)
        cache[at, 1, to % page_size] = v[:m]
        return out
    if not _lib.is_current(index):
        with torch.cuda.device(index):
            return append_kv_rotary(q, k, v, cache, batch_indices, positions, page_ids, page_indptr, page_size, table, interleaved,
                                    num_tokens, out, slots)
    lib, sms, status = _lib.launch_env(index)
    rc = lib.rb_kv_append_rotary(_APPEND_CALL.pack(
        q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), out.data_ptr(), out.stride(0) if n > 1 else H * D,
        cache.data_ptr(), pages, batch_indices.data_ptr(), positions.data_ptr(), 0 if slots is None else slots.data_ptr(),
        page_ids.data_ptr(), page_indptr.data_ptr(), 0 if num_tokens is None else num_tokens.data_ptr(), table.data_ptr(), status, _lib.raw_stream(index), n, H, Hkv, D,
        page_indptr.shape[0] - 1, page_size, page_ids.shape[0], table.shape[0], table.shape[1], interleaved, q.dtype is torch.bfloat16, sms))
    _lib.check(rc, "rb_kv_append_rotary")
    return out


# ----------------------------------------------------------------------------- attention
def _attention_ref(q, keys, values, sees, scale: float):
    """q [n, H, D], keys / values [m, Hkv, D], sees [n, m] -> (o [n, H, D], lse [n, H]); rows that see nothing: 0, -inf."""
    n, H, D = q.shape
    G = H // keys.shape[1]
    x = torch.einsum("nhgd,mhd->hgnm", q.view(n, -1, G, D), keys) * scale
    x = x.masked_fill(~sees, -math.inf)
    lse = torch.logsumexp(x, dim=-1)
    p = torch.exp(x - lse.masked_fill(lse == -math.inf, 0.0).unsqueeze(-1))
    seen = sees.any(dim=0)                                              # what nobody sees may be anything
    o = torch.einsum("hgnm,mhd->nhgd", p, values.masked_fill(~seen[:, None, None], 0.0))
    return o.reshape(n, H, D), lse.permute(2, 0, 1).reshape(n, H)


def softmax_attention_ref(q, kv_cache, q_offsets, k_offsets, page_ids, page_indptr, page_size: int, scale: Optional[float] = None,
                          window: int = 0, num_sinks: int = 0, prefix_offsets=None, prefix_page_ids=None, prefix_page_indptr=None,
                          group_offsets=None, dtype: torch.dtype = torch.float32):
    """``(o [T, H, D] in dtype, lse [T, H])`` of the two attention operators, request by request in ``dtype``.  A page of keys
    that some query sees has to be there; the others' may be gone."""
    H, D = q.shape[1], q.shape[2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    qo, ko, ip = q_offsets.tolist(), k_offsets.tolist(), page_indptr.tolist()
    group = None
    if prefix_offsets is not None:
        po, pp = prefix_offsets.tolist(), prefix_page_indptr.tolist()
        go = [0, len(qo) - 1] if group_offsets is None else group_offsets.tolist()
        group = {b: g for g in range(len(go) - 1) for b in range(go[g], go[g + 1])}

    def fetch(ids, n, seen):
        """K and V of a sequence's first n keys, of which ``seen [n]`` are needed."""
        L, pages = (n + page_size - 1) // page_size, kv_cache.shape[0]
        ids = torch.nn.functional.pad(ids[:L].long(), (0, max(L - ids.numel(), 0)), value=-1)
        there = (ids >= 0) & (ids < pages)
        if (torch.nn.functional.pad(seen, (0, L * page_size - n)).view(L, page_size).any(dim=1) & ~there).any():
            raise IndexError("a page of keys that a query sees does not exist")
        c = kv_cache[torch.where(there, ids, 0)] if pages else kv_cache.new_zeros(L, *kv_cache.shape[1:])
        return [c[:, i].reshape(L * page_size, c.shape[3], D)[:n].to(dtype) for i in (0, 1)]

    out = torch.zeros(q.shape[0], H, D, dtype=dtype, device=q.device)
    lse = torch.full((q.shape[0], H), -math.inf, dtype=dtype, device=q.device)
    for b in range(len(qo) - 1):
        n, m = qo[b + 1] - qo[b], ko[b + 1] - ko[b]
        if n == 0:
            continue
        i = torch.arange(m - n, m, device=q.device)[:, None]
        j = torch.arange(m, device=q.device)[None, :]
        sees = j <= i
        if window > 0:
            sees = sees & ((j > i - window) | (j < num_sinks))
        k, v = fetch(page_ids[ip[b]:ip[b + 1]], m, sees.any(dim=0))
        if group is not None and b in group:
            g = group[b]
            kp, vp = fetch(prefix_page_ids[pp[g]:pp[g + 1]], po[g + 1] - po[g], torch.ones(po[g + 1] - po[g], dtype=torch.bool, device=q.device))
            k, v = torch.cat([kp, k]), torch.cat([vp, v])
            sees = torch.cat([torch.ones(n, kp.shape[0], dtype=torch.bool, device=q.device), sees], dim=1)
        if k.shape[0]:
            out[qo[b]:qo[b + 1]], lse[qo[b]:qo[b + 1]] = _attention_ref(q[qo[b]:qo[b + 1]].to(dtype), k, v, sees, scale)
    return out, lse


@functools.lru_cache(maxsize=1024)
def _plan(sms: int, *sizes):
    """-> (bytes of workspace, kernels launched)."""
    return _lib.lib().rb_softmax_attn_workspace(sms, *sizes), _lib.lib().rb_softmax_attn_kernels(*sizes)


def _attend(q, kv_cache, q_offsets, k_offsets, page_ids, page_indptr, page_size, scale, window, num_sinks, return_lse, prefix=None):
    cache = _cache(kv_cache, page_size, _HEAD_DIMS)
    pages, _, _, Hkv, D = cache.shape
    index = cache.get_device()
    q = _rows("q", q, None, D, cache)
    T, H, _ = q.shape
    ld_q = q.stride(0)
    if (ld_q < H * D or ld_q % D) and index >= 0:
        q = q.contiguous()                                              # a tensor map's strides are whole multiples, and do not overlap
        ld_q = H * D
    if H == 0 or H % Hkv:
        raise ValueError("%d query heads cannot share %d key heads" % (H, Hkv))
    B = q_offsets.numel() - 1
    if B < 0:
        raise ValueError("q_offsets must be [requests + 1]")
    q_offsets, k_offsets = _ints("q_offsets", q_offsets, index), _ints("k_offsets", k_offsets, index, B + 1, differences=True)
    page_ids, page_indptr = _ints("page_ids", page_ids, index), _ints("page_indptr", page_indptr, index, B + 1)
    if window < 0 or num_sinks < 0:
        raise ValueError("window and num_sinks must not be negative")
    scale = D ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    groups, g_off, p_off, p_ids, p_ptr = 0, None, None, None, None
    if prefix is not None:
        g_off, p_off, p_ids, p_ptr = prefix
        groups = p_off.numel() - 1
        if groups < 0 or (g_off is None and groups != 1):
            raise ValueError("prefix_offsets must be [groups + 1], and [2] without group_offsets")
        p_off, p_ids = _ints("prefix_offsets", p_off, index, differences=True), _ints("prefix_page_ids", p_ids, index)
        p_ptr = _ints("prefix_page_indptr", p_ptr, index, groups + 1)
        if g_off is not None:
            g_off = _ints("group_offsets", g_off, index, groups + 1)
    if not cache.is_cuda:
        o, lse = softmax_attention_ref(q, cache, q_offsets, k_offsets, page_ids, page_indptr, page_size, scale, window, num_sinks,
                                       p_off, p_ids, p_ptr, g_off)
        return (o.to(q.dtype), lse) if return_lse else o.to(q.dtype)
    if page_size % 16:
        raise ValueError("page_size must be a multiple of 16, got %d" % page_size)
    if T and B == 0:
        raise ValueError("q holds %d tokens but there are no requests" % T)
    if pages == 0:
        raise ValueError("kv_cache holds no pages")
    if not _lib.is_current(index):
        with torch.cuda.device(index):
            return _attend(q, cache, q_offsets, k_offsets, page_ids, page_indptr, page_size, scale, window, num_sinks, return_lse, prefix)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty((T, H), dtype=torch.float32, device=cache.device) if return_lse else None
    if T:
        lib, sms, status = _lib.launch_env(index)
        nbytes, kernels = _plan(sms, T, H, Hkv, D, B, groups, scale)
        ws = q.new_empty(nbytes // 2)                                   # (16-bit elements)
        rc = lib.rb_softmax_attn_paged(_ATTEND_CALL.pack(
            q.data_ptr(), ld_q, T, cache.data_ptr(), pages, q_offsets.data_ptr(), k_offsets.data_ptr(), page_ids.data_ptr(),
            page_indptr.data_ptr(), 0 if g_off is None else g_off.data_ptr(), p_off.data_ptr() if groups else 0,
            p_ids.data_ptr() if groups else 0, p_ptr.data_ptr() if groups else 0, out.data_ptr(), H * D,
            0 if lse is None else lse.data_ptr(), ws.data_ptr(), nbytes, status, _lib.raw_stream(index), H, Hkv, D, page_size,
            page_ids.shape[0], B, p_ids.shape[0] if groups else 0, groups, min(window, 1 << 30), min(num_sinks, 1 << 30),
            q.dtype is torch.bfloat16, sms, scale))
        _lib.check(rc, "rb_softmax_attn_paged")
        _lib.launch_count += kernels
    return (out, lse) if return_lse else out


def softmax_attention_paged(q: torch.Tensor, kv_cache: torch.Tensor, q_offsets: torch.Tensor, k_offsets: torch.Tensor,
                            page_ids: torch.Tensor, page_indptr: torch.Tensor, page_size: int, scale: Optional[float] = None,
                            window: int = 0, num_sinks: int = 0, return_lse: bool = False):
    """Causal softmax attention of the new tokens (``q [T, heads, head_dim]``, jagged by ``q_offsets``) over the paged cache.

    Request ``b`` has ``k_offsets[b + 1] - k_offsets[b]`` keys in the pages ``page_ids[page_indptr[b]:page_indptr[b + 1]]``,
    the last of which are its new tokens' own (already appended); its ``i``-th query sits at the position of the ``i``-th of
    them.  A query sees the keys up to its position - with ``window > 0`` only the last ``window`` of them (itself
    included) and the first ``num_sinks`` tokens.  Pages that lie wholly before the window and after the sinks are not
    read and may be gone.  ``heads`` is a multiple of the cache's ``kv_heads``; query head ``h`` reads key head
    ``h // (heads / kv_heads)``.  ``scale`` defaults to ``head_dim ** -0.5``.

    Returns ``[T, heads, head_dim]`` (and, ``return_lse``, fp32 ``[T, heads]``: log of the sum of the exponentials).  A
    query that sees no key gives 0 and ``-inf``; rows of ``q`` behind the last request are undefined in the result.  bf16 or
    fp16, head_dim 64 or 128, page_size a multiple of 16.  Stale values in slots that a block of queries does not see do no
    harm; a non-finite VALUE that one query sees can spread to neighbouring queries of the same request that do not.  A
    missing page reads as zeros and is reported by ``_lib.check_status`` (on CPU tensors it is refused).  Where requests
    have many queries, one whose largest score (``scale`` times the product) lies beyond 5 * 10^6 on either side of 0 is reported
    in the same way; its result is undefined.

    Scores, weights and their sums are fp32; a weight is rounded to the inputs' type for its product with the values and the
    result once more, half a step each."""
    return _attend(q, kv_cache, q_offsets, k_offsets, page_ids, page_indptr, page_size, scale, window, num_sinks, return_lse)


def softmax_attention_shared_prefix(q: torch.Tensor, kv_cache: torch.Tensor, q_offsets: torch.Tensor, k_offsets: torch.Tensor,
                                    page_ids: torch.Tensor, page_indptr: torch.Tensor, prefix_offsets: torch.Tensor,
                                    prefix_page_ids: torch.Tensor, prefix_page_indptr: torch.Tensor, page_size: int,
                                    group_offsets: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                                    return_lse: bool = False):
    """:func:`softmax_attention_paged` for requests that share what stands before their own keys.

    Group ``g`` is the requests ``group_offsets[g]:group_offsets[g + 1]`` (without ``group_offsets``: one group of all);
    all of its queries see the ``prefix_offsets[g + 1] - prefix_offsets[g]`` keys of the pages
    ``prefix_page_ids[prefix_page_indptr[g]:prefix_page_indptr[g + 1]]``, then - causally - their request's own keys, which
    ``k_offsets``, ``page_ids`` and ``page_indptr`` describe without the prefix (a request need not have any).  The result is that of one
    attention over prefix and own keys together; the prefix is read once for the group instead of once per request."""
    return _attend(q, kv_cache, q_offsets, k_offsets, page_ids, page_indptr, page_size, scale, 0, 0, return_lse,
                   (group_offsets, prefix_offsets, prefix_page_ids, prefix_page_indptr))
