"""A key/value cache in pages: appending a step's tokens, attention over what is there.

Caches are (Pages, KV_Heads, Page_Size, Dim) views - (page, head, slot, Dim) storage, or
(page, slot, head, Dim) storage seen through ``transpose(1, 2)``.  ``page_table`` (Batch,
Max_Pages) names the pages of each sequence in order; ``cache_lens`` (Batch,) counts the tokens
a sequence had before this step; ``new_lens`` (Batch,), where sequences bring different numbers
of tokens, says how many of the step's SeqLen rows are real.  The same tensors serve both calls:

    q = paged_kv_append(k, v, k_cache, v_cache, page_table, cache_lens, cos, sin, q=q, ...)
    out = paged_attention(q, k_cache, v_cache, page_table, cache_lens, ...)
    cache_lens += 1                       # or by the drafts that were accepted

No counterpart among the reference's samples.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from .rope import (aligned_table, check_no_grad, check_out, check_positions, check_table, check_weights,
                   empty_rows, rows_view)

_APPEND = _lib.LayoutPlans("b200k_paged_kv_append", _lib.PagedKvAppendArgs)
_ATTENTION = _lib.LayoutPlans("b200k_paged_attention", _lib.PagedAttentionArgs)


def _check_cache(k_cache, v_cache, page_table, cache_lens, new_lens, batch, heads, dim, dtype, device):
    if k_cache.ndim != 4 or k_cache.shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must both be (Pages, KV_Heads, Page_Size, Dim).")
    if k_cache.shape[1] != heads or k_cache.shape[3] != dim:
        raise ValueError(f"the cache holds {k_cache.shape[1]} heads of {k_cache.shape[3]}, "
                         f"the call {heads} of {dim}")
    if k_cache.dtype != dtype or v_cache.dtype != dtype:
        raise ValueError("the cache must have the data type of the tokens.")
    if k_cache.shape[2] == 0:
        raise ValueError("pages must hold at least one token")
    for c, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        if c.numel() and (c.stride(3) != 1 or any(s == 0 and n > 1 for s, n in zip(c.stride(), c.shape))):
            raise ValueError(f"{name} must have contiguous rows that do not overlap")
    if page_table.ndim != 2 or page_table.shape[0] != batch:
        raise ValueError(f"page_table must be ({batch}, Max_Pages), got {tuple(page_table.shape)}")
    for t, name, shape in ((page_table, "page_table", None), (cache_lens, "cache_lens", (batch,)),
                           (new_lens, "new_lens", (batch,))):
        if t is None:
            continue
        if t.dtype != torch.int32:
            raise TypeError(f"{name} must be int32")
        if shape is not None and t.shape != shape:
            raise ValueError(f"{name} must be ({batch},), got {tuple(t.shape)}")
        if t.numel() > 1 and t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"{name} must be contiguous along its last axis")
    for t in (k_cache, v_cache, page_table, cache_lens, new_lens):
        if t is not None and t.device != device:
            raise ValueError("caches, page_table and lengths must be on the device of the tokens.")


def paged_kv_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    page_table: torch.Tensor, cache_lens: torch.Tensor,
                    cos: torch.Tensor | None = None, sin: torch.Tensor | None = None, *,
                    q: torch.Tensor | None = None,
                    q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                    positions: torch.Tensor | None = None, new_lens: torch.Tensor | None = None,
                    eps: float = 1e-6, interleaved: bool = False,
                    q_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Stores k and v (Batch, KV_Heads, SeqLen, Dim), float16 or bfloat16, as tokens
    cache_lens[b], cache_lens[b] + 1, ... of their sequences; k is normed (with ``k_weight``) and
    rotated (with ``cos`` / ``sin``) on the way, as in ``qk_norm_rope``.  With ``q`` (Batch, Heads,
    SeqLen, Dim) the step's queries are normed and rotated in the same launch and returned (in
    ``q_out``, which may be q itself).

    ``positions`` (SeqLen,) or (Batch, SeqLen) are the tokens' positions where those are not their
    places in the cache (drafts of one depth in a tree share a position); one outside the table
    makes the rotated values of its rows NaN, in the cache too.  Rows behind new_lens[b] are
    padding: their cache slots stay as they are, as do their rows of a given ``q_out``; in a q_out
    made here they are zero.  A token whose page lies outside the table or the cache is not stored.
    ``raise_on_device_error()`` names the token or the sequence.  Sequences may share the pages that
    they only read: of two tokens that a call stores in one slot, parts of either may stay.  Outputs
    overlap no input, but for q_out = q.

    Dim is a multiple of 8 up to 256 and pages hold any number of tokens; ``paged_attention`` reads
    caches of heads up to 128 and pages of a multiple of 8 tokens, and nothing else here reads others."""
    tensors = (k, v, q, k_cache, v_cache, page_table, cache_lens, cos, sin, q_weight, k_weight, positions, new_lens, q_out)
    scalars = eps, interleaved
    done = _APPEND.call(tensors, scalars)
    if done is not NotImplemented:
        return done
    a, rows, tables = _append_args(k, v, k_cache, v_cache, page_table, cache_lens, cos, sin, q, q_weight, k_weight,
                                   positions, new_lens, eps, interleaved, q_out)
    if any(r is not t for r, t in zip(rows, (k, v, q))) or tables[0] is not cos:      # the call on copies of them
        return paged_kv_append(rows[0], rows[1], k_cache, v_cache, page_table, cache_lens, *tables, q=rows[2],
                               q_weight=q_weight, k_weight=k_weight, positions=positions, new_lens=new_lens,
                               eps=float(eps), interleaved=bool(interleaved), q_out=q_out)
    scalars = float(eps), bool(interleaved)
    own_out = q is not None and q_out is None
    return _APPEND.add(tensors, scalars, a,
                       inputs=(("k", 0), ("v", 1), ("q", 2), ("k_cache", 3), ("v_cache", 4), ("page_table", 5),
                               ("cache_lens", 6), ("cos", 7), ("sin", 8), ("q_weight", 9), ("k_weight", 10),
                               ("positions", 11), ("new_lens", 12), ("q_out", 13)),
                       outputs=(("q_out", 2),) if own_out else (),
                       returns=(0 if own_out else (None if q is None else -14),))


def _append_args(k, v, k_cache, v_cache, page_table, cache_lens, cos, sin, q, q_weight, k_weight, positions,
                 new_lens, eps, interleaved, q_out):
    """Checks a call: every field of it but the pointers, its rows and tables as the kernel takes them."""
    if k.ndim != 4 or k.shape != v.shape:
        raise ValueError("k and v must both be 4D (Batch, KV_Heads, SeqLen, Dim).")
    if not k.is_cuda or v.device != k.device:
        raise ValueError("k and v must be on the same CUDA device.")
    if k.dtype != v.dtype:
        raise ValueError("k and v must have the same data type.")
    if k.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("paged_kv_append supports float16 and bfloat16")
    batch, heads, tokens, dim = k.shape
    device = k.device
    if dim % 8 or not 0 < dim <= 256:
        raise ValueError("the head dimension must be a multiple of 8 up to 256")
    check_no_grad("paged_kv_append", "", k, v, q, q_weight, k_weight, cos, sin, k_cache, v_cache, q_out)
    _check_cache(k_cache, v_cache, page_table, cache_lens, new_lens, batch, heads, dim, k.dtype, device)
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if q is None and (q_weight is not None or q_out is not None):
        raise ValueError("q_weight and q_out need q")
    k, v, q = rows_view(k), rows_view(v), rows_view(q)
    a = _lib.PagedKvAppendArgs()
    if cos is not None:
        a.rotary_dim = check_table(cos, sin, dim, device)
        cos, sin = aligned_table(cos, sin)
        a.table_rows, a.table_stride = cos.shape[0], cos.stride(0)
    weight_dtype = check_weights(dim, k.dtype, device, q_weight, k_weight)
    a.position_stride_b, a.position_stride_t, a.positions_are_int64 = check_positions(positions, batch, tokens, device)
    if q is not None:
        if q.ndim != 4 or (q.shape[0], q.shape[2], q.shape[3]) != (batch, tokens, dim):
            raise ValueError("q must be (Batch, Heads, SeqLen, Dim) like k.")
        if q.device != device or q.dtype != k.dtype:
            raise ValueError("q must have the device and data type of k.")
        a.zero_padding = 1 if q_out is None else 0
        qo = empty_rows(q) if q_out is None else check_out(q_out, q, "q_out")
        a.heads_q = q.shape[1]
        a.q_stride_b, a.q_stride_h, a.q_stride_t, _ = q.stride()
        a.qo_stride_b, a.qo_stride_h, a.qo_stride_t, _ = qo.stride()
    a.batch, a.tokens, a.heads_kv = batch, tokens, heads
    a.k_stride_b, a.k_stride_h, a.k_stride_t, _ = k.stride()
    a.v_stride_b, a.v_stride_h, a.v_stride_t, _ = v.stride()
    a.kc_stride_p, a.kc_stride_h, a.kc_stride_s, _ = k_cache.stride()
    a.vc_stride_p, a.vc_stride_h, a.vc_stride_s, _ = v_cache.stride()
    a.num_pages, a.page_size = k_cache.shape[0], k_cache.shape[2]
    a.max_pages, a.page_table_stride = page_table.shape[1], page_table.stride(0)
    a.head_dim, a.interleaved = dim, 1 if interleaved else 0
    a.dtype, a.weight_dtype, a.eps = _lib.dtype_enum(k.dtype), _lib.dtype_enum(weight_dtype), eps
    return a, (k, v, q), (cos, sin)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    page_table: torch.Tensor, cache_lens: torch.Tensor, *,
                    new_lens: torch.Tensor | None = None, tree_mask: torch.Tensor | None = None,
                    qk_scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(qk_scale * q K^T) V of a step's queries q (Batch, Heads, SeqLen, Dim) over the
    cache, after ``paged_kv_append`` of the same step: query t of sequence b reads the
    cache_lens[b] tokens that were there before and those of the step's tokens j for which
    ``tree_mask`` ((SeqLen, SeqLen) or (Batch, SeqLen, SeqLen), bool) is True at [t, j]; without a
    mask the tokens j <= t.  One token per sequence is a decode step, a mask of ancestors
    scores a tree of drafts.

    float16 or bfloat16, heads a multiple of the cache's, Dim a multiple of 8 up to 128, pages
    of a multiple of 8 tokens, qk_scale in (0, 2e38] (None: 1 / sqrt(Dim)); up to 65535 sequences, and
    their tables may name up to 2^38 tokens together, counted once per key/value head and 256 query
    rows of it (2^29 each).  Scores, maxima, sums and the output's sum are fp32; the weights are
    rounded to the inputs' type before they multiply V, and where more than 128 queries share a
    cache head every fourth pair of them is computed to 7.5e-5.

    A query that sees no token gives zeros.  Slots that hold none of the sequence's tokens are never
    used; NaN and infinities of the step's tokens reach only the queries that see them.  (An infinite
    value of an earlier token gives infinity, or NaN where its weight rounds to zero.)  Rows behind
    new_lens[b] are padding: they stay as they are in a given ``out`` (which overlaps no input) and
    are zero in one made here.  Sequences may share pages.  A length or page outside the table or
    the cache is not followed: that sequence's rows mean nothing, and ``raise_on_device_error()``
    names it."""
    tensors, scalars = (q, k_cache, v_cache, page_table, cache_lens, new_lens, tree_mask, out), (qk_scale,)
    done = _ATTENTION.call(tensors, scalars)
    if done is not NotImplemented:
        return done
    a = _attention_args(q, k_cache, v_cache, page_table, cache_lens, new_lens, tree_mask, qk_scale, out)
    if qk_scale is not None:
        qk_scale = float(qk_scale)
    # the kernel's copies want the queries' rows on 16-byte boundaries
    if q.stride(-1) != 1 or q.data_ptr() % 16 or any([s % 8 or s == 0 for s in q.stride()[:-1]]):
        return paged_attention(empty_rows(q).copy_(q), k_cache, v_cache, page_table, cache_lens, new_lens=new_lens,
                               tree_mask=tree_mask, qk_scale=qk_scale, out=out)
    scalars = (qk_scale,)
    with torch.cuda.device(q.device):
        a.workspace_bytes = _lib.lib().b200k_paged_attention_workspace_bytes(ctypes.byref(a))
    return _ATTENTION.add(tensors, scalars, a,
                          inputs=(("q", 0), ("k_cache", 1), ("v_cache", 2), ("page_table", 3), ("cache_lens", 4),
                                  ("new_lens", 5), ("tree_mask", 6), ("out", 7)),
                          outputs=(("out", 0),) if out is None else (), workspace="workspace",
                          returns=(0 if out is None else -8,))


def _attention_args(q, k_cache, v_cache, page_table, cache_lens, new_lens, tree_mask, qk_scale, out):
    """Checks a call; every field of it but the pointers."""
    if q.ndim != 4:
        raise ValueError("q must be 4D (Batch, Heads, SeqLen, Dim).")
    if not q.is_cuda:
        raise ValueError("q must be on a CUDA device.")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("paged_attention supports float16 and bfloat16")
    batch, heads, tokens, dim = q.shape
    device = q.device
    check_no_grad("paged_attention", "", q, k_cache, v_cache, out)
    heads_kv = k_cache.shape[1] if k_cache.ndim == 4 else 0
    _check_cache(k_cache, v_cache, page_table, cache_lens, new_lens, batch, heads_kv, dim, q.dtype, device)
    if heads_kv == 0 or heads % heads_kv:
        raise ValueError("the number of query heads must be a multiple of the cache's heads.")
    if heads > 128 * heads_kv:
        raise ValueError("at most 128 query heads may share a cache head.")
    if dim % 8 or not 0 < dim <= 128:
        raise ValueError("the head dimension must be a multiple of 8 up to 128")
    if k_cache.shape[2] % 8:
        raise ValueError("pages must hold a multiple of 8 tokens")
    qk_scale = 1.0 / math.sqrt(dim) if qk_scale is None else float(qk_scale)
    if not 0.0 < qk_scale <= 2.0e38:
        raise ValueError("qk_scale must be positive and at most 2e38")
    for c, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        if c.data_ptr() % 16 or any(s % 8 for s in c.stride()[:3]):
            raise ValueError(f"{name} must start on a 16-byte boundary with strides of whole 16-byte units")
    a = _lib.PagedAttentionArgs()
    if tree_mask is not None:
        if tree_mask.dtype != torch.bool:
            raise TypeError("tree_mask must be bool")
        if tree_mask.device != device:
            raise ValueError("tree_mask must be on the device of the queries.")
        if tree_mask.shape == (tokens, tokens):
            a.mask_stride_t, a.mask_stride_j = tree_mask.stride()
        elif tree_mask.shape == (batch, tokens, tokens):
            a.mask_stride_b, a.mask_stride_t, a.mask_stride_j = tree_mask.stride()
        else:
            raise ValueError(f"tree_mask must be ({tokens}, {tokens}) or ({batch}, {tokens}, {tokens}), "
                             f"got {tuple(tree_mask.shape)}")
    a.zero_padding = 1 if out is None else 0
    o = empty_rows(q) if out is None else check_out(out, q, "out")
    a.batch, a.tokens, a.heads_q, a.heads_kv = batch, tokens, heads, heads_kv
    a.q_stride_b, a.q_stride_h, a.q_stride_t, _ = q.stride()
    a.o_stride_b, a.o_stride_h, a.o_stride_t, _ = o.stride()
    a.kc_stride_p, a.kc_stride_h, a.kc_stride_s, _ = k_cache.stride()
    a.vc_stride_p, a.vc_stride_h, a.vc_stride_s, _ = v_cache.stride()
    a.num_pages, a.page_size = k_cache.shape[0], k_cache.shape[2]
    a.max_pages, a.page_table_stride = page_table.shape[1], page_table.stride(0)
    a.head_dim, a.dtype, a.qk_scale = dim, _lib.dtype_enum(q.dtype), qk_scale
    return a
