"""A key/value cache in pages: appending a step's tokens.

Caches are (Pages, KV_Heads, Page_Size, Dim) views - (page, head, slot, Dim) storage, or
(page, slot, head, Dim) storage seen through ``transpose(1, 2)``.  ``page_table`` (Batch,
Max_Pages) names the pages of each sequence in order; ``cache_lens`` (Batch,) counts the tokens
a sequence had before this step; ``new_lens`` (Batch,), where sequences bring different numbers
of tokens, says how many of the step's SeqLen rows are real.  
No counterpart among the reference's samples.
"""
from __future__ import annotations

import torch

from . import _lib
from .rope import (check_no_grad, check_out, check_positions, check_table, check_weights, launch,
                   rows_view)


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
    places in the cache (drafts of one depth in a tree share a position).  Rows behind
    new_lens[b] are padding: their cache slots stay as they are, as do their rows of a given
    ``q_out``; in a q_out made here they are zero.  A token whose page lies outside the table
    or the cache is not stored, and ``raise_on_device_error()`` names its sequence."""
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
    check_no_grad("paged_kv_append", "", k, v, q, q_weight, k_weight, k_cache, v_cache)
    _check_cache(k_cache, v_cache, page_table, cache_lens, new_lens, batch, heads, dim, k.dtype, device)
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if q is None and (q_weight is not None or q_out is not None):
        raise ValueError("q_weight and q_out need q")
    a = _lib.PagedKvAppendArgs()
    rotary = 0
    if cos is not None:
        cos, sin, rotary = check_table(cos, sin, dim, device)
        a.cos, a.sin = cos.data_ptr(), sin.data_ptr()
        a.table_rows, a.table_stride = cos.shape[0], cos.stride(0)
    weight_dtype = check_weights(dim, k.dtype, device, q_weight, k_weight)
    a.positions, a.position_stride_b, a.position_stride_t, a.positions_are_int64 = check_positions(
        positions, batch, tokens, device)
    qo = None
    if q is not None:
        if q.ndim != 4 or (q.shape[0], q.shape[2], q.shape[3]) != (batch, tokens, dim):
            raise ValueError("q must be (Batch, Heads, SeqLen, Dim) like k.")
        if q.device != device or q.dtype != k.dtype:
            raise ValueError("q must have the device and data type of k.")
        qo = torch.empty(q.shape, dtype=q.dtype, device=device) if q_out is None else check_out(q_out, q, "q_out")
        q = rows_view(q)
        a.q, a.q_out, a.q_weight, a.heads_q = q.data_ptr(), qo.data_ptr(), _lib.ptr(q_weight), q.shape[1]
        a.q_stride_b, a.q_stride_h, a.q_stride_t, _ = q.stride()
        a.qo_stride_b, a.qo_stride_h, a.qo_stride_t, _ = qo.stride()
        a.zero_padding = 1 if q_out is None else 0
    k, v = rows_view(k), rows_view(v)
    a.k, a.v, a.k_cache, a.v_cache = k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    a.k_weight = _lib.ptr(k_weight)
    a.page_table, a.cache_lens, a.new_lens = page_table.data_ptr(), cache_lens.data_ptr(), _lib.ptr(new_lens)
    a.batch, a.tokens, a.heads_kv = batch, tokens, heads
    a.k_stride_b, a.k_stride_h, a.k_stride_t, _ = k.stride()
    a.v_stride_b, a.v_stride_h, a.v_stride_t, _ = v.stride()
    a.kc_stride_p, a.kc_stride_h, a.kc_stride_s, _ = k_cache.stride()
    a.vc_stride_p, a.vc_stride_h, a.vc_stride_s, _ = v_cache.stride()
    a.num_pages, a.page_size = k_cache.shape[0], k_cache.shape[2]
    a.max_pages, a.page_table_stride = page_table.shape[1], page_table.stride(0)
    a.head_dim, a.rotary_dim, a.interleaved = dim, rotary, 1 if interleaved else 0
    a.dtype, a.weight_dtype, a.eps = _lib.dtype_enum(k.dtype), _lib.dtype_enum(weight_dtype), eps
    launch("b200k_paged_kv_append", a, device)
    return qo
