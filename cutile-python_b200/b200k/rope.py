"""Norm of every query and key head and rotation by position, one pass; with its gradient.

The operators between a projection GEMM and ``cutile_fmha``: both take and give the attention
wrappers' (Batch, Heads, SeqLen, Dim) views, so queries and keys may lie side by side in one
(Batch, SeqLen, Heads, Dim) projection.  No counterpart among the reference's samples.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad

from . import _lib


def rope_table(max_positions: int, rotary_dim: int, theta: float = 10000.0,
               device: torch.device | str | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """cos, sin of position * theta^(-2 i / rotary_dim), each (max_positions, rotary_dim / 2)
    float32.  The angles are taken in float64: at position 10^5 a float32 angle is already
    off by 4e-3."""
    if max_positions <= 0 or rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("max_positions must be positive, rotary_dim positive and even")
    inv = theta ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def rows_view(t: torch.Tensor | None) -> torch.Tensor | None:
    """The tensor itself where its rows are contiguous, else a copy that has them so."""
    return t if t is None or t.stride(-1) == 1 or not t.numel() else t.contiguous()


def check_no_grad(name: str, instead: str, *tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{name} is not recorded by autograd: call it under torch.no_grad(){instead}")
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError(f"{name} is not recorded by autograd: it passes no tangents on")


def check_out(t: torch.Tensor, like: torch.Tensor, name: str) -> torch.Tensor:
    if t.shape != like.shape or t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name} must have the shape, dtype and device of its input")
    if t.numel() and t.stride(-1) != 1 or any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape)):
        raise ValueError(f"{name} must have contiguous rows that do not overlap")
    return t


def check_table(cos: torch.Tensor, sin: torch.Tensor, dim: int, device: torch.device) -> int:
    """rotary_dim of a pair of tables."""
    if cos.ndim != 2 or cos.shape != sin.shape:
        raise ValueError("cos and sin must both be (positions, rotary_dim / 2)")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise TypeError("cos and sin must be float32")
    if cos.device != device or sin.device != device:
        raise ValueError("cos and sin must be on the device of the rows")
    rotary = 2 * cos.shape[1]
    if rotary > dim or rotary % 16:
        raise ValueError(f"rotary_dim must be a multiple of 16 up to the head dimension (got {rotary} of {dim})")
    if cos.shape[0] == 0:
        raise ValueError("the rotation table has no positions")
    return rotary


def check_positions(positions: torch.Tensor | None, batch: int, tokens: int, device: torch.device):
    """(batch stride, token stride, is int64)"""
    if positions is None:
        return 0, 0, 0
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError("positions must be int32 or int64")
    if positions.device != device:
        raise ValueError("positions must be on the device of the rows")
    if positions.shape == (tokens,):
        stride_b, stride_t = 0, positions.stride(0)
    elif positions.shape == (batch, tokens):
        stride_b, stride_t = positions.stride()
    else:
        raise ValueError(f"positions must be ({tokens},) or ({batch}, {tokens}), got {tuple(positions.shape)}")
    return stride_b, stride_t, int(positions.dtype == torch.int64)


def check_weights(dim: int, dtype: torch.dtype, device: torch.device, *weights) -> torch.dtype:
    """The weights' dtype (the rows' where there are none)."""
    found = None
    for w in weights:
        if w is None:
            continue
        if w.shape != (dim,):
            raise ValueError(f"norm weights must be ({dim},), got {tuple(w.shape)}")
        if w.device != device:
            raise ValueError("norm weights must be on the device of the rows")
        if w.dtype not in (dtype, torch.float32):
            raise TypeError("norm weights must have the rows' dtype or be float32")
        if w.stride(0) != 1 and dim > 1:
            raise ValueError("norm weights must be contiguous")
        if found is not None and w.dtype != found:
            raise TypeError("both norm weights must have one dtype")
        found = w.dtype
    return found or dtype


def _check_rows(q: torch.Tensor, k: torch.Tensor) -> None:
    if q.ndim != 4 or k.ndim != 4:
        raise ValueError("q and k must be 4D (Batch, Heads, SeqLen, Dim).")
    if q.shape[0] != k.shape[0] or q.shape[2:] != k.shape[2:]:
        raise ValueError("q and k must agree in Batch, SeqLen and Dim.")
    if q.device != k.device or not q.is_cuda:
        raise ValueError("q and k must be on the same CUDA device.")
    if q.dtype != k.dtype:
        raise ValueError("q and k must have the same data type.")
    if q.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise TypeError("q and k must be float16, bfloat16 or float32")
    if q.shape[3] % 8 or not 0 < q.shape[3] <= 256:
        raise ValueError("the head dimension must be a multiple of 8 up to 256")


def empty_rows(like: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(like, memory_format=torch.contiguous_format)


def aligned_table(cos, sin):
    """The tables themselves, or 16-byte aligned copies of a common layout."""
    if cos is None or sin is None or not cos.numel() or (
            (cos.data_ptr() | sin.data_ptr()) % 16 == 0 and cos.stride() == sin.stride()
            and cos.stride(-1) == 1 and cos.stride(0) % 4 == 0 and cos.stride(0) >= cos.shape[1]):
        return cos, sin
    width = -(-cos.shape[1] // 4) * 4                # rows of whole 16-byte units
    return tuple(torch.empty(t.shape[0], width, dtype=t.dtype, device=t.device)[:, :t.shape[1]].copy_(t)
                 for t in (cos, sin))


_FORWARD = _lib.LayoutPlans("b200k_qk_norm_rope", _lib.QkNormRopeArgs)
_BACKWARD = _lib.LayoutPlans("b200k_qk_norm_rope_backward", _lib.QkNormRopeArgs)


def _fill(a, q, k, q_out, k_out, q_weight, k_weight, cos, sin, positions, eps, interleaved):
    """Checks the rest of a call and fills in every field but its pointers; the tables to call with."""
    batch, heads, tokens, dim = q.shape
    rotary = check_table(cos, sin, dim, q.device)
    cos, sin = aligned_table(cos, sin)
    weight_dtype = check_weights(dim, q.dtype, q.device, q_weight, k_weight)
    a.table_rows, a.table_stride = cos.shape[0], cos.stride(0)
    a.position_stride_b, a.position_stride_t, a.positions_are_int64 = check_positions(
        positions, batch, tokens, q.device)
    a.batch, a.tokens, a.heads_q, a.heads_kv = batch, tokens, heads, k.shape[1]
    a.q_stride_b, a.q_stride_h, a.q_stride_t, _ = q.stride()
    a.k_stride_b, a.k_stride_h, a.k_stride_t, _ = k.stride()
    a.qo_stride_b, a.qo_stride_h, a.qo_stride_t, _ = q_out.stride()
    a.ko_stride_b, a.ko_stride_h, a.ko_stride_t, _ = k_out.stride()
    a.head_dim, a.rotary_dim, a.interleaved = dim, rotary, 1 if interleaved else 0
    a.dtype, a.weight_dtype, a.eps = _lib.dtype_enum(q.dtype), _lib.dtype_enum(weight_dtype), eps
    return cos, sin


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor,
                 q_weight: torch.Tensor | None, k_weight: torch.Tensor | None,
                 cos: torch.Tensor, sin: torch.Tensor,
                 positions: torch.Tensor | None = None, *,
                 eps: float = 1e-6, interleaved: bool = False,
                 q_out: torch.Tensor | None = None,
                 k_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Every row of q (Batch, Heads, SeqLen, Dim) and k (Batch, KV_Heads, SeqLen, Dim), float16,
    bfloat16 or float32, divided by its root mean square, times the (Dim,) weight, with its
    first rotary_dim = 2 * cos.shape[1] values turned by the token's position: one launch, each
    row read and written once, fp32 inside.

    A weight of None leaves that norm out (rotation alone).  ``cos`` / ``sin`` are tables by
    position (``rope_table``); ``positions`` is (SeqLen,) or (Batch, SeqLen), None = 0, 1, 2, ...
    Pairs are (i, i + rotary_dim / 2), or neighbours with ``interleaved``.  ``q_out`` / ``k_out``
    may be q / k themselves and overlap nothing else.  A position outside the table makes the rotated
    values of its rows NaN, and ``raise_on_device_error()`` names it."""
    tensors, scalars = (q, k, q_weight, k_weight, cos, sin, positions, q_out, k_out), (eps, interleaved)
    done = _FORWARD.call(tensors, scalars)
    if done is not NotImplemented:
        return done
    _check_rows(q, k)
    check_no_grad("qk_norm_rope", " and take gradients from qk_norm_rope_backward", q, k, q_weight, k_weight,
                  cos, sin, q_out, k_out)
    if q_out is not None:
        check_out(q_out, q, "q_out")
    if k_out is not None:
        check_out(k_out, k, "k_out")
    a = _lib.QkNormRopeArgs()
    rows = rows_view(q), rows_view(k)
    tables = _fill(a, *rows, empty_rows(q) if q_out is None else q_out, empty_rows(k) if k_out is None else k_out,
                   q_weight, k_weight, cos, sin, positions, eps, interleaved)
    if rows[0] is not q or rows[1] is not k or tables[0] is not cos:      # the call on copies of them
        return qk_norm_rope(*rows, q_weight, k_weight, *tables, positions, eps=float(eps),
                            interleaved=bool(interleaved), q_out=q_out, k_out=k_out)
    scalars = float(eps), bool(interleaved)
    outputs = [f for f in (("q_out", 0) if q_out is None else None, ("k_out", 1) if k_out is None else None) if f]
    numbers = iter(range(2))
    return _FORWARD.add(tensors, scalars, a,
                        inputs=(("q", 0), ("k", 1), ("q_weight", 2), ("k_weight", 3), ("cos", 4), ("sin", 5),
                                ("positions", 6), ("q_out", 7), ("k_out", 8)),
                        outputs=outputs,
                        returns=(next(numbers) if q_out is None else -8, next(numbers) if k_out is None else -9))


def qk_norm_rope_backward(dq: torch.Tensor, dk: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                          q_weight: torch.Tensor | None, k_weight: torch.Tensor | None,
                          cos: torch.Tensor, sin: torch.Tensor,
                          positions: torch.Tensor | None = None, *,
                          eps: float = 1e-6, interleaved: bool = False):
    """Gradients (of q, of k, of q_weight, of k_weight) from the gradients ``dq``, ``dk`` of
    qk_norm_rope's outputs and its inputs (in-place outputs lose them).  The weights' gradients
    are summed in fp32 over all rows in a fixed order and rounded to the weights' dtype; None
    for a weight of None.  A position outside the table makes the gradients that depend on it NaN,
    and ``raise_on_device_error()`` names it."""
    tensors, scalars = (dq, dk, q, k, q_weight, k_weight, cos, sin, positions), (eps, interleaved)
    done = _BACKWARD.call(tensors, scalars)
    if done is not NotImplemented:
        return done
    _check_rows(q, k)
    check_no_grad("qk_norm_rope_backward", "", dq, dk, q, k, q_weight, k_weight, cos, sin)
    for g, x, name in ((dq, q, "dq"), (dk, k, "dk")):
        if g.shape != x.shape or g.dtype != x.dtype or g.device != x.device:
            raise ValueError(f"{name} must have the shape, dtype and device of {name[1]}")
    a = _lib.QkNormRopeArgs()
    rows = tuple(rows_view(t) for t in (dq, dk, q, k))
    tables = _fill(a, rows[2], rows[3], empty_rows(q), empty_rows(k), q_weight, k_weight, cos, sin, positions, eps,
                   interleaved)
    if any(r is not t for r, t in zip(rows, tensors)) or tables[0] is not cos:      # the call on copies of them
        return qk_norm_rope_backward(*rows, q_weight, k_weight, *tables, positions, eps=float(eps),
                                     interleaved=bool(interleaved))
    scalars = float(eps), bool(interleaved)
    a.dq_stride_b, a.dq_stride_h, a.dq_stride_t, _ = dq.stride()
    a.dk_stride_b, a.dk_stride_h, a.dk_stride_t, _ = dk.stride()
    if q_weight is not None or k_weight is not None:
        with torch.cuda.device(q.device):
            a.workspace_bytes = _lib.lib().b200k_qk_norm_rope_backward_workspace_bytes(ctypes.byref(a))
    outputs, returns = [("q_out", 2), ("k_out", 3)], [0, 1]
    for field, i in (("dq_weight", 4), ("dk_weight", 5)):
        returns.append(None if tensors[i] is None else len(outputs))
        if tensors[i] is not None:
            outputs.append((field, i))
    return _BACKWARD.add(tensors, scalars, a,
                         inputs=(("dq_out", 0), ("dk_out", 1), ("q", 2), ("k", 3), ("q_weight", 4), ("k_weight", 5),
                                 ("cos", 6), ("sin", 7), ("positions", 8)),
                         outputs=outputs, workspace="workspace", returns=returns)
