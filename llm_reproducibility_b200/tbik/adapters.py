"""Low-rank adapters of many requests beside a shared projection.

The rows of a batch share one base weight (`matmul_tp_persistent`, the patched row-parallel layer) while each row may
carry an adapter of its own: out = y + scale * B (A x).  `groups = group_rows(adapter_of_row, num_adapters)` is made once
a step and serves every layer; a row with id -1 has no adapter.

The sum over K runs in fp32 over at most eight leaves joined in the fixed tree, whatever else is in the batch, so a
row's bits do not depend on the batch.  A row-split layer calls `lora_shrink` on its shard of x and A with the leaf of
the unsharded K (`leaf_for_adapters`), adds the ranks' results in the rank-pair tree, and calls `lora_expand_add`.
Serving operators: they record no gradient.  There is no CPU path.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _lib
from .row_groups import RowGroups, empty, launch, need_cuda, overlap, overwritten, refuse_grad
from .tree_based_matmul import _DTYPE_CODE


def leaf_for_adapters(K_total: int, max_tp: int = 8) -> int:
    """Leaf width of the sum over a row-split layer's full K: K_total / 8, so that every rank of every tensor-parallel
    degree up to `max_tp` (a power of two up to 8) holds whole leaves."""
    if max_tp not in (1, 2, 4, 8):
        raise ValueError("max_tp must be 1, 2, 4 or 8")
    if K_total % 256 != 0:
        if max_tp > 1:
            raise ValueError(f"K = {K_total} does not split into 8 leaves that are multiples of 32")
        return (K_total + 255) // 256 * 32
    return K_total // 8


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """Rows of contiguous elements on 16-byte boundaries; anything else is copied once."""
    step, one = t.stride()
    if one == 1 and (t.shape[0] == 1 or (step % 8 == 0 and step >= t.shape[1])) and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _weights16(t: torch.Tensor) -> torch.Tensor:
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _check(what, rows, groups: RowGroups, adapters: int, rank: int, widths, *tensors) -> torch.device:
    if not 8 <= rank <= _lib.MAX_RANK or rank % 8:
        raise ValueError(f"{what}: the rank must be a multiple of 8 up to {_lib.MAX_RANK} (pad with zeros), got {rank}")
    if not 1 <= adapters <= _lib.MAX_GROUPS:
        raise ValueError(f"{what}: 1 .. {_lib.MAX_GROUPS} adapters, got {adapters}")
    for w in widths:
        if not 8 <= w < 1 << 24 or w % 8:
            raise ValueError(f"{what}: widths must be positive multiples of 8 below 2^24, got {widths}")
    order, _, offsets = groups
    if order.dtype != torch.int32 or order.shape != (rows,):
        raise ValueError(f"{what}: groups.order must be {rows} int32 values, got {tuple(order.shape)} of {order.dtype}")
    if offsets.dtype != torch.int32 or offsets.shape != (adapters + 1,):
        raise ValueError(f"{what}: groups.offsets must be {adapters + 1} int32 values, got {tuple(offsets.shape)} of {offsets.dtype}")
    return need_cuda(what, *tensors, order, offsets)


def _types(what, first, *others) -> None:
    if first.dtype not in _DTYPE_CODE:
        raise NotImplementedError(f"{what}: dtype {first.dtype} is not supported")
    for t in others:
        if t.dtype != first.dtype:
            raise ValueError(f"{what}: operands of {first.dtype} and {t.dtype}")


def _check_leaf(what, K: int, leaf: Optional[int]) -> int:
    if leaf is None:
        return 0
    if leaf < 32 or leaf % 32 or (K + leaf - 1) // leaf > 8:
        raise ValueError(f"{what}: leaf must be a multiple of 32 with at most 8 leaves covering K = {K}, got {leaf}")
    return min(leaf, (K + 31) // 32 * 32)  # (one leaf of all K, however wide it was said to be)


def _check_out(what, y, out, *others):
    """The result's tensor.  It is written while the operands are read: it may be y itself, and else overlaps nothing."""
    rows, cols = y.shape
    if out is None:
        return empty(rows, cols, y.dtype, y.device)
    if any(overlap(out, t) for t in others + (() if _same(out, y) else (y,))):
        raise ValueError(f"{what}: out overlaps an operand")
    if out.shape != y.shape or out.dtype != y.dtype or out.device != y.device or out.stride(1) != 1 or out.data_ptr() % 16 or \
            (rows > 1 and (out.stride(0) % 8 or out.stride(0) < cols)):
        raise ValueError(f"{what}: out must be like y, with contiguous 16-byte aligned rows")
    return out


def _same(out, y) -> bool:
    """Whether out is y, element for element (the stride between the rows of one row says nothing)."""
    return out is y or (out.data_ptr() == y.data_ptr() and out.shape == y.shape and out.stride()[y.shape[0] == 1:] == y.stride()[y.shape[0] == 1:])


def _launch(dev, x, y, out, A, B, scales, h, groups, T, N, K, R, adapters, dtype, leaf):
    order, _, offsets = groups
    order, offsets = order.contiguous(), offsets.contiguous()
    px = ldx = pa = py = ldy = po = ldo = pb = ps = 0
    if x is not None:
        px, ldx, pa = x.data_ptr(), x.stride(0) if T > 1 else K, A.data_ptr()
    if y is not None:
        py, ldy, po, ldo = y.data_ptr(), y.stride(0) if T > 1 else N, out.data_ptr(), out.stride(0) if T > 1 else N
        pb, ps = B.data_ptr(), scales.data_ptr()
    launch("tbik_adapters", dev, px, ldx, py, ldy, po, ldo, pa, pb, ps, 0 if h is None else h.data_ptr(), order.data_ptr(),
           offsets.data_ptr(), T, N, K, R, adapters, _DTYPE_CODE[dtype], leaf)


def lora_add(y: torch.Tensor, x: torch.Tensor, A: torch.Tensor, B: torch.Tensor, groups: RowGroups, scales: torch.Tensor, *,
             leaf: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y + scales[a] * B[a] (A[a] x), row by row with the row's adapter a; rows without adapter keep y.

    y [T, N], x [T, K], A [L, R, K], B [L, N, R] of one 16-bit type, scales [L] float32.  K, N and R multiples of 8,
    R up to 128; adapters of several ranks are padded with zeros.  Both products are taken in fp32 and the result is
    rounded once.  Returns a new tensor, or `out`, which may be y itself."""
    what = "lora_add"
    refuse_grad(what, "adapters are a serving operator", y, x, A, B, scales, out)
    shape_y, shape_x, shape_a, shape_b = y.shape, x.shape, A.shape, B.shape
    if len(shape_y) != 2 or len(shape_x) != 2 or len(shape_a) != 3 or shape_y[0] != shape_x[0] or shape_a[2] != shape_x[1] or \
            shape_b != (shape_a[0], shape_y[1], shape_a[1]):
        raise ValueError(f"{what}: y [T, N], x [T, K], A [L, R, K], B [L, N, R]; got {tuple(shape_y)}, {tuple(shape_x)}, "
                         f"{tuple(shape_a)}, {tuple(shape_b)}")
    _types(what, x, y, A, B)
    (T, K), N, (L, R, _) = shape_x, shape_y[1], shape_a
    if scales.shape != (L,) or scales.dtype != torch.float32:
        raise ValueError(f"{what}: scales must be [{L}] float32, got {tuple(scales.shape)} of {scales.dtype}")
    leaf = _check_leaf(what, K, leaf)
    dev = _check(what, T, groups, L, R, (K, N), x, y, A, B, scales)
    res = _check_out(what, y, out, x, A, B)
    if T:
        src = y if _same(res, y) else _rows16(y)
        _launch(dev, _rows16(x), src, res, _weights16(A), _weights16(B), scales.contiguous(), None, groups, T, N, K, R, L,
                x.dtype, leaf)
        if out is not None:
            overwritten(out)
    return res


def lora_shrink(x: torch.Tensor, A: torch.Tensor, groups: RowGroups, *, leaf: Optional[int] = None) -> torch.Tensor:
    """h[t] = A[a] x[t] in float32, [T, R]; zeros for rows without adapter.  With the leaf of the unsharded K
    (`leaf_for_adapters`) a rank's result is the subtree of its shard: the ranks' results add up, in the rank-pair tree,
    to the bits of the unsharded call."""
    what = "lora_shrink"
    refuse_grad(what, "adapters are a serving operator", x, A)
    if x.dim() != 2 or A.dim() != 3 or A.shape[2] != x.shape[1]:
        raise ValueError(f"{what}: x [T, K], A [L, R, K]; got {tuple(x.shape)}, {tuple(A.shape)}")
    _types(what, x, A)
    (T, K), (L, R, _) = x.shape, A.shape
    leaf = _check_leaf(what, K, leaf)
    dev = _check(what, T, groups, L, R, (K,), x, A)
    h = empty(T, R, torch.float32, dev)
    if T:
        _launch(dev, _rows16(x), None, None, _weights16(A), None, None, h, groups, T, 8, K, R, L, x.dtype, leaf)
    return h


def lora_expand_add(y: torch.Tensor, h: torch.Tensor, B: torch.Tensor, groups: RowGroups, scales: torch.Tensor, *,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y + scales[a] * B[a] h, the second half of `lora_add`: h [T, R] float32 as `lora_shrink` (summed over the ranks)
    gives it.  Returns a new tensor, or `out`, which may be y itself."""
    what = "lora_expand_add"
    refuse_grad(what, "adapters are a serving operator", y, h, B, scales, out)
    if y.dim() != 2 or h.dim() != 2 or B.dim() != 3 or y.shape[0] != h.shape[0] or B.shape[1] != y.shape[1] or B.shape[2] != h.shape[1]:
        raise ValueError(f"{what}: y [T, N], h [T, R], B [L, N, R]; got {tuple(y.shape)}, {tuple(h.shape)}, {tuple(B.shape)}")
    _types(what, y, B)
    if h.dtype != torch.float32:
        raise ValueError(f"{what}: h must be float32, got {h.dtype}")
    (T, N), (L, _, R) = y.shape, B.shape
    if scales.shape != (L,) or scales.dtype != torch.float32:
        raise ValueError(f"{what}: scales must be [{L}] float32, got {tuple(scales.shape)} of {scales.dtype}")
    dev = _check(what, T, groups, L, R, (N,), y, h, B, scales)
    res = _check_out(what, y, out, h, B)
    if T:
        src = y if _same(res, y) else _rows16(y)
        _launch(dev, None, src, res, None, _weights16(B), scales.contiguous(), _weights16(h), groups, T, N, 8, R, L, y.dtype, 0)
        if out is not None:
            overwritten(out)
    return res
