"""`grouped_matmul_tp_persistent`: the tree-ordered matmul for rows grouped by expert, ragged sizes.

Row i of the result is row i of A times the weight of the group that row i belongs to.  The arithmetic is that of
`matmul_tp_persistent(..., node_dtype=torch.float32)`: K is summed in fp32 in an order that depends on (K, leaf) alone
and rounded once, so a row's bits depend neither on the other rows, nor on the sizes of the groups, nor -- with the
layer's leaf -- on the tensor-parallel degree; they equal what `matmul_tp_persistent` gives for the group's rows alone.
There is no CPU path.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _lib
from .row_groups import empty, launch, need_cuda, overlap, overwritten, refuse_grad
from .tree_based_matmul import _DTYPE_CODE


def _aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """t [.., rows, cols] with contiguous elements in a row, 16-byte aligned rows; of matrices, one behind the other or their
    rows in turn.  Anything else is copied once."""
    cols = t.shape[-1]
    *steps, last = t.stride()
    # (a stride that is never stepped says nothing, but the kernel's tensor maps read it all the same)
    if (last == 1 or cols == 1) and t.data_ptr() % 16 == 0:
        for s in steps:
            if s % 8 or s < cols:
                break
        else:
            if len(steps) == 1:
                return t
            outer, inner = steps
            if outer >= (t.shape[1] - 1) * inner + cols or inner >= (t.shape[0] - 1) * outer + cols or t.shape[0] == 1:
                return t
    pad = (cols + 7) // 8 * 8
    buf = torch.empty(t.shape[:-1] + (pad,), dtype=t.dtype, device=t.device)
    buf[..., :cols].copy_(t)
    return buf[..., :cols]


def _check_offsets(what: str, offsets: torch.Tensor, groups: int) -> torch.Tensor:
    if offsets.dtype != torch.int32:
        raise ValueError(f"{what}: offsets must be int32, got {offsets.dtype}")
    if not 1 <= groups <= _lib.MAX_GROUPS:
        raise ValueError(f"{what}: the number of groups must be in 1 .. {_lib.MAX_GROUPS}, got {groups}")
    if offsets.dim() != 1 or offsets.numel() != groups + 1:
        raise ValueError(f"{what}: offsets must have {groups + 1} entries, got {tuple(offsets.shape)}")
    return offsets.contiguous()


def _check_types(what: str, a: torch.Tensor, b: torch.Tensor) -> None:
    if a.dtype not in _DTYPE_CODE:
        raise NotImplementedError(f"{what}: dtype {a.dtype} is not supported by the sm_100a kernel")
    if b.dtype != a.dtype:
        raise ValueError(f"{what}: operands of {a.dtype} and {b.dtype}")


def grouped_matmul_tp_persistent(A: torch.Tensor, W: torch.Tensor, offsets: torch.Tensor, *, leaf: Optional[int] = None,
                                 out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                                 max_ctas: int = 0) -> torch.Tensor:
    """C[i] = A[i] @ W[g]^T for offsets[g] <= i < offsets[g + 1]; returns [M, N].

    A: [M, K], rows sorted by group; W: [G, N, K] (used in place when its K or its N is contiguous); offsets: [G + 1]
    int32 on the device, non-decreasing, as `group_rows` / `route_topk` return them.  Rows of no group are zero in a new
    result and left as they were in `out`.
    `leaf`: leaf width of the tree over K (a multiple of 64 that divides K); a row-split layer passes
    `leaf_for_fp32_nodes(K_total, max_tp)`.  Default: K is one leaf, and may then be any size.
    `out_dtype=torch.float32`: the unrounded sums, what a tensor-parallel rank contributes to the cross-rank levels.
    `tbik.autograd.tree_grouped_linear` is the differentiable form."""
    refuse_grad("grouped_matmul_tp_persistent", "use tbik.autograd.tree_grouped_linear", A, W, out)
    return _grouped(A, W, offsets, leaf, out, out_dtype, max_ctas)


def _grouped(A, W, offsets, leaf=None, out=None, out_dtype=None, max_ctas=0):
    what = "grouped_matmul_tp_persistent"
    if A.dim() != 2 or W.dim() != 3 or A.shape[1] != W.shape[2]:
        raise ValueError(f"{what}: A must be [M, K] and W [G, N, K], got {tuple(A.shape)} and {tuple(W.shape)}")
    _check_types(what, A, W)
    M, K = A.shape
    G, N, _ = W.shape
    offsets = _check_offsets(what, offsets, G)
    if not 1 <= K < 1 << 30 or N >= 1 << 30:
        raise ValueError(f"{what}: K in 1 .. 2^30 - 1 and N below 2^30, got {K} and {N}")
    if leaf is not None and (leaf < 64 or leaf % 64 or K % leaf):
        raise ValueError(f"{what}: leaf must be a multiple of 64 that divides K = {K}, got {leaf}")
    if out_dtype not in (None, A.dtype, torch.float32):
        raise ValueError(f"{what}: out_dtype is the operand type or torch.float32")
    dev = need_cuda(what, A, W, offsets)
    c_dtype = out_dtype or A.dtype
    if out is None:
        C = empty(M, N, c_dtype, dev)
    else:
        C = out
        if C.shape != (M, N) or C.dtype != c_dtype or C.device != dev or (N > 1 and C.stride(1) != 1) or \
                (M > 1 and C.stride(0) < N):
            raise ValueError(f"{what}: out must be a row-major {(M, N)} tensor of {c_dtype} on {dev}")
        if overlap(C, A) or overlap(C, W):
            raise ValueError(f"{what}: out overlaps an operand")
    if M == 0 or N == 0:
        return C
    A = _aligned_rows(A)
    # K contiguous as torch.nn.Linear stores a weight, or N contiguous (its transposed view): both are read in place
    layout = _lib.W_K_CONTIGUOUS
    if W.stride(2) != 1 and W.stride(1) == 1:
        layout = _lib.W_N_CONTIGUOUS
        W = W.transpose(1, 2)
    W = _aligned_rows(W)
    step_w, ldw, _ = W.stride()
    code = _DTYPE_CODE[A.dtype]
    launch("tbik_grouped_gemm", dev, A.data_ptr(), W.data_ptr(), C.data_ptr(), offsets.data_ptr(), M, N, K, G, A.stride(0), ldw,
           step_w, max(C.stride(0), N), layout, code, _lib.DTYPE_FP32 if c_dtype == torch.float32 else code, leaf or 0, out is None,
           max_ctas)
    if out is not None:
        overwritten(out)
    return C


def grouped_weight_gradient(dC: torch.Tensor, A: torch.Tensor, offsets: torch.Tensor, *,
                            out_dtype: Optional[torch.dtype] = None, max_ctas: int = 0) -> torch.Tensor:
    """dW[g] = dC[rows of g]^T @ A[rows of g], [G, N, K]: the gradient of `grouped_matmul_tp_persistent` with respect to W.

    The rows of a group are added in their order in fp32 and rounded once (not at all with out_dtype=torch.float32), so
    the bits depend on the group's rows alone.  The gradient of an empty group is zero."""
    refuse_grad("grouped_weight_gradient", "it is a gradient itself", dC, A)
    return _weight_gradient(dC, A, offsets, out_dtype, max_ctas)


def _weight_gradient(dC, A, offsets, out_dtype=None, max_ctas=0):
    what = "grouped_weight_gradient"
    if dC.dim() != 2 or A.dim() != 2 or dC.shape[0] != A.shape[0]:
        raise ValueError(f"{what}: dC must be [M, N] and A [M, K], got {tuple(dC.shape)} and {tuple(A.shape)}")
    _check_types(what, A, dC)
    if out_dtype not in (None, A.dtype, torch.float32):
        raise ValueError(f"{what}: out_dtype is the operand type or torch.float32")
    groups = offsets.numel() - 1
    offsets = _check_offsets(what, offsets, groups)
    M, N, K = A.shape[0], dC.shape[1], A.shape[1]
    if N >= 1 << 30 or K >= 1 << 30:
        raise ValueError(f"{what}: N and K below 2^30, got {N} and {K}")
    dev = need_cuda(what, A, dC, offsets)
    dW = torch.empty((groups, N, K), dtype=out_dtype or A.dtype, device=dev)
    if N == 0 or K == 0:
        return dW
    if M == 0:
        return dW.zero_()
    A, dC = _aligned_rows(A), _aligned_rows(dC)
    code = _DTYPE_CODE[A.dtype]
    launch("tbik_grouped_gemm_wgrad", dev, dC.data_ptr(), A.data_ptr(), dW.data_ptr(), offsets.data_ptr(), M, N, K, groups,
           dC.stride(0), A.stride(0), code, _lib.DTYPE_FP32 if dW.dtype == torch.float32 else code, max_ctas)
    return dW
