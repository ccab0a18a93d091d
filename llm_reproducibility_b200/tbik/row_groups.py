"""Rows grouped by an id, and the router that gives rows their ids.

`group_rows(ids, G)` sorts the rows of a batch by expert or by adapter, stably; `route_topk(logits, k)` picks each
token's k experts with their softmax weights and groups the (token, slot) rows that result.  Both leave everything on
the device: nothing here waits for the GPU, so both can be captured in a CUDA graph.  There is no CPU path.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from .. import _lib
from .tree_based_matmul import _raw_stream

_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_LOGITS_CODE = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16, torch.float32: _lib.DTYPE_FP32}


class RowGroups(NamedTuple):
    """Rows sorted by group (int32 tensors).

    order[p] is the row that comes p-th, rows of one group in their own order; position is its inverse;
    offsets[g] .. offsets[g + 1] are group g's places.  Rows of no group come last, behind offsets[-1]."""
    order: torch.Tensor
    position: torch.Tensor
    offsets: torch.Tensor


class Routing(NamedTuple):
    weights: torch.Tensor  # [T, k] float32, largest first
    ids: torch.Tensor      # [T, k] int32
    groups: RowGroups      # of the T * k flat entries of ids: row i is token i // k


def launch(name: str, device: torch.device, *args) -> None:
    """Call the library's function `name` with `args` and, as its last argument, the current stream of `device`, which is
    made the current device for the call."""
    fn, index = getattr(_lib.lib(), name), device.index
    if _current_device() == index:  # (the callers hold CUDA tensors: there is a device)
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _raw_stream(index))
    if rc != 0:
        _lib.check(rc, name)


def empty(rows: int, cols: int, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """torch.empty((rows, cols)) by the quicker of its ways: a microsecond of a decode step's few."""
    return torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=device)


def need_cuda(what: str, *tensors: torch.Tensor) -> torch.device:
    """The tensors' one CUDA device."""
    device, index = tensors[0].device, tensors[0].get_device()  # (numbers compare quicker than devices; -1 off the GPU)
    for t in tensors:
        if t.get_device() != index or index < 0:
            if not t.is_cuda or index < 0:
                raise RuntimeError(f"{what} needs CUDA tensors (there is no CPU fallback)")
            raise RuntimeError(f"{what}: tensors on {device} and {t.device}")
    return device


def refuse_grad(what: str, instead: str, *tensors) -> None:
    """A call that records no gradient must not swallow one, backward or forward: of an operand, or of the tensor that it
    overwrites (which may be None)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{what} records no gradient: {instead}")
    if getattr(forward_ad, "_current_level", 0) >= 0:  # inside a dual level: a tangent says nothing through requires_grad
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{what} carries no tangent (there is no forward-mode derivative)")


def overwritten(out: torch.Tensor) -> None:
    """Tells autograd that a kernel has written into a caller's tensor, as torch's own operators do: a backward pass that saved
    what it held before then fails instead of reading what it holds now."""
    increment_version(out)


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors may share memory: whether the spans that they step over meet, unless both are columns of one
    matrix, each its own."""
    def span(t):
        if t.numel() == 0:
            return 0, 0
        steps = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (steps + 1) * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    if a0 >= b1 or b0 >= a1:
        return False
    if a.dim() == b.dim() == 2 and a.stride() == b.stride() and a.stride(1) == 1 and a.element_size() == b.element_size():
        pitch = a.stride(0) * a.element_size()
        if pitch:
            at = (b0 - a0) % pitch  # b's first byte in a row of the matrix that begins with a's
            return at < a.shape[1] * a.element_size() or at + b.shape[1] * b.element_size() > pitch
    return True


def _empty_groups(M: int, groups: int, device: torch.device):
    """An empty RowGroups and the kernels' workspace (pointer, bytes), in one allocation."""
    nbytes = _lib.lib().tbik_group_workspace_bytes(M, groups)
    sizes = [M, M, groups + 1, nbytes // 4]
    buf = torch.empty_strided((sum(sizes),), (1,), dtype=torch.int32, device=device)
    order, position, offsets, ws = buf.split_with_sizes(sizes)
    return RowGroups(order, position, offsets), ws.data_ptr(), nbytes


def _check_groups(num_groups: int) -> None:
    if not 1 <= num_groups <= _lib.MAX_GROUPS:
        raise ValueError(f"the number of groups must be in 1 .. {_lib.MAX_GROUPS}, got {num_groups}")


def group_rows(ids: torch.Tensor, num_groups: int) -> RowGroups:
    """Stable grouping of the rows whose ids are given (int32, flattened).  An id outside 0 .. num_groups - 1 (-1, say:
    a row without adapter, a padded token) puts its row in no group."""
    if ids.dtype != torch.int32:
        raise ValueError(f"group_rows: ids must be int32, got {ids.dtype}")
    _check_groups(num_groups)
    if ids.numel() >= 1 << 31:
        raise ValueError("group_rows: fewer than 2^31 rows")
    dev = need_cuda("group_rows", ids)
    ids = ids.contiguous()
    g, ws, nbytes = _empty_groups(ids.numel(), num_groups, dev)
    launch("tbik_group_rows", dev, ids.data_ptr(), ids.numel(), num_groups, g.order.data_ptr(), g.position.data_ptr(),
           g.offsets.data_ptr(), ws, nbytes)
    return g


def _check_logits(logits: torch.Tensor, k: int) -> torch.Tensor:
    if logits.dim() != 2:
        raise ValueError(f"route_topk: logits must be [tokens, experts], got {tuple(logits.shape)}")
    if logits.dtype not in _LOGITS_CODE:
        raise NotImplementedError(f"route_topk: dtype {logits.dtype} is not supported")
    T, E = logits.shape
    if not 1 <= E <= _lib.MAX_GROUPS:
        raise ValueError(f"route_topk: the number of experts must be in 1 .. {_lib.MAX_GROUPS}, got {E}")
    if not 1 <= k <= min(E, _lib.MAX_TOPK):
        raise ValueError(f"route_topk: k must be in 1 .. {min(E, _lib.MAX_TOPK)}, got {k}")
    if T * k >= 1 << 31:
        raise ValueError("route_topk: fewer than 2^31 (token, slot) rows")
    if not logits.is_cuda:
        need_cuda("route_topk", logits)
    # rows may be strided or broadcast; the experts of a row must be contiguous
    return logits if logits.stride(1) == 1 or E == 1 else logits.contiguous()


def route_topk(logits: torch.Tensor, k: int, *, renormalize: bool = True) -> Routing:
    """The k experts with the largest logits of each token, their weights, and the rows grouped by expert.

    Equal logits: the lower index first.  `renormalize`: the weights are the softmax over the k chosen, else their
    share of the softmax over all experts.  -inf masks an expert (weight 0); a token whose experts are all masked gets
    weights 0.  `tbik.autograd.tree_route_topk` is the differentiable form."""
    refuse_grad("route_topk", "use tbik.autograd.tree_route_topk", logits)
    return _route(logits, k, renormalize)


def _route(logits: torch.Tensor, k: int, renormalize: bool) -> Routing:
    logits = _check_logits(logits, k)
    T, E = logits.shape
    dev = logits.device
    weights, ids = empty(T, k, torch.float32, dev), empty(T, k, torch.int32, dev)
    g, ws, nbytes = _empty_groups(T * k, E, dev)
    launch("tbik_route_topk", dev, logits.data_ptr(), logits.stride(0), T, E, k, _LOGITS_CODE[logits.dtype], renormalize,
           weights.data_ptr(), ids.data_ptr(), g.order.data_ptr(), g.position.data_ptr(), g.offsets.data_ptr(), ws, nbytes)
    return Routing(weights, ids, g)


def _route_backward(logits, weights, ids, dweights, renormalize: bool) -> torch.Tensor:
    logits = _check_logits(logits, ids.shape[1])
    T, E = logits.shape
    if dweights.dtype != torch.float32 or not dweights.is_contiguous():
        dweights = dweights.to(torch.float32).contiguous()
    dlogits = empty(T, E, logits.dtype, logits.device)
    launch("tbik_route_topk_backward", logits.device, logits.data_ptr(), logits.stride(0), T, E, ids.shape[1],
           _LOGITS_CODE[logits.dtype], renormalize, weights.data_ptr(), ids.data_ptr(), dweights.data_ptr(), dlogits.data_ptr(), E)
    return dlogits
