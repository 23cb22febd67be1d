"""Operators on rows held in torch tensors on the GPU, for programs that use clusters inside a model.

    lookup          vectors of a codebook by assignment, scaled; differentiable in the codebook and the scales
    group_rows      the order of rows by cluster
    to_clusters     rows to the places of their clusters, and
    from_clusters   back with weights; both differentiable
    quantize_rows   rows in 8 bits with a scale each
    product_8bit    their product with a matrix in 8 bits, or with a matrix of each cluster's own

A thin layer over the functions of the same names in include/skm_b200.h.  Every call works on the current stream of its tensors'
device (which need not be the current device), allocates its outputs and its workspace through torch, waits for nothing and can be
captured into a CUDA graph.  Calls with tensors that need no conversion take a short cut in C++ (csrc/ops_calls.cpp), which answers None
where there is something to refuse, copy or record; those are made here.  Tensors that are used on another stream than the one they were made on need `record_stream`, as with
any operator of torch.  Rows may have any distance from one another; the values of a row lie side by side, or the rows are copied
first.  Arguments that do not fit raise ValueError, and so do tensors whose memory is not there (a storage that was freed).  Gradients are
those of `backward`.  NotImplementedError is raised for what torch would record or carry along without the operators' part: tensors with a
derivative forward (torch.autograd.forward_ad), torch.jit.trace, make_fx and other tracing with fake tensors, transforms of torch.func.
(torch.compile breaks its graph at a call, and a CUDA graph captures it.)
"""
from __future__ import annotations

import sysconfig
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad

from ._lib import check, lib

try:
    from . import _ops_calls as _calls

    if _calls.built_for != f"torch {torch.__version__}, CUDA {torch.version.cuda}, {sysconfig.get_config_var('SOABI')}":
        raise ImportError(f"the short cuts were built for {_calls.built_for}")
except (ImportError, AttributeError):   # (not built, or for another torch or Python: every call takes the way through ctypes)

    class _calls:   # noqa: N801
        ordinary = lookup = lookup_grad = lookup_scale_grad = group_rows = to_clusters = from_clusters = from_clusters_grad = quantize_rows = product_8bit = staticmethod(lambda *_: None)


# (looked up once: a call on a few rows takes as long as the host takes to make it)
_op_lookup, _op_lookup_grad, _op_lookup_scale_grad = lib.skm_op_lookup, lib.skm_op_lookup_grad, lib.skm_op_lookup_scale_grad
_op_group_rows, _op_to_clusters, _op_from_clusters = lib.skm_op_group_rows, lib.skm_op_to_clusters, lib.skm_op_from_clusters
_op_from_clusters_grad, _op_quantize_rows, _op_product_8bit = lib.skm_op_from_clusters_grad, lib.skm_op_quantize_rows, lib.skm_op_product_8bit

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_ID_BITS = {torch.int32: 32, torch.uint32: 32, torch.int64: 64}
_MOST = 2**31 - 1


class RowGroups(NamedTuple):
    """Pairs (row, choice) in the order of their cluster, as `group_rows` makes them; all int32.

    order[slot]: the pair (row * m + choice) in that slot;  position[row, choice]: the slot of that pair;  offsets[c]: the first slot
    of cluster c, c = 0 .. n_clusters.  Slots from offsets[-1] on hold the pairs without a cluster."""

    order: torch.Tensor
    position: torch.Tensor
    offsets: torch.Tensor


class QuantizedRows(NamedTuple):
    """Rows in 8 bits: row i stands for values[i] * scales[i]."""

    values: torch.Tensor
    scales: torch.Tensor


# ---- checks ---------------------------------------------------------------------------------------------------------------------


def _check_memory(t, name: str) -> None:
    """A storage may be smaller than a tensor of its reaches (freed by `resize_`), or not be there at all (zeros and fakes that torch holds as
    shapes only): the address of a part of it would be followed all the same."""
    if t.numel() == 0:
        return
    storage = t.untyped_storage()
    ends = t.storage_offset() + 1 + sum((n - 1) * step for n, step in zip(t.shape, t.stride()))
    if storage.device != t.device or t._is_zerotensor() or storage.nbytes() < ends * t.element_size() or storage.data_ptr() == 0:
        raise ValueError(f"{name} has no memory, or less than its shape takes")


def _named(groups) -> dict:
    return dict(zip(RowGroups._fields, groups))


# Modes of torch in which an allocation is recorded, or made as a shape only, and what a kernel writes into it is not.  (Another torch may have
# other names for them.)
_RECORDERS = [key for key in (getattr(getattr(torch._C, "_TorchDispatchModeKey", None), name, None) for name in ("PROXY", "FAKE", "FUNCTIONAL")) if key is not None]
_modes_before_dispatch = getattr(torch._ops, "_len_torch_dispatch_stack_pre_dispatch", lambda: 0)
_is_wrapped = getattr(torch._C._functorch, "is_functorch_wrapped_tensor", lambda _: False)


def _is_recorded() -> bool:
    return torch.jit.is_tracing() or _modes_before_dispatch() > 0 or any(torch._C._get_dispatch_mode(key) is not None for key in _RECORDERS)


def _check_ordinary(**tensors) -> None:
    """What no call can do without, whatever it goes on to ask for."""
    if _calls.ordinary(*tensors.values()):
        return
    if _is_recorded():
        raise NotImplementedError("the operators on rows are not recorded by torch.jit.trace, make_fx or tracing with fake tensors: a trace would hold their outputs as allocations only")
    for name, t in tensors.items():
        if isinstance(t, torch.Tensor):
            if _is_wrapped(t) or torch._is_functional_tensor(t):
                raise NotImplementedError(f"{name} is a tensor of a torch.func transform, which the operators on rows do not take")
            if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{name} carries a derivative forward, which the operators on rows would lose: use backward, or unpack_dual")
            _check_memory(t, name)


def _on_gpu(t, name: str, like=None) -> None:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a torch tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a CUDA device")
    if like is not None and t.get_device() != like.get_device():
        raise ValueError(f"{name} must be on {like.device}, got {t.device}")


def _rows(t, name: str, like=None, dtype=None) -> Tuple[torch.Tensor, int, int, int, int]:
    """The rows with their values side by side, how many they are and how wide, the distance from one to the next, and their type."""
    _on_gpu(t, name, like)
    shape = t.shape
    if len(shape) != 2:
        raise ValueError(f"{name} must be 2-dimensional, got {t.dim()}")
    kind = _DTYPES.get(t.dtype)
    if kind is None:
        raise ValueError(f"{name} must have dtype float32, float16 or bfloat16, got {t.dtype}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} must have dtype {dtype}, got {t.dtype}")
    n, d = shape
    if d == 0:
        raise ValueError(f"{name} must have at least one column")
    t = t.resolve_neg()   # (the imaginary part of a conjugate is a view whose values are the negatives of what lies there)
    ld, step = t.stride()
    if step != 1 and d > 1:
        t = t.contiguous()
        ld = d
    return t, n, d, ld if n > 1 else d, kind


def _ids(ids, name: str, like=None) -> Tuple[torch.Tensor, int]:
    _on_gpu(ids, name, like)
    bits = _ID_BITS.get(ids.dtype)
    if bits is None:
        raise ValueError(f"{name} must have dtype int32, uint32 or int64, got {ids.dtype}")
    if ids.numel() > _MOST:
        raise ValueError(f"{name} must have no more than 2**31 - 1 entries")
    return ids if ids.is_contiguous() else ids.contiguous(), bits


def _floats(t, name: str, shape, like) -> torch.Tensor:
    _on_gpu(t, name, like)
    if t.dtype != torch.float32:
        raise ValueError(f"{name} must have dtype float32, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    t = t.resolve_neg()
    return t if t.is_contiguous() else t.contiguous()


def _groups(groups: RowGroups, like) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, int, int, int]:
    """order, position, offsets, number of clusters, rows, choices to a row"""
    order, position, offsets = groups
    for t, name in ((order, "order"), (position, "position"), (offsets, "offsets")):
        _on_gpu(t, name, like)
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous and have dtype int32")
    if position.dim() not in (1, 2) or offsets.dim() != 1 or offsets.shape[0] < 2:
        raise ValueError("position must have one or two dimensions, offsets one with at least two entries")
    if tuple(order.shape) != (position.numel(),):
        raise ValueError(f"order must have shape ({position.numel()},), got {tuple(order.shape)}")
    m = position.shape[1] if position.dim() == 2 else 1
    if m == 0:
        raise ValueError("a row must have at least one choice")
    return order, position, offsets, offsets.shape[0] - 1, position.shape[0], m


def _clusters(n_clusters: int) -> int:
    n_clusters = int(n_clusters)
    if not 0 < n_clusters < _MOST:
        raise ValueError("the number of clusters must be positive and below 2**31 - 1")
    return n_clusters


# The handle of a stream without the Stream around it (2 us less where a call took 13), outputs from `new_empty`, no workspace where
# none is needed.
try:
    from torch._C import _cuda_getCurrentRawStream as _raw_stream
except ImportError:   # (a torch without CUDA, or another torch)

    def _raw_stream(index: int) -> int:
        return torch.cuda.current_stream(index).cuda_stream


def _check(status: int) -> None:
    if status:
        check(status)


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _workspace(n_bytes: int, like: torch.Tensor) -> Tuple[Optional[torch.Tensor], Optional[int], int]:
    """The workspace, its address and its size."""
    if n_bytes == 0:
        return None, None, 0
    space = like.new_empty(n_bytes, dtype=torch.uint8)
    return space, space.data_ptr(), n_bytes


def _wants_grad(*tensors) -> bool:
    for t in tensors:
        if isinstance(t, torch.Tensor) and t.requires_grad:
            return torch.is_grad_enabled()
    return False


# ---- lookup ---------------------------------------------------------------------------------------------------------------------


def _lookup(table, ids, scale, row_scales):
    rows, k, d, ld, kind = _rows(table, "table")
    at, bits = _ids(ids, "ids", table)
    _clusters(k)
    if row_scales is not None:
        row_scales = _floats(row_scales, "row_scales", ids.shape, table)
    out = rows.new_empty((*at.shape, d))
    index = rows.get_device()
    _check(_op_lookup(index, rows.data_ptr(), ld, kind, k, d, at.data_ptr(), bits, at.numel(), scale, _p(row_scales), out.data_ptr(), _raw_stream(index)))
    return out


class _Lookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale, row_scales):
        ctx.scale, ctx.k = scale, table.shape[0]
        # (the table itself is needed for the scales' gradient only)
        ctx.save_for_backward(table if row_scales is not None and ctx.needs_input_grad[3] else None, ids, row_scales)
        return _lookup(table, ids, scale, row_scales)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        table, ids, row_scales = ctx.saved_tensors
        grad = grad.reshape(-1, grad.shape[-1])
        flat = ids.reshape(-1)
        grad_table = grad_scales = None
        if ctx.needs_input_grad[0]:
            grad_table = lookup_grad(grad, flat, ctx.k, ctx.scale, None if row_scales is None else row_scales.reshape(-1))
        if ctx.needs_input_grad[3]:
            grad_scales = lookup_scale_grad(grad, table, flat, ctx.scale).reshape(ids.shape)
        return grad_table, None, None, grad_scales


def lookup(table: torch.Tensor, ids: torch.Tensor, scale: float = 1.0, row_scales: Optional[torch.Tensor] = None) -> torch.Tensor:
    """scale * row_scales * table[ids]: the vectors of `ids` (any shape; int32, uint32 or int64, as the assignments of a model), out of
    a table of k x d values in fp32, fp16 or bf16.  `row_scales`, if given, has the shape of `ids` and dtype float32.  An id that is no
    row of the table (-1 as padding) gives zeros and no gradient.  Differentiable in `table` (see lookup_grad) and `row_scales`."""
    scale = float(scale)
    out = _calls.lookup(table, ids, scale, row_scales)
    if out is not None:
        return out
    _check_ordinary(table=table, ids=ids, row_scales=row_scales)
    if _wants_grad(table, row_scales):
        return _Lookup.apply(table, ids, scale, row_scales)
    return _lookup(table, ids, scale, row_scales)


def lookup_grad(grad: torch.Tensor, ids: torch.Tensor, n_rows: int, scale: float = 1.0, row_scales: Optional[torch.Tensor] = None,
                dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Gradient of a table of `n_rows` rows: row c is the sum of scale * row_scales[i] * grad[i] over ids[i] = c, zeros where there is no such
    i.  Summed in fp32, in short chains and an order that depends on the ids alone, and rounded once to `dtype` (that of `grad`, or float32).
    No gradient is recorded (nor by the other functions whose names end in _grad)."""
    if dtype is None:
        out = _calls.lookup_grad(grad, ids, n_rows, float(scale), row_scales)
        if out is not None:
            return out
    _check_ordinary(grad=grad, ids=ids, row_scales=row_scales)
    rows, n, d, ld, kind = _rows(grad, "grad")
    at, bits = _ids(ids, "ids", grad)
    if at.shape != (n,):
        raise ValueError(f"ids must have shape ({n},), got {tuple(at.shape)}")
    k = _clusters(n_rows)
    if row_scales is not None:
        row_scales = _floats(row_scales, "row_scales", ids.shape, grad)
    if dtype is None or dtype == rows.dtype:
        out, out_kind = rows.new_empty((k, d)), kind
    elif dtype == torch.float32:
        out, out_kind = rows.new_empty((k, d), dtype=dtype), 0
    else:
        raise ValueError(f"dtype must be {grad.dtype} or float32, got {dtype}")
    space, address, size = _workspace(lib.skm_op_lookup_grad_workspace(n, k, d, kind), rows)
    index = rows.get_device()
    _check(_op_lookup_grad(index, rows.data_ptr(), ld, kind, k, d, at.data_ptr(), bits, n, float(scale), _p(row_scales), out.data_ptr(), out_kind, address, size,
                               _raw_stream(index)))
    return out


def lookup_scale_grad(grad: torch.Tensor, table: torch.Tensor, ids: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """Gradient of the row scales of a lookup, float32: scale * <grad[i], table[ids[i]]>, zero where the id is no row of the table."""
    out = _calls.lookup_scale_grad(grad, table, ids, float(scale))
    if out is not None:
        return out
    _check_ordinary(grad=grad, table=table, ids=ids)
    rows, n, d, ld, kind = _rows(grad, "grad")
    t, k, d_t, ld_t, _ = _rows(table, "table", grad, grad.dtype)
    at, bits = _ids(ids, "ids", grad)
    if d_t != d:
        raise ValueError(f"grad and table must have the same dimensionality, got {d} and {d_t}")
    if at.shape != (n,):
        raise ValueError(f"ids must have shape ({n},), got {tuple(at.shape)}")
    _clusters(k)
    out = rows.new_empty(n, dtype=torch.float32)
    index = rows.get_device()
    _check(_op_lookup_scale_grad(index, rows.data_ptr(), ld, t.data_ptr(), ld_t, kind, k, d, at.data_ptr(), bits, n, float(scale), out.data_ptr(),
                                       _raw_stream(index)))
    return out


# ---- rows to their clusters and back --------------------------------------------------------------------------------------------


def group_rows(ids: torch.Tensor, n_clusters: int) -> RowGroups:
    """The order of rows by cluster: `ids` has one entry for each row (n), or one for each of its m choices (n x m).  Pairs of the same
    cluster keep their order; those without one (an id outside 0 .. n_clusters - 1) come last.  The offsets stay on the device."""
    out = _calls.group_rows(ids, n_clusters)
    if out is not None:
        return RowGroups(*out)
    _check_ordinary(ids=ids)
    at, bits = _ids(ids, "ids")
    if at.dim() not in (1, 2) or (at.dim() == 2 and at.shape[1] == 0):
        raise ValueError(f"ids must have shape (n,) or (n, m) with m > 0, got {tuple(at.shape)}")
    k, n = _clusters(n_clusters), at.numel()
    whole = at.new_empty(2 * n + k + 1, dtype=torch.int32)
    order, position, offsets = whole.split((n, n, k + 1))
    space, address, size = _workspace(lib.skm_op_group_rows_workspace(n, k), at)
    index = at.get_device()
    first = whole.data_ptr()
    _check(_op_group_rows(index, at.data_ptr(), bits, n, k, first, first + 4 * n, first + 8 * n, address, size, _raw_stream(index)))
    return RowGroups(order, position if at.dim() == 1 else position.view(at.shape), offsets)


def _to_clusters(x, groups):
    rows, n_x, d, ld, kind = _rows(x, "x")
    order, position, offsets, k, n, m = _groups(groups, x)
    if n_x != n:
        raise ValueError(f"x must have {n} rows, got {n_x}")
    out = rows.new_empty((n * m, d))
    index = rows.get_device()
    _check(_op_to_clusters(index, rows.data_ptr(), ld, kind, d, order.data_ptr(), position.data_ptr(), offsets.data_ptr(), k, n, m, out.data_ptr(), _raw_stream(index)))
    return out


def _from_clusters(y, groups, weights, name="y"):
    rows, n_y, d, ld, kind = _rows(y, name)
    order, position, offsets, k, n, m = _groups(groups, y)
    if n_y != n * m:
        raise ValueError(f"{name} must have {n * m} rows, got {n_y}")
    if weights is not None:
        weights = _floats(weights, "weights", position.shape, y)
    out = rows.new_empty((n, d))
    index = rows.get_device()
    _check(_op_from_clusters(index, rows.data_ptr(), ld, kind, d, order.data_ptr(), position.data_ptr(), offsets.data_ptr(), k, n, m, _p(weights), out.data_ptr(), _raw_stream(index)))
    return out


def _from_clusters_grad(grad, y, groups, weights, want_y, want_weights):
    rows, n_grad, d, ld, kind = _rows(grad, "grad")
    order, position, offsets, k, n, m = _groups(groups, grad)
    if n_grad != n:
        raise ValueError(f"grad must have {n} rows, got {n_grad}")
    if weights is not None:
        weights = _floats(weights, "weights", position.shape, grad)
    from_y, ld_y = None, 0
    if want_weights:
        from_y, n_y, d_y, ld_y, _ = _rows(y, "y", grad, grad.dtype)
        if (n_y, d_y) != (n * m, d):
            raise ValueError(f"y must have shape {(n * m, d)}, got {(n_y, d_y)}")
    grad_y = rows.new_empty((n * m, d)) if want_y else None
    grad_weights = rows.new_empty(position.shape, dtype=torch.float32) if want_weights else None
    index = rows.get_device()
    _check(_op_from_clusters_grad(index, rows.data_ptr(), ld, _p(from_y), ld_y, kind, d, order.data_ptr(), position.data_ptr(), offsets.data_ptr(), k, n, m, _p(weights), _p(grad_y),
                                        _p(grad_weights), _raw_stream(index)))
    return grad_y, grad_weights


class _ToClusters(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, order, position, offsets):
        ctx.save_for_backward(order, position, offsets)
        return _to_clusters(x, RowGroups(order, position, offsets))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return to_clusters_grad(grad, RowGroups(*ctx.saved_tensors)), None, None, None


class _FromClusters(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, order, position, offsets):
        # (y is needed for the weights' gradient only)
        ctx.save_for_backward(y if weights is not None and ctx.needs_input_grad[1] else None, weights, order, position, offsets)
        return _from_clusters(y, RowGroups(order, position, offsets), weights)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        y, weights, *groups = ctx.saved_tensors
        _check_ordinary(grad=grad, y=y, weights=weights, **_named(groups))
        grad_y, grad_weights = _from_clusters_grad(grad, y, RowGroups(*groups), weights, ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        return grad_y, grad_weights, None, None, None


def to_clusters(x: torch.Tensor, groups: RowGroups) -> torch.Tensor:
    """Rows in the order of their clusters: n x d to (n * m) x d, row i once for each of its m choices, at groups.position[i, j].  The rows of
    cluster c are offsets[c] .. offsets[c + 1] - 1; behind the last cluster the slots of choices without one hold zeros.
    Differentiable in x (see to_clusters_grad)."""
    out = _calls.to_clusters(x, *groups)
    if out is not None:
        return out
    _check_ordinary(x=x, **_named(groups))
    if _wants_grad(x):
        return _ToClusters.apply(x, *groups)
    return _to_clusters(x, groups)


def to_clusters_grad(grad: torch.Tensor, groups: RowGroups) -> torch.Tensor:
    """Gradient of the rows of to_clusters: the sum over a row's choices of their slots' gradients (n x d), without those that have no
    cluster."""
    out = _calls.from_clusters(grad, *groups, None)
    if out is not None:
        return out
    _check_ordinary(grad=grad, **_named(groups))
    return _from_clusters(grad, groups, None, "grad")


def from_clusters(y: torch.Tensor, groups: RowGroups, weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows back from the order of their clusters: out[i] = sum over j of weights[i, j] * y[position[i, j]], n x d.  Choices without a cluster
    contribute nothing, whatever their slots hold.  `weights` (float32, the shape of groups.position) is 1 if not given.
    Differentiable in y and weights (see from_clusters_grad)."""
    out = _calls.from_clusters(y, *groups, weights)
    if out is not None:
        return out
    _check_ordinary(y=y, weights=weights, **_named(groups))
    if _wants_grad(y, weights):
        return _FromClusters.apply(y, weights, *groups)
    return _from_clusters(y, groups, weights)


def from_clusters_grad(grad: torch.Tensor, y: torch.Tensor, groups: RowGroups, weights: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Gradients of from_clusters: of y, weights[i, j] * grad[i] at position[i, j] and zeros in the slots of choices without a cluster; and of the
    weights (float32; None where there are none), <grad[i], y[position[i, j]]>."""
    out = _calls.from_clusters_grad(grad, y, *groups, weights)
    if out is not None:
        return out
    _check_ordinary(grad=grad, y=y, weights=weights, **_named(groups))
    return _from_clusters_grad(grad, y, groups, weights, True, weights is not None)


# ---- products in 8 bits ---------------------------------------------------------------------------------------------------------


def quantize_rows(x: torch.Tensor) -> QuantizedRows:
    """Rows in 8 bits: scales[i] = max |x[i]| / 127 (float32), values[i] = x[i] * (127 / max |x[i]|), both in float32, rounded to the nearest whole number,
    int8.  A row of zeros has scale 0; a row with a value that is no finite number has scale NaN and zeros.  The rows of the result begin on 16
    bytes.  No gradient is recorded."""
    out = _calls.quantize_rows(x)
    if out is not None:
        return QuantizedRows(*out)
    _check_ordinary(x=x)
    rows, n, d, ld, kind = _rows(x, "x")
    if n > _MOST:
        raise ValueError("x must have no more than 2**31 - 1 rows")
    pitch = (d + 15) // 16 * 16
    q = rows.new_empty((n, pitch), dtype=torch.int8)
    scales = rows.new_empty(n, dtype=torch.float32)
    index = rows.get_device()
    _check(_op_quantize_rows(index, rows.data_ptr(), ld, kind, n, d, q.data_ptr(), pitch, scales.data_ptr(), _raw_stream(index)))
    return QuantizedRows(q[:, :d] if pitch != d else q, scales)


def _bytes(t, name: str, like=None) -> torch.Tensor:
    _on_gpu(t, name, like)
    if t.dtype != torch.int8:
        raise ValueError(f"{name} must have dtype int8, got {t.dtype}")
    return t.contiguous() if t.shape[-1] > 1 and t.stride(-1) != 1 else t


def product_8bit(x: torch.Tensor, x_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, offsets: Optional[torch.Tensor] = None,
                 dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """x w^T of rows in 8 bits: out[i, c] = x_scales[i] * w_scales[c] * sum_j x[i, j] * w[c, j], the sum exact.  x is n x d, w m x d (both int8), the
    scales float32, the result n x m of `dtype`.

    With `offsets` (int32, from group_rows) w is n_clusters x m x d and w_scales n_clusters x m: row i is multiplied by the matrix of the cluster c with
    offsets[c] <= i < offsets[c + 1]; rows of no cluster come out as zeros.

    Rows that do not begin on 16 bytes are copied first; quantize_rows makes rows that do.  d is at most 131071.  No gradient is recorded."""
    kind = _DTYPES.get(dtype)
    if kind is None:
        raise ValueError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
    out = _calls.product_8bit(x, x_scales, w, w_scales, offsets, kind)
    if out is not None:
        return out
    _check_ordinary(x=x, x_scales=x_scales, w=w, w_scales=w_scales, offsets=offsets)
    _on_gpu(x, "x")
    _on_gpu(w, "w", x)
    if x.dim() != 2:
        raise ValueError(f"x must be 2-dimensional, got {x.dim()}")
    if w.dim() != (2 if offsets is None else 3):
        raise ValueError(f"w must be {2 if offsets is None else 3}-dimensional, got {w.dim()}")
    x, w = _bytes(x, "x"), _bytes(w, "w", x)
    n, d = x.shape
    m, e = w.shape[-2], 0
    if w.shape[-1] != d:
        raise ValueError(f"x and w must have the same dimensionality, got {d} and {w.shape[-1]}")
    if not 0 < d <= 131071:
        raise ValueError(f"the dimensionality of a product in 8 bits must be positive and at most 131071, got {d}")
    if offsets is not None:
        e = _clusters(w.shape[0])
        _on_gpu(offsets, "offsets", x)
        if offsets.dtype != torch.int32 or tuple(offsets.shape) != (e + 1,) or not offsets.is_contiguous():
            raise ValueError(f"offsets must be {e + 1} contiguous int32")
        if e > 1 and m > 0 and w.stride(0) != m * (w.stride(1) if m > 1 else w.stride(0)):
            w = w.contiguous()
    x_scales = _floats(x_scales, "x_scales", (n,), x)
    w_scales = _floats(w_scales, "w_scales", w.shape[:-1], x)
    ld_x = x.stride(0) if n > 1 else d
    ld_w = w.stride(-2) if m > 1 else w.stride(0) if e > 1 else d
    out = x_scales.new_empty((n, m), dtype=dtype)
    x_at, w_at = x.data_ptr(), w.data_ptr()
    space, address, size = _workspace(lib.skm_op_product_8bit_workspace(x_at, ld_x, w_at, ld_w, n, m, d, e), x)
    index = x.get_device()
    _check(_op_product_8bit(index, x_at, ld_x, x_scales.data_ptr(), w_at, ld_w, w_scales.data_ptr(), n, m, d, e, _p(offsets), out.data_ptr(), kind, address, size,
                                  _raw_stream(index)))
    return out


def check_products(device=None) -> None:
    """Waits for the current stream of `device` and raises RuntimeError if a product on it gave up waiting inside its kernel (the next
    product_8bit on the device raises it too)."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    check(lib.skm_op_product_8bit_status(-1 if device.index is None else device.index, torch.cuda.current_stream(device).cuda_stream))


__all__ = [
    "RowGroups", "QuantizedRows", "lookup", "lookup_grad", "lookup_scale_grad", "group_rows", "to_clusters", "to_clusters_grad", "from_clusters", "from_clusters_grad",
    "quantize_rows", "product_8bit", "check_products",
]
