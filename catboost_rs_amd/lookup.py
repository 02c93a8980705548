"""Sums of looked-up rows of a table that lives on the GPU, and the table's gradient: whole-number inputs
(bins of :func:`quantize`, buckets of :func:`perfect_hash`, leaves of trees) for a model that is trained by
gradients.

They take torch tensors on the GPU, enqueue on torch's current stream and record no autograd graph, as the
operators on class scores do.
"""
from __future__ import annotations

from .class_scores import _TYPE, _addr, _bind, _on, _state, _stream, _vector, _workspace


def _matrix(torch, x, what):
    """Type, sizes and strides of a matrix."""
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise ValueError(f"{what} must be a torch tensor of two dimensions")
    t = _TYPE.get(x.dtype)
    if t is None:
        raise ValueError(f"{what} must be float32, float16 or bfloat16, not {x.dtype}")
    if not x.is_cuda:
        raise ValueError(f"{what} must be on the GPU")
    return (t, *x.shape, *x.stride())


def _index(torch, index, rows, like):
    """Contiguous i32 [rows] or [rows][list], and the list's length."""
    if not isinstance(index, torch.Tensor) or index.dim() not in (1, 2) or (rows is not None and index.shape[0] != rows):
        raise ValueError("index must be a torch tensor [rows] or [rows][list]")
    return _vector(torch, index, index.shape, torch.int32, like, "index"), index.shape[1] if index.dim() == 2 else 1


def _fits(entries, dim, index, many):
    """Refuses what 32 bits would cut off on the way to the library, and before anything of that size is allocated."""
    if not 1 <= entries < 1 << 31:
        raise _state["error"](-2, "entries must be in 1 .. 2^31 - 1")
    if not 1 <= dim <= 1 << 24:
        raise _state["error"](-2, "dim must be in 1 .. 2^24")
    if index.shape[0] * many >= 1 << 31:
        raise _state["error"](-2, "rows times list must be below 2^31")


def lookup_rows(table, index, scale=1.0):
    """``scale`` times the sum of the table's rows that ``index`` names (``cbh_lookup_rows``): [rows][dim] of the
    table's type.  ``table`` [entries][dim] f32, f16 or bf16 of any strides; ``index`` i32 [rows] or [rows][list], an
    index outside the entries adds nothing.  The sum is f32, in the list's order."""
    torch = _state.get("torch") or _bind()
    t, entries, dim, rs, cs = _matrix(torch, table, "table")
    index, many = _index(torch, index, None, table)
    _fits(entries, dim, index, many)
    rows = index.shape[0]
    with _on(table):
        out = torch.empty((rows, dim), dtype=table.dtype, device=table.device)
        _state["check"](_state["lookup"](table.data_ptr(), t, entries, dim, rs, cs, index.data_ptr(), rows, many,
                                         float(scale), out.data_ptr(), _stream(table)))
    return out


def lookup_gradients(grad, index, entries, scale=1.0, dtype=None):
    """The gradient [entries][dim] by the table of :func:`lookup_rows`, from that by its result ``grad``
    [rows][dim] (any strides, also expanded ones) (``cbh_lookup_gradients``): sums in f32, the same in every run, rounded once to
    ``dtype`` (None: that of ``grad``).  Entries that do not occur have 0."""
    torch = _state.get("torch") or _bind()
    t, rows, dim, rs, cs = _matrix(torch, grad, "grad")
    index, many = _index(torch, index, rows, grad)
    dtype = grad.dtype if dtype is None else dtype
    if dtype not in _TYPE:
        raise ValueError(f"dtype must be float32, float16 or bfloat16, not {dtype}")
    entries = int(entries)
    _fits(entries, dim, index, many)
    with _on(grad):
        out = torch.empty((entries, dim), dtype=dtype, device=grad.device)
        size = _state["table_grad_ws"](rows, many, entries, dim)
        ws = _workspace(torch, size, grad)
        _state["check"](_state["table_grad"](grad.data_ptr(), t, rows, dim, rs, cs, index.data_ptr(), many, entries,
                                             float(scale), out.data_ptr(), _TYPE[dtype], _addr(ws), size, _stream(grad)))
    return out
