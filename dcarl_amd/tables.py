"""Rows of a table by dense state id, with the gradient of the table by sorted ids.

A table has one row of D values per state (``state_ids`` / ``index_states`` hand out the ids, the samplers -1 for a visit they drop);
``lookup`` reads the rows of a batch of ids, its gradient adds a batch's rows up per id, always in the same order."""
from __future__ import annotations

import torch

from . import _lib, _sequence as _seq


def _check_ids(ids, n_rows: int, validate: bool):
    ids = _seq.whole_numbers("ids", ids)
    if validate and ids.numel():
        if ids.device.type == "cuda" and _seq.capturing():
            raise ValueError("ids cannot be checked while a graph is captured: pass validate=False")
        lo, hi = (int(v) for v in torch.aminmax(ids))
        if lo < -1 or hi >= n_rows:
            raise IndexError(f"ids out of range: [{lo},{hi}] vs {n_rows} rows (-1 = no row)")
    return ids.contiguous()


def _gather(table, ids, scale):
    dev = table.device
    t, ld = _seq.rows_of(table)
    S, D = t.shape
    out = torch.empty(*ids.shape, D, dtype=t.dtype, device=dev)
    _lib.check(_lib.load().dcarl_rows_gather(_seq.at(t), _seq.TYPES[t.dtype], ld, S, _seq.at(ids), ids.element_size(), ids.numel(), D, scale,
                                             _seq.at(out), _seq.stream(dev)), "dcarl_rows_gather")
    return out


def _gradient(dout, ids, n_rows, scale):
    lib, dev = _lib.load(), dout.device
    N, D = ids.numel(), dout.shape[-1]
    d, ldd = _seq.rows_of(dout if dout.dim() == 2 else dout.reshape(N, D))
    code = _seq.TYPES[d.dtype]
    grad = torch.empty(n_rows, D, dtype=d.dtype, device=dev)
    ws = torch.empty(max(lib.dcarl_rows_workspace_bytes(N, n_rows, D, code), 16), dtype=torch.uint8, device=dev)
    _lib.check(lib.dcarl_rows_gradient(_seq.at(d), code, ldd, _seq.at(ids), ids.element_size(), N, D, n_rows, scale, _seq.at(ws), _seq.at(grad),
                                       _seq.stream(dev)), "dcarl_rows_gradient")
    return grad


class _Lookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale):
        ctx.save_for_backward(ids)
        ctx.rest = table.shape[0], scale
        ctx.captured = _seq.capturing()
        return _seq.run_on(table.device, _gather, table, ids, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        if not ctx.captured and _seq.capturing():
            raise ValueError("the forward pass ran outside of the graph that its backward pass is captured into")
        _seq.recordable(True, dout)
        return _seq.run_on(dout.device, _gradient, dout, ctx.saved_tensors[0], *ctx.rest), None, None


def lookup(table, ids, scale: float = 1.0, *, validate: bool = True):
    """``scale * table[ids]``, zeros where an id is -1; ids of any shape, the result has a dimension D behind it.

    table: (S, D) float64, float32, bfloat16 or float16 on the GPU, rows at any distance; ids: int32 or int64.
    The gradient of the table is dense, of the table's type: per id the sum over the batch in ascending order, held in f32 (f64), scaled and
    rounded once; rows no id names are zero.  A table that carries a tangent is refused (no forward mode).  validate: raise IndexError for ids outside [-1, S), which waits for them; with
    ``validate=False`` nothing waits (a captured call needs it) and such ids count as -1.
    A backward pass is captured into a graph as that of ``episodes.gated_recurrence`` is: with its forward pass, through ``torch.autograd.grad`` on
    leaves of the graph's own, or by ``lookup_gradient``.  A call that torch.jit.trace or make_fx would record without its launch is refused."""
    _seq.type_code("table", table)
    if table.dim() != 2:
        raise ValueError(f"table must be (S, D), not {tuple(table.shape)}")
    gradient = _seq.wants_gradient(table)
    _seq.recordable(not gradient, table)
    scale = _seq.number("scale", scale)
    ids = _check_ids(ids, table.shape[0], validate)
    dev = _seq.on_device(("table", table), ("ids", ids if ids.is_cuda else None))
    if ids.device != dev:
        ids = _seq.from_host("ids", ids, dev)
    if gradient:
        return _Lookup.apply(table, ids, scale)
    return _seq.run_on(dev, _gather, table, ids, scale)


def lookup_gradient(dout, ids, n_rows: int, scale: float = 1.0, *, validate: bool = True):
    """The gradient of ``lookup``'s table by itself: (n_rows, D) with row s = scale * the sum of ``dout`` (ids' shape, D) over ids == s.
    Sums of f32 are held in f32: ``lookup_gradient(dout.double(), ...)`` holds them in f64.  It has no gradient of its own: a dout that requires one is refused."""
    _seq.type_code("dout", dout)
    _seq.recordable(True, dout)
    if _seq.wants_gradient(dout):
        raise ValueError("lookup_gradient has no gradient of its own: detach dout")
    scale = _seq.number("scale", scale)
    n_rows = int(n_rows)
    if n_rows < 0:
        raise ValueError(f"n_rows = {n_rows} is negative")
    ids = _check_ids(ids, n_rows, validate)
    if dout.dim() < 1 or tuple(dout.shape[:-1]) != tuple(ids.shape):
        raise ValueError(f"dout {tuple(dout.shape)} has no row for each of the ids {tuple(ids.shape)}")
    dev = _seq.on_device(("dout", dout), ("ids", ids if ids.is_cuda else None))
    if ids.device != dev:
        ids = _seq.from_host("ids", ids, dev)
    return _seq.run_on(dev, _gradient, dout, ids, n_rows, scale)
