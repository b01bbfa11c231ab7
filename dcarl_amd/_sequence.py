"""What the sequence operators share (``episodes.gated_recurrence``, ``tables.lookup``, ``candidates.adjust``): storage types, the
checks of ids and offsets, the device a call runs on."""
from __future__ import annotations

import torch
import torch.autograd.forward_ad as _forward
import torch.fx._symbolic_trace as _fx

from . import _lib

TYPES = {torch.float64: 0, torch.float32: 1, torch.bfloat16: 2, torch.float16: 3}          # DCARL_F64 ... of include/dcarl.h


def type_code(name: str, t: torch.Tensor, allowed=TYPES) -> int:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor, not {type(t).__name__}")
    if t.dtype not in allowed:
        raise TypeError(f"{name} is {t.dtype}: " + ", ".join(str(k).replace("torch.", "") for k in allowed) + " are supported")
    return TYPES[t.dtype]


def on_device(*named) -> torch.device:
    """The one GPU that all of the (name, tensor or None) live on; raises where one lives elsewhere (there is no CPU path)."""
    first = None
    for name, t in named:
        if t is None:
            continue
        if not t.is_cuda:
            raise _lib.DcarlError(f"{name} is on {t.device}: the operator has no CPU path")
        if first is None:
            first, index = (name, t), t.get_device()
        elif t.get_device() != index:
            raise ValueError(f"{name} is on {t.device}, {first[0]} on {first[1].device}")
    return first[1].device


def run_on(device: torch.device, call, *args):
    """call(*args) with everything in it — allocations, the current stream, the launches — on `device`, whatever the current device is."""
    if torch.cuda.current_device() == device.index:
        return call(*args)
    with torch.cuda.device(device):
        return call(*args)


def stream(device: torch.device) -> int:
    """The handle of the device's current stream (the wrapper object that torch.cuda.current_stream builds costs 3 us a call)."""
    return _raw_stream(device.index)


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def at(t):
    """The address of a tensor, None where there is none.  A wrapper that has elements and no address (functionalize's, a tangent's lazy zeros) is no
    absent operand."""
    if t is None:
        return None
    p = t.data_ptr()
    if not p and t.numel():
        raise ValueError(f"an operand {tuple(t.shape)} has no memory behind it that a kernel could read")
    return p


def like(t: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of t's shape, type and device (empty_like by itself keeps the order of a transposed one's strides)."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def wants_gradient(*tensors) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def number(name: str, v) -> float:
    """A strength, scale or discount; one that wants a gradient is refused, since none comes back to it."""
    if isinstance(v, torch.Tensor):
        if wants_gradient(v):
            raise ValueError(f"{name} has no gradient: detach it")
        recordable(False, v)
    return float(v)


_proxies, _tracing = torch._C._TorchDispatchModeKey.PROXY, torch._C._get_tracing_state


def recordable(launched: bool, *tensors) -> None:
    """Refuses calls of which a record or a derivative would lack the launch, which goes through addresses and leaves no node behind.
    A tangent: the operators have no forward-mode gradient.  A trace: it would hold the allocation of the result alone and replay whatever lies there;
    an autograd function (launched False) is a node of torch.jit's own and runs again on replay, to make_fx it is none."""
    if _forward._current_level >= 0:                         # inside of a dual_level, the only place where there are tangents
        if any(isinstance(t, torch.Tensor) and _forward.unpack_dual(t).tangent is not None for t in tensors):
            raise ValueError("the operator has no forward-mode gradient: an operand carries a tangent")
    if _fx._is_fx_tracing_flag and torch._C._get_dispatch_mode(_proxies) is not None or launched and _tracing() is not None:
        raise ValueError("the operator cannot be traced: the trace would not hold its launch (capture a graph instead)")


def plain(t):
    """A tensor whose memory holds its values: a lazily negated view (the imaginary part of a conjugate) is written out."""
    return t.resolve_neg() if t is not None and t.is_neg() else t


def rows_of(t: torch.Tensor, far: int = 1 << 62):
    """(tensor, elements between its rows) of a 2-D operand whose channels are contiguous; a copy where they are not.  Rows may lie
    anywhere at a non-negative distance (slices, one row expanded to many) of up to `far` elements, or of their own width."""
    t = plain(t)
    step, one = t.stride()
    if one != 1 and t.shape[1] > 1 or step < 0 or step > far and step > t.shape[1]:
        t = t.contiguous()
        step = t.stride(0)
    return t, step


def from_host(name: str, t, device):
    """Ids or offsets that lie on the host, moved to the call's device."""
    if capturing():
        raise ValueError(f"{name} must lie on the GPU while a graph is captured")
    return t.to(device)


def capturing() -> bool:
    return torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()


def whole_numbers(name: str, t) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        t = torch.as_tensor(t)
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be int32 or int64, not {t.dtype}")
    return t


def offsets(name: str, off, n: int, segments, validate: bool) -> torch.Tensor:
    """The offsets of ragged segments over `n` entries as a contiguous int64 tensor, checked: they rise from 0 to at most `n`.  Offsets on the
    GPU are checked through a copy to the host that waits for them; ``validate=False`` leaves that out, and is what a captured call needs."""
    off = whole_numbers(name, off)
    if off.dim() != 1 or off.numel() < 1:
        raise ValueError(f"{name} must be one-dimensional with an entry more than there are segments")
    if segments is not None and off.numel() != segments + 1:
        raise ValueError(f"{name} has {off.numel()} entries for {segments} segments: {segments + 1} are needed")
    if validate:
        if off.device.type == "cuda" and capturing():
            raise ValueError(f"{name} cannot be checked while a graph is captured: pass validate=False")
        host = off.cpu().to(torch.int64)
        if int(host[0]) != 0 or int(host[-1]) > n or bool((host[1:] < host[:-1]).any()):
            raise ValueError(f"{name} must rise from 0 to at most {n}")
    return off if off.dtype == torch.int64 and off.is_contiguous() else off.to(torch.int64).contiguous()
