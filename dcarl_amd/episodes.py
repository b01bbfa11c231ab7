"""Episode-return reduction on MI355X: the step that produces the cumulative-reward column.

* ``episode_returns`` — the CARLA collector's arithmetic: step reward ``0.1*sqrt(v)``, -100 on a collision, 0 when stuck
  (Test_Scenarios/TestScenario_Town03.py:402-421) summed per episode (Agent/drl_library/dqn/dqn_value_collect.py:119),
  plus the AveSpeed the collector logs.
* ``nstep_backup`` — the field vehicle's ``RLS.add_data`` value stream (stable_baselines/deepq/RLS.py:185-215): a 10-deep
  trajectory buffer; a transition leaves it with its own reward, the last ten of a finished episode get the terminal
  reward times ``gamma**k``.
* ``gated_recurrence`` — a state carried along every episode, h[t] = gate[t] * h[t-1] + x[t], with its gradients; and
  ``discounted_returns``, the returns of a discount, which are that recurrence reversed (neither has a counterpart in the reference)."""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from . import _lib, _sequence as _seq

COLLISION, PASSED, STUCK = 1, 2, 4          # flag bits of a step (TS:406, 413, 418)


def _dev64(x, dev, dtype=torch.float64):
    return torch.as_tensor(x).to(device=dev, dtype=dtype).contiguous()


def episode_returns(vx, vy, flags, ep_off, want_steps: bool = True):
    """Returns (episode_reward f64 [E], ave_speed f64 [E], step_reward f64 [N] or None)."""
    dev = _lib.require_gpu()
    lib = _lib.load()
    vx, vy = _dev64(vx, dev), _dev64(vy, dev)
    flags = _dev64(flags, dev, torch.uint8)
    ep_off = _dev64(ep_off, dev, torch.int64)
    E, N = ep_off.numel() - 1, vx.numel()
    if vy.numel() != N or flags.numel() != N:
        raise ValueError("vx, vy and flags must have one entry per step")
    if E < 0 or (E > 0 and (int(ep_off[0]) != 0 or int(ep_off[-1]) != N or bool((ep_off[1:] < ep_off[:-1]).any()))):
        raise ValueError("ep_off must rise from 0 to the number of steps")
    ep = torch.empty(max(E, 0), dtype=torch.float64, device=dev)
    sp = torch.empty(max(E, 0), dtype=torch.float64, device=dev)
    st = torch.empty(N, dtype=torch.float64, device=dev) if want_steps else None
    _lib.check(lib.dcarl_episode_returns_f64(_lib.ptr(vx), _lib.ptr(vy), _lib.ptr(flags), _lib.ptr(ep_off), max(E, 0),
                                             _lib.ptr(st), _lib.ptr(ep), _lib.ptr(sp), _lib.stream_ptr()),
               "dcarl_episode_returns_f64")
    return ep, sp, st


def gamma_powers(gamma: float, horizon: int) -> np.ndarray:
    out = (C.c_double * max(horizon, 1))()
    _lib.load().dcarl_gamma_powers(float(gamma), int(horizon), out)
    return np.array(out[:horizon], dtype=np.float64)


def nstep_backup(rew, ep_off, ep_done, gamma: float = 0.95, horizon: int = 10):
    """RLS.add_data (RLS:185-215) for whole streams: returns (value f64 [N], recorded bool [N])."""
    dev = _lib.require_gpu()
    lib = _lib.load()
    rew = _dev64(rew, dev)
    ep_off = _dev64(ep_off, dev, torch.int64)
    ep_done = _dev64(ep_done, dev, torch.uint8)
    E, N = ep_off.numel() - 1, rew.numel()
    if ep_done.numel() != E:
        raise ValueError("ep_done must have one entry per episode")
    if E > 0 and (int(ep_off[0]) != 0 or int(ep_off[-1]) != N or bool((ep_off[1:] < ep_off[:-1]).any())):
        raise ValueError("ep_off must rise from 0 to the number of transitions")
    gp = torch.from_numpy(gamma_powers(gamma, horizon)).to(dev)
    value = torch.empty(N, dtype=torch.float64, device=dev)
    rec = torch.empty(N, dtype=torch.uint8, device=dev)
    _lib.check(lib.dcarl_nstep_backup_f64(_lib.ptr(rew), _lib.ptr(ep_off), _lib.ptr(ep_done), max(E, 0), _lib.ptr(gp),
                                          int(horizon), _lib.ptr(value), _lib.ptr(rec), _lib.stream_ptr()),
               "dcarl_nstep_backup_f64")
    return value, rec.bool()


# ---- the recurrence along episodes --------------------------------------------------------------------------------------------
_FAR = 1 << 17          # a tile's rows are addressed by 32-bit offsets: operands with rows further apart are copied


def _recurrence_args(x, gate, ep_off, h0, gate_value, reverse):
    kind = 0 if gate is None else 2 if gate.dim() == 2 else 1
    x, ldx = _seq.rows_of(x, _FAR)
    ldg = 0
    if kind == 2:
        gate, ldg = _seq.rows_of(gate, _FAR)
    elif kind == 1:
        gate = _seq.plain(gate)
        gate, ldg = (gate, gate.stride(0)) if 0 <= gate.stride(0) <= _FAR else (gate.contiguous(), 1)
    ldh0 = 0
    if h0 is not None:
        h0, ldh0 = _seq.rows_of(h0)
    N, D = x.shape
    a = _lib.CRecurrence(N, D, ep_off.numel() - 1, _seq.at(ep_off), _seq.at(x), ldx, _seq.at(gate), ldg,
                         _seq.at(h0), ldh0, gate_value, kind, int(reverse), _seq.TYPES[x.dtype], 0)
    return a, (x, gate, h0)                                   # the tensors: alive until the launch


def _bytes(n, dev):
    return torch.empty(n, dtype=torch.uint8, device=dev) if n else None


def _recurrence_forward(x, gate, ep_off, h0, gate_value, reverse, want_last, want_states):
    lib, dev = _lib.load(), x.device
    a, keep = _recurrence_args(x, gate, ep_off, h0, gate_value, reverse)
    h = _seq.like(x)
    last = torch.empty(a.E, a.D, dtype=x.dtype, device=dev) if want_last else None
    sizes = (a.N, a.D, a.E, a.type, a.gate_kind)
    states = _bytes(lib.dcarl_recurrence_states_bytes(*sizes), dev) if want_states else None
    ws = _bytes(lib.dcarl_recurrence_workspace_bytes(*sizes), dev)
    _lib.check(lib.dcarl_recurrence_forward(C.byref(a), _seq.at(states), _seq.at(ws), _seq.at(h), _seq.at(last), _seq.stream(dev)),
               "dcarl_recurrence_forward")
    return h, last, states


def _recurrence_backward(x, gate, ep_off, h0, gate_value, reverse, states, dh, dlast, want):
    lib, dev = _lib.load(), x.device
    a, keep = _recurrence_args(x, gate, ep_off, h0, gate_value, reverse)
    dh, lddh = _seq.rows_of(dh, _FAR)
    dlast = None if dlast is None else _seq.plain(dlast).contiguous()
    dx = _seq.like(x) if want[0] else None
    dgate = _seq.like(gate) if want[1] else None
    dh0 = _seq.like(h0) if want[2] else None
    ws = _bytes(lib.dcarl_recurrence_workspace_bytes(a.N, a.D, a.E, a.type, a.gate_kind), dev)
    _lib.check(lib.dcarl_recurrence_backward(C.byref(a), _seq.at(states), _seq.at(ws), _seq.at(dh), lddh, _seq.at(dlast), _seq.at(dx),
                                             _seq.at(dgate), _seq.at(dh0), _seq.stream(dev)), "dcarl_recurrence_backward")
    if a.D == 0 and dgate is not None:
        dgate.zero_()                                        # a sum over no channels
    return dx, dgate, dh0


class _Recurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, h0, ep_off, gate_value, reverse, want_last):
        h, last, states = _seq.run_on(x.device, _recurrence_forward, x, gate, ep_off, h0, gate_value, reverse, want_last, True)
        ctx.save_for_backward(x, gate, h0, ep_off, states)
        ctx.rest = gate_value, reverse
        ctx.captured = _seq.capturing()
        return (h, last) if want_last else h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dlast=None):
        if not ctx.captured and _seq.capturing():
            raise ValueError("the forward pass ran outside of the graph that its backward pass is captured into")
        _seq.recordable(True, dh, dlast)
        x, gate, h0, ep_off, states = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dgate, dh0 = _seq.run_on(x.device, _recurrence_backward, x, gate, ep_off, h0, *ctx.rest, states, dh, dlast, need[:3])
        return dx, dgate, dh0, None, None, None, None


def gated_recurrence(x, gate, ep_off, h0=None, *, reverse: bool = False, want_last: bool = False, validate: bool = True):
    """``h[t] = gate[t] * h[t-1] + x[t]`` per channel along each episode, with gradients for ``x``, ``gate`` and ``h0``.

    x: (N, D) steps, or (N,) for one channel; float64, float32, bfloat16 or float16 (sums in f32; f64 for float64; each result rounded once).
    gate: (N, D) like x, (N,) shared by the channels of a step, or a number.  ep_off: (E+1,) int offsets of the episodes as in
    ``episode_returns``; steps behind ``ep_off[E]`` belong to none: what they hold counts nowhere, the results are zero there.
    h0: (E, D) (or (E,)) states before the first steps; one step of E live episodes is N == E with every length 1.
    reverse: mirrored, ``h[t] = gate[t] * h[t+1] + x[t]`` from the end of each episode.
    Products of consecutive gates are formed by themselves, in the type of the sums: gates of magnitude up to 1 are right over any length; where a product of
    larger ones leaves that type's range, states that are not zero read inf or NaN, also where later gates would bring them back, and an
    infinite state may read NaN further on.
    want_last: also the (E, D) states that the episodes end with (``h0`` or zero for an empty one).
    validate: check ep_off's values; where it lies on the GPU this waits for it.  ``validate=False`` never waits and is what a captured call
    needs; offsets that do not rise from 0 to at most N then give unspecified results (and no access out of range).

    Everything runs on the tensors' device and its current stream; nothing is kept between calls.  The gradient has no gradient of its own, and there is
    none in forward mode: operands that carry a tangent are refused.
    A backward pass can be captured into a graph together with its forward pass, through ``torch.autograd.grad``; by itself, of a forward pass
    that ran outside, it is refused.  (``Tensor.backward`` inside a capture while an eager graph of the same leaves is alive makes autograd wait
    for the eager stream, which ends the process: capture with leaves of their own, as ``torch.autograd.grad`` on detached tensors has.)
    A call that torch.jit.trace or make_fx would record without its launch is refused."""
    code = _seq.type_code("x", x)
    flat = x.dim() == 1
    if x.dim() not in (1, 2):
        raise ValueError(f"x must be (N, D) or (N,), not {tuple(x.shape)}")
    N = x.shape[0]
    value = 0.0
    if isinstance(gate, torch.Tensor):
        if gate.dtype != x.dtype:
            raise TypeError(f"gate is {gate.dtype}, x {x.dtype}")
        if tuple(gate.shape) not in (tuple(x.shape), (N,)):
            raise ValueError(f"gate {tuple(gate.shape)} fits neither x {tuple(x.shape)} nor its {N} steps")
    else:
        value, gate = float(gate), None
    gradient = _seq.wants_gradient(x, gate, h0)
    _seq.recordable(not gradient, x, gate, h0)
    E = None
    if h0 is not None:
        if _seq.type_code("h0", h0) != code:
            raise TypeError(f"h0 is {h0.dtype}, x {x.dtype}")
        if h0.dim() != x.dim() or h0.shape[1:] != x.shape[1:]:
            raise ValueError(f"h0 {tuple(h0.shape)} does not hold a state like x {tuple(x.shape)} for every episode")
        E = h0.shape[0]
    off = _seq.offsets("ep_off", ep_off, N, E, validate)
    dev = _seq.on_device(("x", x), ("gate", gate), ("h0", h0), ("ep_off", off if off.is_cuda else None))
    if off.device != dev:
        off = _seq.from_host("ep_off", off, dev)
    if flat:
        x, h0 = x.unsqueeze(1), None if h0 is None else h0.unsqueeze(1)
    if gate is not None and gate.dim() == 1 and x.shape[1] == 1:
        gate = gate.unsqueeze(1)                              # one channel: shared or not is the same
    if gradient:
        out = _Recurrence.apply(x, gate, h0, off, value, bool(reverse), bool(want_last))
    else:
        h, last, _ = _seq.run_on(dev, _recurrence_forward, x, gate, off, h0, value, bool(reverse), bool(want_last), False)
        out = (h, last) if want_last else h
    if flat:
        out = tuple(o.squeeze(1) for o in out) if want_last else out.squeeze(1)
    return out


def check_recurrence(stream=None) -> None:
    """Waits for ``stream`` (a handle; default: the current one) and raises DcarlError if a recurrence on the current device gave up a wait between its
    workgroups since the last check: NaN stands behind it then.  No launch has been seen to; every wait ends by the order of the launch."""
    if _seq.capturing():
        raise ValueError("a stream cannot be waited for while a graph is captured: check after its replay")
    _lib.check(_lib.load().dcarl_recurrence_status(_lib.stream_ptr() if stream is None else C.c_void_p(stream)), "dcarl_recurrence_status")


def discounted_returns(rew, ep_off, gamma: float = 0.95, *, validate: bool = True):
    """``R[t] = rew[t] + gamma * R[t+1]`` to the end of each episode: the cumulative-reward column for a discount, where ``nstep_backup``
    has the field recorder's ten-step rule.  rew: (N,) (or (N, D): D streams side by side), a tensor of a type of ``gated_recurrence`` or anything
    that becomes a float64 one; moved to the GPU where it lies elsewhere.  For types below float64 gamma is rounded to f32 and states are held in f32: an error of
    about 3e-8 / (1 - gamma) of a return.  Where that is too much, as for discounts near 1, hand over float64 rewards."""
    gamma = _seq.number("gamma", gamma)
    if not isinstance(rew, torch.Tensor):
        rew = _dev64(rew, _lib.require_gpu())
    elif rew.device.type != "cuda":
        rew = rew.to(_lib.require_gpu())
    return gated_recurrence(rew, gamma, ep_off, reverse=True, validate=validate)
