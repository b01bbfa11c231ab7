"""Candidate scores before the arg-max: penalties for what was taken already, biases, masks.

``frenet.select`` and the gates of ``rls`` decide between a few trajectories; here a policy's scores over any number of candidates are adjusted
by each observation's own history, by biases, and by which candidates are allowed (``frenet``'s feasibility bits, a grammar's next symbols)."""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib, _sequence as _seq

SCORE_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def pack_allowed(allowed):
    """(..., V) truth values -> (..., ceil(V/32)) int32 words as ``adjust`` wants them: candidate v in bit v % 32 of word v // 32."""
    allowed = torch.as_tensor(allowed).to(torch.bool)
    V = allowed.shape[-1]
    bits = torch.nn.functional.pad(allowed, (0, -V % 32)).unflatten(-1, (-1, 32)).to(torch.int64) if V else allowed.new_zeros((*allowed.shape[:-1], 0, 32), dtype=torch.int64)
    words = (bits << torch.arange(32, device=allowed.device)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def _strength(name, v, B):
    """A number, or a float32 tensor with one per row."""
    if isinstance(v, torch.Tensor):
        if v.dtype != torch.float32 or v.shape != (B,):
            raise ValueError(f"{name} must be a number or a float32 tensor ({B},), not {v.dtype} {tuple(v.shape)}")
        return _seq.plain(v).contiguous(), 0.0
    v = float(v)
    if v != v or (name == "repetition" and not v > 0.0):
        raise ValueError(f"{name} = {v}" + (" is not positive" if name == "repetition" else ""))
    return None, v


def _per_row(name, t, B, width, dtype):
    if t is None:
        return None, 0
    if not isinstance(t, torch.Tensor) or t.dtype != dtype:
        raise TypeError(f"{name} must be a {dtype} tensor")
    if t.shape == (width,):
        return (_seq.plain(t) if dtype.is_floating_point else t).contiguous(), 0
    if t.shape != (B, width):
        raise ValueError(f"{name} {tuple(t.shape)} is neither ({width},) nor ({B}, {width})")
    return _seq.rows_of(t)


def _half_over(scores, out) -> bool:
    """Whether rows of out share memory with other places of scores (out being scores itself is fine)."""
    B, V = scores.shape
    if not (B and V) or out.device != scores.device or (out.data_ptr() == scores.data_ptr() and (B == 1 or out.stride(0) == scores.stride(0)) and (V == 1 or scores.stride(1) == 1)):
        return False
    if V > 1 and scores.stride(1) != 1 or scores.stride(0) < 0:
        return False                                         # read from a copy
    size = scores.element_size()
    a0, b0 = scores.data_ptr(), out.data_ptr()
    la, lb = scores.stride(0), out.stride(0)
    if a0 + ((B - 1) * la + V) * size <= b0 or b0 + ((B - 1) * lb + V) * size <= a0:
        return False
    if B > 1 and la == lb and (b0 - a0) % size == 0:         # side by side in one wider buffer
        d = (b0 - a0) // size % la
        return d < V or la - d < V
    return True


def _end(t) -> int:
    """The address behind a tensor's last element."""
    return t.data_ptr() + (1 + sum((n - 1) * step for n, step in zip(t.shape, t.stride()))) * t.element_size()


def _over(t, out) -> bool:
    """Whether an operand that all of a row's workgroups read shares memory with out."""
    return t is not None and t.device == out.device and t.numel() > 0 and out.numel() > 0 and t.data_ptr() < _end(out) and out.data_ptr() < _end(t)


def adjust(scores, taken=None, taken_off=None, *, given=None, repetition=1.0, frequency=0.0, presence=0.0, bias=None, allowed=None, out=None,
           validate: bool = False):
    """For each of B rows of V scores:  z = score;  taken before: z = z / r if z > 0 else z * r;  z -= f * n + p where n > 0;
    z += bias;  z = -inf where not allowed, whatever it was.  -> (B, V) of the scores' type, computed in f32, rounded once.

    scores: (B, V) float32, bfloat16 or float16, rows at any distance.  taken: the rows' histories one after the other (int32 or int64 ids, moved
    to the GPU where they lie on the host, as taken_off is; ids outside [0, V), such as -1, count nowhere), row b's is ``taken[taken_off[b]:taken_off[b+1]]``.  given: (B,) int32, how many
    entries at a history's front were handed to the policy and not chosen by it: ``n`` counts the others, "taken before" looks at all.
    repetition (> 0), frequency, presence: r, f, p, a number or a float32 tensor (B,).  bias: float32 (V,) or (B, V).
    allowed: int32 words of ``pack_allowed``, (ceil(V/32),) or (B, ceil(V/32)); a row that allows nothing is -inf throughout.
    out: where the result goes; ``out=scores`` adjusts in place, and out lies over no other operand.  Autograd sees that write as it sees torch's own
    in-place ones: a gradient that needs what out held before raises.  validate: check taken_off's values (waits for them when they are on
    the GPU); without it, which is the default since this call stands in an answer's path, offsets are held to the range of ``taken``.
    No gradient flows through: scores that require one, or carry a tangent, are refused, and so is a call under torch.jit.trace or make_fx, whose record would not hold it."""
    if not isinstance(scores, torch.Tensor) or scores.dtype not in SCORE_TYPES:
        raise TypeError("scores must be a float32, bfloat16 or float16 tensor")
    if scores.dim() != 2:
        raise ValueError(f"scores must be (B, V), not {tuple(scores.shape)}")
    if _seq.wants_gradient(scores, *[t if isinstance(t, torch.Tensor) else None for t in (repetition, frequency, presence, bias)]):
        raise ValueError("adjust has no gradient: detach the scores, strengths and biases")
    _seq.recordable(True, scores, repetition, frequency, presence, bias, out)
    B, V = scores.shape
    if (taken is None) != (taken_off is None):
        raise ValueError("taken and taken_off come together")
    off = None
    if taken is not None:
        taken = _seq.whole_numbers("taken", taken)
        if taken.dim() != 1:
            raise ValueError("taken must be one-dimensional")
        taken = taken.contiguous()
        off = _seq.offsets("taken_off", taken_off, taken.numel(), B, validate)
    if given is not None and (not isinstance(given, torch.Tensor) or given.dtype != torch.int32 or given.shape != (B,)):
        raise ValueError(f"given must be an int32 tensor ({B},)")
    (rep, rep0), (freq, freq0), (pres, pres0) = (_strength(n, v, B) for n, v in (("repetition", repetition), ("frequency", frequency), ("presence", presence)))
    bias, ld_bias = _per_row("bias", bias, B, V, torch.float32)
    allowed, ld_allowed = _per_row("allowed", allowed, B, (V + 31) // 32, torch.int32)
    if out is not None:
        if not isinstance(out, torch.Tensor) or out.dtype != scores.dtype or out.shape != scores.shape:
            raise ValueError(f"out must be a {scores.dtype} tensor {tuple(scores.shape)}")
        if V > 1 and out.stride(1) != 1 or B > 1 and out.stride(0) < V:
            raise ValueError("out must have contiguous rows that do not overlap")
        if out.is_neg():
            raise ValueError("out is a lazily negated view")
        if out.requires_grad:
            raise ValueError("out requires a gradient")
        if _half_over(scores, out):
            raise ValueError("out lies partly over scores: it is scores itself or apart from it")
        for name, t in (("taken", taken), ("taken_off", off), ("given", given), ("repetition", rep), ("frequency", freq), ("presence", pres), ("allowed", allowed)):
            if _over(t, out):
                raise ValueError(f"out lies over {name}")
        if bias is not None and (_half_over(bias, out) if bias.dim() == 2 and bias.dtype == out.dtype else _over(bias, out)):
            raise ValueError("out lies partly over bias: it is bias itself or apart from it")
    dev = _seq.on_device(("scores", scores), ("taken", taken if taken is not None and taken.is_cuda else None), ("taken_off", off if off is not None and off.is_cuda else None), ("given", given), ("repetition", rep), ("frequency", freq),
                         ("presence", pres), ("bias", bias), ("allowed", allowed), ("out", out))
    if taken is not None and taken.device != dev:
        taken = _seq.from_host("taken", taken, dev)
    if off is not None and off.device != dev:
        off = _seq.from_host("taken_off", off, dev)
    return _seq.run_on(dev, _adjust, scores, taken, off, given, rep, rep0, freq, freq0, pres, pres0, bias, ld_bias, allowed, ld_allowed, out)


def _adjust(scores, taken, off, given, rep, rep0, freq, freq0, pres, pres0, bias, ld_bias, allowed, ld_allowed, out):
    B, V = scores.shape
    dev = scores.device
    s, ld = _seq.rows_of(scores)
    z = _seq.like(s) if out is None else out
    given = None if given is None else given.contiguous()
    at = _seq.at
    a = _lib.CScores(at(s), B, V, ld, at(taken), at(off), 0 if taken is None else taken.numel(), at(given), at(rep), at(freq), at(pres), at(bias),
                     ld_bias, at(allowed), ld_allowed, rep0 if rep is None else 1.0, freq0, pres0, _seq.TYPES[s.dtype],
                     4 if taken is None else taken.element_size(), 0)
    _lib.check(_lib.load().dcarl_adjust_scores(C.byref(a), at(z), z.stride(0), _seq.stream(dev)), "dcarl_adjust_scores")
    if out is not None:
        torch.autograd.graph.increment_version(out)          # written through its address: autograd sees what it saved there change
    return z
