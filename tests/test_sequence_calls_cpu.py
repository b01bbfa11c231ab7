"""What the sequence operators hand to their kernels and leave behind, seen on the CPU: the launch is replaced by one that computes a marked result in
the same memory."""
import ctypes
import os
import sys

import numpy as np
import pytest
import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, REPO)
from dcarl_amd import _lib, _sequence, candidates, episodes, tables  # noqa: E402

OFF = torch.tensor([0, 2, 5])


def f32(address, n):
    return np.ctypeslib.as_array((ctypes.c_float * n).from_address(address)) if n else np.zeros(0, np.float32)


class Launches:
    """f32 operands alone: adjust adds 100, the recurrence 1000, its gradient is 7 dh; rows by numpy."""
    calls = 0

    def seen(self, a):
        """The first word of every operand, as it lies in memory during the launch."""
        self.first = {k: f32(p, 1)[0] for k, t in a._fields_ if t is ctypes.c_void_p and (p := getattr(a, k))}
        return a

    def dcarl_recurrence_states_bytes(self, *sizes):
        return 64

    dcarl_recurrence_workspace_bytes = dcarl_rows_workspace_bytes = dcarl_recurrence_states_bytes

    def dcarl_adjust_scores(self, a, out, ld, stream):
        self.calls += 1
        a = self.seen(a._obj)
        for b in range(a.B):
            f32(out + 4 * b * ld, a.V)[:] = f32(a.scores + 4 * b * a.ld_scores, a.V) + 100
        return 0

    def dcarl_recurrence_forward(self, a, states, ws, h, last, stream):
        self.calls += 1
        a = self.seen(a._obj)
        f32(h, a.N * a.D)[:] = np.concatenate([f32(a.x + 4 * n * a.ldx, a.D) for n in range(a.N)]) + 1000
        return 0

    def dcarl_recurrence_backward(self, a, states, ws, dh, lddh, dlast, dx, dgate, dh0, stream):
        self.calls += 1
        a = a._obj
        f32(dx, a.N * a.D)[:] = 7 * np.concatenate([f32(dh + 4 * n * lddh, a.D) for n in range(a.N)])
        return 0

    def dcarl_rows_gather(self, table, type_, ld, S, ids, width, N, D, scale, out, stream):
        self.calls += 1
        f32(out, N * D)[:] = scale * np.concatenate([f32(table + 4 * n * ld, D) for n in range(N)])
        return 0

    def dcarl_rows_gradient(self, dout, type_, ldd, ids, width, N, D, S, scale, ws, grad, stream):
        self.calls += 1
        f32(grad, S * D)[:] = np.concatenate([f32(dout + 4 * n * ldd, D) for n in range(S)])
        return 0


@pytest.fixture
def launches(monkeypatch):
    lib = Launches()
    monkeypatch.setattr(_lib, "load", lambda *a: lib)
    monkeypatch.setattr(_lib, "check", lambda *a: None)
    monkeypatch.setattr(_sequence, "on_device", lambda *named: torch.device("cpu"))
    monkeypatch.setattr(_sequence, "run_on", lambda device, call, *args: call(*args))
    monkeypatch.setattr(_sequence, "stream", lambda device: 0)
    return lib


def test_adjust_into_a_saved_tensor_is_seen_by_autograd(launches):
    for into in (lambda p: dict(out=p.detach()), lambda p: dict(out=p.detach()[:, :2], cut=2), lambda p: dict(out=p.detach(), apart=True)):
        kw = into(p := torch.zeros(3, 4, requires_grad=True).exp())           # exp keeps its result for its gradient
        scores = torch.zeros(3, 4) if kw.pop("apart", False) else p.detach()[:, :kw.pop("cut", 4)]
        candidates.adjust(scores, **kw)
        assert launches.calls and float(p.detach()[0, 0]) >= 100
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            p.sum().backward()
    fresh = torch.zeros(3, 4)
    candidates.adjust(fresh)
    assert fresh._version == 0                                               # nothing is written there
    with torch.inference_mode():
        kept = torch.zeros(3, 4)
        assert candidates.adjust(kept, out=kept) is kept


def test_tangents_are_refused_not_dropped(launches):
    x, h0, table, dout = torch.ones(5, 3), torch.ones(2, 3), torch.ones(4, 3), torch.ones(2, 3)
    gate, per_row = torch.ones(5, 3), torch.ones(5)
    need = torch.ones(5, 3, requires_grad=True)
    back = episodes.gated_recurrence(need, 0.5, OFF)
    rows_need = torch.ones(4, 3, requires_grad=True)
    rows_back = tables.lookup(rows_need, [0, 1])
    with torch.autograd.forward_ad.dual_level():
        dual = lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))      # noqa: E731
        before = launches.calls
        for call in (lambda: episodes.gated_recurrence(dual(x), 0.5, OFF),
                     lambda: episodes.gated_recurrence(dual(x).requires_grad_(), 0.5, OFF),
                     lambda: episodes.gated_recurrence(x, dual(gate), OFF),
                     lambda: episodes.gated_recurrence(x, dual(gate)[:, 0], OFF),
                     lambda: episodes.gated_recurrence(x, 0.5, OFF, dual(h0)),
                     lambda: episodes.gated_recurrence(need, gate, OFF, dual(h0)),
                     lambda: episodes.gated_recurrence(dual(x)[:, 0], 0.5, OFF, reverse=True),
                     lambda: torch.autograd.grad(back, need, dual(x)),
                     lambda: tables.lookup(dual(table), [0, 1]),
                     lambda: tables.lookup_gradient(dual(dout), [0, 1], 4),
                     lambda: torch.autograd.grad(rows_back, rows_need, dual(dout)),
                     lambda: candidates.adjust(dual(x)),
                     lambda: candidates.adjust(x, bias=dual(x)),
                     lambda: candidates.adjust(x, bias=dual(x)[0]),
                     lambda: candidates.adjust(x, repetition=dual(per_row)),
                     lambda: candidates.adjust(x, frequency=dual(per_row)),
                     lambda: candidates.adjust(x, presence=dual(per_row)),
                     lambda: candidates.adjust(x, out=dual(x.clone()))):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
        assert launches.calls == before
        episodes.gated_recurrence(x, 0.5, OFF)                               # no tangent: an ordinary call inside the level too
        assert launches.calls == before + 1
    episodes.gated_recurrence(x, 0.5, OFF)


def make_fx(f, *args):
    from torch.fx.experimental.proxy_tensor import make_fx
    return make_fx(f)(*args)


def test_a_trace_that_would_hold_no_launch_is_refused(launches):
    x, ids = torch.arange(15.0).view(5, 3), torch.tensor([0, 1])
    calls = (lambda x: episodes.gated_recurrence(x, 0.5, OFF, validate=False), lambda x: episodes.gated_recurrence(x[:, 0], 0.5, OFF, validate=False, want_last=True)[0],
             lambda x: tables.lookup(x, ids, validate=False), lambda x: tables.lookup_gradient(x[:2], ids, 4, validate=False), lambda x: candidates.adjust(x),
             lambda x: candidates.adjust(torch.zeros(5, 3), bias=x))
    for call in calls:
        with pytest.raises(ValueError, match="trace"):
            torch.jit.trace(call, x, check_trace=False)
        with pytest.raises(ValueError, match="trace"):
            make_fx(call, x)
        call(x)
    for call in calls[:3]:
        with pytest.raises(ValueError, match="trace"):                       # with gradients too: the launch is in no such record
            make_fx(call, x.clone().requires_grad_())
    # what runs the operators again on replay is a record of them: torch.jit.trace through the autograd function, torch.compile around them
    f = torch.jit.trace(calls[0], x.clone().requires_grad_(), check_trace=False)
    assert torch.equal(f(x + 1), x + 1001)
    y = (x + 2).requires_grad_()
    assert torch.equal(f(y), x + 1002) and torch.equal(torch.autograd.grad(f(y).sum(), y)[0], torch.full((5, 3), 7.0))


def test_operands_without_memory_are_refused_not_left_out(launches):
    """Wrappers that have a shape but no address: an optional operand of that kind must not count as absent."""
    x, h0, bias, allowed = torch.ones(5, 3), torch.ones(2, 3), torch.ones(3), torch.ones(1, dtype=torch.int32)
    functional = torch.func.functionalize
    for call, arg in ((lambda b: candidates.adjust(x, bias=b), bias), (lambda b: candidates.adjust(x, bias=b), torch.ones(5, 3)), (lambda b: candidates.adjust(x, allowed=b), allowed),
                      (lambda b: candidates.adjust(x, given=b), torch.ones(5, dtype=torch.int32)), (lambda b: candidates.adjust(x, repetition=b), torch.ones(5)),
                      (lambda b: candidates.adjust(x, b, torch.zeros(6, dtype=torch.int64)), torch.ones(2, dtype=torch.int64)),
                      (lambda b: candidates.adjust(x, torch.ones(2, dtype=torch.int64), b), torch.zeros(6, dtype=torch.int64)), (candidates.adjust, x),
                      (lambda b: episodes.gated_recurrence(x, 0.5, OFF, b), h0), (lambda b: episodes.gated_recurrence(x, b, OFF, h0), torch.ones(5)),
                      (lambda b: episodes.gated_recurrence(b, 0.5, OFF, h0), x), (lambda b: tables.lookup(b, [0, 1]), x), (lambda b: tables.lookup_gradient(b, [0, 1], 2), torch.ones(2, 3))):
        before = launches.calls
        with pytest.raises(ValueError, match="no memory"):
            functional(call)(arg)
        assert launches.calls == before
        call(arg)


def negated(t):
    """t as a lazily negated view: what lies in memory has the other sign."""
    n = torch.complex(torch.zeros_like(t), -t).conj().imag
    assert n.is_neg() and torch.equal(n, t)
    return n


def test_lazily_negated_operands_have_their_sign(launches):
    x, table = torch.randn(5, 3), torch.randn(4, 1)
    for v in (x, x[:, :1], x[:, 0]):
        assert torch.equal(episodes.gated_recurrence(negated(v), 0.5, OFF), v + 1000)
        need = v.clone().requires_grad_()
        h = episodes.gated_recurrence(need, 0.5, OFF)
        assert torch.equal(torch.autograd.grad(h, need, negated(v))[0], 7 * v)
        need = v.clone().requires_grad_()
        h = episodes.gated_recurrence(torch._neg_view(need), 0.5, OFF)       # through the view's own gradient
        assert torch.equal(h, 1000 - v) and torch.equal(torch.autograd.grad(h, need, torch.ones_like(h))[0], torch.full_like(v, -7))
    for gate in (x, x[:, 0]):
        episodes.gated_recurrence(x, negated(gate), OFF, negated(x[:2]))
        assert launches.first["gate"] == gate.flatten()[0] and launches.first["h0"] == x[0, 0]
    assert torch.equal(tables.lookup(negated(table), [0, 1]), table[:2]) and torch.equal(tables.lookup_gradient(negated(table), [0, 1, 2, 3], 2, validate=False), table[:2])
    need = torch.randn(4, 1, requires_grad=True)
    assert torch.equal(torch.autograd.grad(tables.lookup(need, [0, 1, 2, 3]), need, negated(table))[0], table)
    for s in (x, x[:, :1]):
        assert torch.equal(candidates.adjust(negated(s)), s + 100)
    for name, v in (("bias", x), ("bias", x[0]), ("repetition", x[:, 0].abs()), ("frequency", x[:, 0]), ("presence", x[:, 0])):
        candidates.adjust(x, **{name: negated(v)})
        assert launches.first[name] == v.flatten()[0]
    before = launches.calls
    with pytest.raises(ValueError, match="negated"):
        candidates.adjust(x, out=torch._neg_view(torch.zeros(5, 3)))
    assert launches.calls == before


def test_gradients_that_no_one_would_get_are_refused(launches):
    dout = torch.ones(2, 3, requires_grad=True)
    k = torch.tensor(0.5, requires_grad=True)
    x, ids = torch.ones(4, 3), [0, 1]
    for call in (lambda: tables.lookup_gradient(dout, ids, 4), lambda: tables.lookup_gradient(dout.detach(), ids, 4, k), lambda: tables.lookup(x, ids, k),
                 lambda: tables.lookup(x.clone().requires_grad_(), ids, k), lambda: episodes.discounted_returns(x, [0, 4], k), lambda: episodes.gated_recurrence(x, 0.5 * k, [0, 4]),
                 lambda: candidates.adjust(x, frequency=k)):
        with pytest.raises(ValueError):
            call()
    assert launches.calls == 0
    with torch.no_grad():
        assert torch.equal(tables.lookup_gradient(dout, ids, 2), torch.ones(2, 3)) and torch.equal(tables.lookup(x, ids, k), torch.full((2, 3), 0.5))
    assert torch.equal(tables.lookup(x, ids, k.detach()), torch.full((2, 3), 0.5))


def test_adjust_takes_histories_from_the_host(monkeypatch):
    """As the other two take their ids and offsets: whole numbers on the host are moved to the scores' device."""
    seen, moved = {}, []
    monkeypatch.setattr(_sequence, "on_device", lambda *named: seen.update(named) or torch.device("meta"))
    monkeypatch.setattr(_sequence, "run_on", lambda device, call, *args: moved.extend(args))
    scores = torch.zeros(2, 5, device="meta")
    candidates.adjust(scores, [1, 2, 4], [0, 1, 3])
    assert seen["taken"] is None and seen["taken_off"] is None and seen["scores"] is scores
    assert [t.device.type for t in moved if isinstance(t, torch.Tensor)] == ["meta"] * 3
    monkeypatch.setattr(_sequence, "capturing", lambda: True)
    for kw in (dict(taken=[1, 2, 4], taken_off=torch.zeros(3, dtype=torch.int64, device="meta")), dict(taken=torch.zeros(3, dtype=torch.int64, device="meta"), taken_off=[0, 1, 3])):
        with pytest.raises(ValueError, match="captured"):
            candidates.adjust(scores, **kw)
