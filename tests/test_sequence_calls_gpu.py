"""Calls of the sequence operators that the other tests do not make: operands from the host, lazily negated, written in place; arguments of the C-ABI that
the Python entry points never hand over; waits between workgroups that fail."""
import ctypes as C
import math
import os
import sys

import numpy as np
import pytest
import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, REPO)
from oracle import sequence_oracle as so  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dc():
    import dcarl_amd
    dcarl_amd.require_gpu()
    return dcarl_amd


def test_adjust_takes_histories_from_the_host(dc):
    s = torch.randn(3, 50, device="cuda")
    taken, off = [4, 4, 9, -1, 49], [0, 2, 2, 5]
    want = dc.candidates.adjust(s, torch.tensor(taken, device="cuda"), torch.tensor(off, device="cuda"), presence=0.5, frequency=0.25, repetition=1.5)
    assert torch.equal(dc.candidates.adjust(s, taken, off, presence=0.5, frequency=0.25, repetition=1.5, validate=True), want)
    assert torch.equal(dc.candidates.adjust(s, np.array(taken, dtype=np.int32), torch.tensor(off, device="cuda"), presence=0.5, frequency=0.25, repetition=1.5), want)
    changed = (want != s).nonzero().tolist()
    assert changed == [[0, 4], [2, 9], [2, 49]]


def test_adjust_in_place_is_seen_by_autograd(dc):
    p = torch.zeros(3, 40, device="cuda", requires_grad=True).exp()
    dc.candidates.adjust(p.detach(), bias=torch.ones(40, device="cuda"), out=p.detach())
    assert bool((p.detach() == 2).all())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        p.sum().backward()


def test_lazily_negated_operands(dc):
    z = torch.randn(40, 1, dtype=torch.complex64, device="cuda")
    x, off = z.conj().imag, [0, 11, 40]
    assert x.is_neg()
    want = dc.episodes.gated_recurrence(-z.imag, 0.5, off)
    assert torch.equal(dc.episodes.gated_recurrence(x, 0.5, off), want) and torch.equal(dc.episodes.gated_recurrence(x[:, 0], 0.5, off), want[:, 0])
    assert torch.equal(dc.tables.lookup(x, [3, 9, -1]), torch.cat([-z.imag[[3, 9]], torch.zeros(1, 1, device="cuda")]))
    assert torch.equal(dc.candidates.adjust(x), -z.imag)


def recurrence(dc, x, gate, off, h0, E, reverse=0):
    N, D = x.shape
    return dc._lib.CRecurrence(N=N, D=D, E=E, ep_off=off.data_ptr(), x=x.data_ptr(), ldx=D, gate=gate.data_ptr(), ldg=D, h0=h0, ldh0=D, gate_kind=2, reverse=reverse, type=1)


@pytest.mark.parametrize("N, D", [(40, 12), (3000, 12), (9000, 1)])
def test_c_abi_states_without_episodes_are_not_looked_at(dc, N, D):
    """No episode: h0 is an array of no rows, its address may be anything (here one row of NaN)."""
    lib, stream = dc.load_library(), dc._lib.stream_ptr()
    x, gate = torch.randn(N, D, device="cuda"), torch.rand(N, D, device="cuda")
    off, nan = torch.zeros(1, dtype=torch.int64, device="cuda"), torch.full((1, D), math.nan, device="cuda")
    r = recurrence(dc, x, gate, off, nan.data_ptr(), 0)
    sizes = (N, D, 0, 1, 2)
    states, ws = (torch.empty(f(*sizes) + 16, dtype=torch.uint8, device="cuda") for f in (lib.dcarl_recurrence_states_bytes, lib.dcarl_recurrence_workspace_bytes))
    h, dx, dg = (torch.full((N, D), math.nan, device="cuda") for _ in range(3))
    at = lambda t: C.c_void_p(t.data_ptr())      # noqa: E731
    assert lib.dcarl_recurrence_forward(C.byref(r), at(states), at(ws), at(h), None, stream) == 0
    assert lib.dcarl_recurrence_backward(C.byref(r), at(states), at(ws), at(x), D, None, at(dx), at(dg), None, stream) == 0
    assert not h.any() and not dx.any() and not dg.any()
