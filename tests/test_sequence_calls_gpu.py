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


@pytest.mark.parametrize("N, D", [(9000, 12), (400_000, 1), (30_000, 70), (100, 5)])
def test_c_abi_backward_of_states_that_no_forward_pass_wrote(dc, N, D):
    """The values are anything, but only the call's own rows are written, and every wait ends: flags, episodes and tiles read from the states stay inside."""
    lib, stream, E = dc.load_library(), dc._lib.stream_ptr(), 3
    gen = torch.Generator(device="cuda").manual_seed(N)
    x, gate = torch.randn(N, D, device="cuda", generator=gen), torch.rand(N, D, device="cuda", generator=gen)
    off = torch.tensor([0, N // 3, N // 2, N], device="cuda")
    rows = torch.full((4, 5 * E, D), 7.0, device="cuda")                  # h0, dlast, dh0, dx's guard
    at = lambda t: C.c_void_p(t.data_ptr())      # noqa: E731
    r = recurrence(dc, x, gate, off, rows[0, 2 * E].data_ptr(), E)
    sizes = (N, D, E, 1, 2)
    states = torch.randint(0, 256, (lib.dcarl_recurrence_states_bytes(*sizes),), dtype=torch.uint8, device="cuda", generator=gen)
    ws = torch.empty(lib.dcarl_recurrence_workspace_bytes(*sizes) + 16, dtype=torch.uint8, device="cuda")
    out = torch.full((2, N + 2, D), 7.0, device="cuda")
    for fill in (None, 0, 255, 127):
        if fill is not None:
            states.fill_(fill)
        assert lib.dcarl_recurrence_backward(C.byref(r), at(states), at(ws), at(x), D, at(rows[1, 2 * E]), at(out[0, 1]), at(out[1, 1]), at(rows[2, 2 * E]), stream) == 0
        torch.cuda.synchronize()
        assert bool((out[:, [0, N + 1]] == 7).all()) and bool((rows[[0, 1, 3]] == 7).all()) and bool((rows[2, :2 * E] == 7).all()) and bool((rows[2, 3 * E:] == 7).all())


def test_backward_of_a_captured_forward_pass_before_and_after_its_replay(dc):
    N, off = 5000, torch.tensor([0, 1700, 1700, 5000], device="cuda")
    x, gate, h0 = torch.randn(N, 9, device="cuda"), torch.rand(N, 9, device="cuda"), torch.randn(3, 9, device="cuda")
    leaf = [v.clone().requires_grad_() for v in (x, gate, h0)]
    want = torch.autograd.grad(dc.episodes.gated_recurrence(leaf[0], leaf[1], off, leaf[2]), leaf, torch.ones_like(x))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        dc.episodes.gated_recurrence(leaf[0], leaf[1], off, leaf[2], validate=False)
    torch.cuda.current_stream().wait_stream(side)
    mine = [v.detach().requires_grad_() for v in leaf]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h = dc.episodes.gated_recurrence(mine[0], mine[1], off, mine[2], validate=False)
    torch.autograd.grad(h, mine, torch.ones_like(x), retain_graph=True)    # of states not written yet: any values, no access out of range
    torch.cuda.synchronize()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(h, mine, torch.ones_like(x)), want))


@pytest.fixture
def no_polls(dc):
    """Every wait between workgroups is given up at its first poll, from here to the end of the test."""
    lib = dc.load_library()
    assert lib.dcarl_recurrence_status(dc._lib.stream_ptr()) == 0
    lib.dcarl_debug_recurrence_polls(0)
    try:
        yield lib
    finally:
        lib.dcarl_debug_recurrence_polls(-1)
        torch.cuda.synchronize()
        lib.dcarl_recurrence_status(dc._lib.stream_ptr())


@pytest.mark.parametrize("D, tile, t", [(9, 512, torch.float32), (9, 512, torch.bfloat16), (1, 4096, torch.float32), (1, 2048, torch.float64), (40, 128, torch.float16)])
def test_waits_given_up_are_reported(dc, no_polls, D, tile, t):
    off = [0, 3 * tile + 100, 20 * tile, 20 * tile, 22 * tile + 7]
    N = off[-1]
    episode = np.searchsorted(off, np.arange(N), side="right") - 1
    starts, ends = np.array(off)[episode], np.array(off)[episode + 1] - 1
    x, gate = torch.ones(N, D, device="cuda", dtype=t), torch.full((N, D), 0.5, device="cuda", dtype=t)
    leaf = [x.requires_grad_(), gate.requires_grad_()]
    no_polls.dcarl_debug_recurrence_polls(-1)
    want = dc.episodes.gated_recurrence(*leaf, off)
    grads = torch.autograd.grad(want, leaf, torch.ones_like(x), retain_graph=True)
    dc.episodes.check_recurrence()                                        # nothing was given up
    no_polls.dcarl_debug_recurrence_polls(0)
    dc.episodes.gated_recurrence(x[:90].detach(), 0.5, [0, 90])          # one tile waits for nothing
    dc.episodes.check_recurrence()
    inside = torch.tensor(starts // tile == np.arange(N) // tile, device="cuda")           # the episode starts in the step's own tile: no wait
    for _ in range(2):
        got = dc.episodes.gated_recurrence(x.detach(), gate.detach(), off)
        with pytest.raises(dc.DcarlError, match="given up"):
            dc.episodes.check_recurrence()
        dc.episodes.check_recurrence()                                    # asking clears it
        assert torch.equal(got[inside], want[inside]) and bool(got[~inside].isnan().all())
    inside = torch.tensor(ends // tile == np.arange(N) // tile, device="cuda")
    for a, b in zip(torch.autograd.grad(want, leaf, torch.ones_like(x)), grads):
        assert torch.equal(a[inside], b[inside]) and bool(a[~inside].isnan().all())
    assert no_polls.dcarl_recurrence_status(dc._lib.stream_ptr()) == -3 and b"given up" in no_polls.dcarl_last_error()
    no_polls.dcarl_debug_recurrence_polls(-1)
    assert torch.equal(dc.episodes.gated_recurrence(x.detach(), gate.detach(), off), want)
    dc.episodes.check_recurrence()


def test_waits_are_not_checked_while_a_graph_is_captured(dc):
    x = torch.ones(5000, 3, device="cuda")
    off = torch.tensor([0, 5000], device="cuda")
    want = dc.episodes.gated_recurrence(x, 0.5, off)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h = dc.episodes.gated_recurrence(x, 0.5, off, validate=False)
        with pytest.raises(ValueError, match="captured"):
            dc.episodes.check_recurrence()
    for _ in range(3):
        graph.replay()
        dc.episodes.check_recurrence()
        assert torch.equal(h, want)
