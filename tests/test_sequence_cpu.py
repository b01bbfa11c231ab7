"""The sequence operators without a GPU: their definitions by hand (oracle/sequence_oracle.py), the checks of arguments of the Python entry points
and of the C-ABI, the packing of masks."""
import ctypes as C
import os
import sys

import numpy as np
import pytest
import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, REPO)
from dcarl_amd import DcarlError, _lib, candidates, episodes, load_library, tables  # noqa: E402
from oracle import sequence_oracle as so  # noqa: E402


# ---- the definitions ---------------------------------------------------------------------------------------------------
def test_recurrence_by_hand():
    x = np.array([[1.0], [2.0], [3.0], [4.0]])
    h, prev, last = so.recurrence(x, 0.5, [0, 1, 1, 4], h0=np.array([[2.0], [7.0], [4.0]]))
    assert h[:, 0].tolist() == [2.0, 4.0, 5.0, 6.5] and prev[:, 0].tolist() == [2.0, 4.0, 4.0, 5.0] and last[:, 0].tolist() == [2.0, 7.0, 6.5]
    h, _, last = so.recurrence(x, 0.5, [0, 1, 1, 4], reverse=True)                   # discounted returns: 2 + .5*(3 + .5*4) ...
    assert h[:, 0].tolist() == [1.0, 4.5, 5.0, 4.0] and last[:, 0].tolist() == [1.0, 0.0, 4.5]


def test_recurrence_gradients_against_differences():
    rng = np.random.default_rng(0)
    off, N, D = [0, 3, 3, 8], 8, 2
    x, g, h0, w, wl = rng.normal(size=(N, D)), rng.uniform(0.2, 1.1, (N, D)), rng.normal(size=(3, D)), rng.normal(size=(N, D)), rng.normal(size=(3, D))
    for reverse in (False, True):
        def f(x, g, h0):
            h, _, last = so.recurrence(x, g, off, h0, reverse)
            return (h * w).sum() + (last * wl).sum()
        _, prev, _ = so.recurrence(x, g, off, h0, reverse)
        got = so.recurrence_gradients(w, g, prev, off, wl, reverse)
        for k, a in enumerate((x, g, h0)):
            for i in np.ndindex(a.shape):
                lo, hi = a.copy(), a.copy()
                lo[i] -= 1e-5
                hi[i] += 1e-5
                args = [x, g, h0]
                d = (f(*(args[:k] + [hi] + args[k + 1:])) - f(*(args[:k] + [lo] + args[k + 1:]))) / 2e-5
                assert got[k][i] == pytest.approx(d, rel=1e-6, abs=1e-8)            # central differences: error ~ 1e-10 f''' + 1e-11


def test_rows_and_scores_by_hand():
    t = np.array([[1.0, 2.0], [3.0, 4.0]])
    assert so.rows(t, [1, -1, 0, 5], 2.0).tolist() == [[6, 8], [0, 0], [2, 4], [0, 0]]
    g, _, n = so.rows_gradient(np.arange(8.0).reshape(4, 2), [1, -1, 1, 0], 3, 2.0)
    assert g.tolist() == [[12, 14], [8, 12], [0, 0]] and n.tolist() == [1, 2, 0]
    z, _ = so.adjust([[2.0, -2.0, 1.0, 0.0]], taken=[0, 1, 2, 2, -1, 9], taken_off=[0, 6], given=[1], repetition=2.0, frequency=0.25, presence=0.5,
                     bias=[0, 0, 0, 1.0], allowed=[True, True, True, True])
    # 0: given only: 2/2.  1: -2*2 - .25 - .5.  2: 1/2 - .25*2 - .5.  3: never taken, bias alone
    assert z.tolist() == [[1.0, -4.75, -0.5, 1.0]]
    assert so.adjust([[1.0, np.nan]], allowed=[False, False])[0].tolist() == [[-np.inf, -np.inf]]


def test_pack_allowed():
    a = torch.zeros(2, 70, dtype=torch.bool)
    a[0, 0] = a[0, 31] = a[0, 32] = a[1, 69] = True
    w = candidates.pack_allowed(a)
    assert w.dtype == torch.int32 and w.tolist() == [[1 - (1 << 31), 1, 0], [0, 0, 1 << 5]]
    assert candidates.pack_allowed([True, False, True]).tolist() == [5] and candidates.pack_allowed(torch.zeros(2, 0)).shape == (2, 0)


# ---- refusals of the Python entry points: every one before anything reaches a GPU ----------------------------------------
X, G, H0 = torch.zeros(5, 3), torch.ones(5, 3), torch.zeros(2, 3)
OFF = torch.tensor([0, 2, 5])


@pytest.mark.parametrize("kw, error, text", [
    (dict(x=[1.0]), TypeError, "tensor"),
    (dict(x=X.int()), TypeError, "int32"),
    (dict(x=torch.zeros(5, 3, 1)), ValueError, "x must be"),
    (dict(gate=G.double()), TypeError, "gate"),
    (dict(gate=G[:4]), ValueError, "fits neither"),
    (dict(gate=torch.ones(3)), ValueError, "fits neither"),
    (dict(h0=H0.half()), TypeError, "h0"),
    (dict(h0=H0[:, :2]), ValueError, "h0"),
    (dict(h0=torch.zeros(3, 3)), ValueError, "4 are needed"),
    (dict(ep_off=torch.tensor([0.0, 5.0])), TypeError, "int32 or int64"),
    (dict(ep_off=torch.zeros(0, dtype=torch.int64)), ValueError, "one-dimensional"),
    (dict(ep_off=torch.tensor([[0, 2, 5]])), ValueError, "one-dimensional"),
    (dict(ep_off=[0, 2, 6]), ValueError, "rise from 0 to at most 5"),
    (dict(ep_off=[1, 2, 5]), ValueError, "rise from 0"),
    (dict(ep_off=[0, 4, 3]), ValueError, "rise from 0"),
    (dict(), DcarlError, "no CPU path"),
])
def test_recurrence_refusals(kw, error, text):
    args = dict(x=X, gate=G, ep_off=OFF, h0=H0)
    args.update(kw)
    with pytest.raises(error, match=text):
        episodes.gated_recurrence(args.pop("x"), args.pop("gate"), args.pop("ep_off"), **args)


def test_returns_refuses_without_gpu():
    if torch.cuda.is_available():
        pytest.skip("a GPU is here")
    with pytest.raises(DcarlError):
        episodes.discounted_returns([1.0, 2.0], [0, 2])


@pytest.mark.parametrize("table, ids, error, text", [
    (torch.zeros(4, 3).long(), [0], TypeError, "int64"),
    (torch.zeros(4), [0], ValueError, r"\(S, D\)"),
    (torch.zeros(4, 3), [0.5], TypeError, "int32 or int64"),
    (torch.zeros(4, 3), [0, 4], IndexError, r"\[0,4\] vs 4"),
    (torch.zeros(4, 3), [-2, 0], IndexError, r"\[-2,0\]"),
    (torch.zeros(4, 3), [-1, 3], DcarlError, "no CPU path"),
])
def test_lookup_refusals(table, ids, error, text):
    with pytest.raises(error, match=text):
        tables.lookup(table, ids)


@pytest.mark.parametrize("dout, ids, n, error, text", [
    (torch.zeros(2, 3), [0], 4, ValueError, "no row for each"),
    (torch.zeros(1, 3), [4], 4, IndexError, "vs 4 rows"),
    (torch.zeros(1, 3), [0], -1, ValueError, "negative"),
    (torch.zeros(1, 3), [0], 4, DcarlError, "no CPU path"),
])
def test_lookup_gradient_refusals(dout, ids, n, error, text):
    with pytest.raises(error, match=text):
        tables.lookup_gradient(dout, ids, n)


S = torch.zeros(2, 40)


@pytest.mark.parametrize("scores, kw, error, text", [
    (S.double(), {}, TypeError, "float32, bfloat16"),
    (S[0], {}, ValueError, r"\(B, V\)"),
    (S.clone().requires_grad_(), {}, ValueError, "no gradient"),
    (S, dict(taken=torch.tensor([1])), ValueError, "together"),
    (S, dict(taken=torch.tensor([1.0]), taken_off=[0, 1, 1]), TypeError, "int32 or int64"),
    (S, dict(taken=torch.tensor([1]), taken_off=[0, 1]), ValueError, "3 are needed"),
    (S, dict(taken=torch.tensor([1]), taken_off=[0, 2, 1], validate=True), ValueError, "rise from 0"),
    (S, dict(given=torch.zeros(2)), ValueError, "given"),
    (S, dict(repetition=0.0), ValueError, "not positive"),
    (S, dict(repetition=float("nan")), ValueError, "nan"),
    (S, dict(frequency=torch.zeros(3)), ValueError, "frequency"),
    (S, dict(presence=torch.zeros(2).double()), ValueError, "presence"),
    (S, dict(bias=torch.zeros(41)), ValueError, "bias"),
    (S, dict(bias=torch.zeros(40).half()), TypeError, "bias"),
    (S, dict(allowed=torch.zeros(2, 40, dtype=torch.bool)), TypeError, "allowed"),
    (S, dict(allowed=torch.zeros(2, 3, dtype=torch.int32)), ValueError, "allowed"),
    (S, dict(out=S.half()), ValueError, "out must be"),
    (S, dict(out=torch.zeros(1, 40).expand(2, 40)), ValueError, "overlap"),
    (S, dict(out=torch.zeros(40, 2).t()), ValueError, "contiguous rows"),
    (S, dict(out=torch.zeros(2, 40, requires_grad=True)), ValueError, "out requires"),
    (S, dict(bias=torch.zeros(40, requires_grad=True)), ValueError, "no gradient"),
    (S, dict(presence=torch.zeros(2, requires_grad=True)), ValueError, "no gradient"),
    (S, {}, DcarlError, "no CPU path"),
])
def test_adjust_refusals(scores, kw, error, text):
    with pytest.raises(error, match=text):
        candidates.adjust(scores, **kw)


def test_adjust_refuses_out_half_over_scores():
    wide = torch.zeros(4, 100)
    for s, o in ((wide[:, :40], wide[:, 39:79]), (wide[:, 10:50], wide[:, :40]), (wide[:, 60:], wide[1:, :40]), (wide[:3, :40], wide[1:, :40]), (wide[0:1, :40], wide[0:1, 20:60])):
        if s.shape == o.shape:
            with pytest.raises(ValueError, match="partly over"):
                candidates.adjust(s, out=o)
    for s, o in ((wide[:, :40], wide[:, 40:80]), (wide[:, 60:], wide[:, :40]), (wide[:2, :40], wide[2:, :40]), (wide[:, :40], wide[:, :40]), (wide[0:1, :40], wide[0:1, 40:80])):
        with pytest.raises(DcarlError, match="no CPU path"):            # past every other check
            candidates.adjust(s, out=o)


# ---- the C-ABI: refused before any launch (the addresses are fakes) --------------------------------------------------------
def test_c_abi_refusals():
    if torch.cuda.is_available():
        pytest.skip("fake addresses: only where nothing can run")
    lib = load_library()
    one, odd, null = C.c_void_p(16), C.c_void_p(8), C.c_void_p(None)
    assert C.sizeof(_lib.CRecurrence) == 13 * 8 and C.sizeof(_lib.CScores) == 15 * 8 + 6 * 4
    err = lambda: lib.dcarl_last_error().decode()      # noqa: E731

    def rec(**kw):
        a = dict(N=4, D=3, E=2, ep_off=16, x=16, ldx=3, gate=16, ldg=3, h0=0, ldh0=0, gate_value=0.0, gate_kind=2, reverse=0, type=1)
        a.update(kw)
        return C.byref(_lib.CRecurrence(**a))
    fwd = lambda r, **k: lib.dcarl_recurrence_forward(r, k.get("states", null), k.get("ws", one), k.get("h", one), null, null)      # noqa: E731
    for kw, text in ((dict(type=4), "type=4"), (dict(N=-1), "out of range"), (dict(N=1 << 31), "out of range"), (dict(N=1 << 30, D=1 << 30), "out of range"),
                     (dict(gate_kind=3), "gate_kind"), (dict(ldx=-1), "ldx"), (dict(ep_off=0), "ep_off"), (dict(x=0), "x / gate"), (dict(gate=0), "x / gate")):
        assert fwd(rec(**kw)) == -1 and text in err(), kw
    assert fwd(rec(ldx=1 << 40)) == -1 and fwd(rec(ldg=1 << 40)) == -1 and "ldg" in err()
    assert lib.dcarl_recurrence_forward(None, null, one, one, null, null) == -1
    assert fwd(rec(), h=null) == -1 and "h is NULL" in err()
    assert fwd(rec(), states=odd) == -1 and "alignment" in err()
    assert fwd(rec(N=0, E=0)) == 0 and fwd(rec(D=0)) == 0
    bwd = lambda r, dh=one, lddh=3, dg=null, st=one: lib.dcarl_recurrence_backward(r, st, one, dh, lddh, null, one, dg, null, null)      # noqa: E731
    assert bwd(rec(gate_kind=0), dg=one) == -1 and "no gradient" in err()
    assert bwd(rec(), dh=null) == -1 and bwd(rec(), st=null) == -1 and bwd(rec(), lddh=-3) == bwd(rec(), lddh=1 << 40) == -1
    assert lib.dcarl_recurrence_workspace_bytes(-1, 3, 2, 1, 2) == 0 and lib.dcarl_recurrence_states_bytes(4, 3, 2, 9, 2) == 0

    g = lambda t=one, ty=1, ld=3, ids=one, ib=8, n=4, out=one: lib.dcarl_rows_gather(t, ty, ld, 5, ids, ib, n, 3, 1.0, out, null)      # noqa: E731
    assert g(t=null) == g(ids=null) == g(out=null) == g(ty=7) == g(ib=2) == g(ld=-1) == g(n=-4) == -1 and g(n=0) == 0
    gr = lambda d=one, ids=one, ws=one, out=one, n=4, s=5: lib.dcarl_rows_gradient(d, 1, 3, ids, 4, n, 3, s, 1.0, ws, out, null)      # noqa: E731
    assert lib.dcarl_rows_gather(one, 1, 3, 5, one, 8, 4, (1 << 23) + 1, 1.0, one, null) == -1 and "above" in err()
    assert gr(d=null) == gr(ids=null) == gr(ws=null) == gr(out=null) == gr(s=-5) == -1 and gr(ws=odd) == -1 and "alignment" in err() and gr(s=0) == 0
    assert lib.dcarl_rows_workspace_bytes(1 << 31, 5, 3, 1) == 0 and lib.dcarl_rows_workspace_bytes(100, 5, 3, 1) > 0

    def sc(ld_out=40, out=one, **kw):
        a = dict(scores=32, B=2, V=40, ld_scores=40, repetition_value=1.0, type=1, id_bytes=4)
        a.update(kw)
        return lib.dcarl_adjust_scores(C.byref(_lib.CScores(**a)), out, ld_out, null)
    for kw, text in ((dict(type=0), "DCARL_F32"), (dict(scores=0), "scores / out"), (dict(out=null), "scores / out"), (dict(ld_out=39), "overlap"),
                     (dict(scores=16, ld_scores=48), "in place"), (dict(taken_off=16, n_taken=3), "taken is NULL"),
                     (dict(taken_off=16, taken=16, n_taken=3, id_bytes=2), "id_bytes"), (dict(repetition_value=0.0), "not positive"),
                     (dict(repetition_value=float("nan")), "not positive"), (dict(B=-1), "out of range"), (dict(ld_bias=-1), "ld_bias")):
        assert sc(**kw) == -1 and text in err(), kw
    assert sc(B=0) == 0 and lib.dcarl_adjust_scores(None, one, 40, null) == -1


def test_c_abi_steps_without_offsets_are_refused():
    if torch.cuda.is_available():
        pytest.skip("fake addresses: only where nothing can run")
    lib = load_library()
    one, null = C.c_void_p(16), C.c_void_p(None)
    for N in (4, 5000):                                       # no episode is one offset, not none
        r = C.byref(_lib.CRecurrence(N=N, D=3, E=0, ep_off=0, x=16, ldx=3, gate=16, ldg=3, gate_kind=2, type=1))
        for rc in (lib.dcarl_recurrence_forward(r, null, one, one, null, null), lib.dcarl_recurrence_backward(r, one, one, one, 3, null, one, one, null, null)):
            assert rc == -1 and "ep_off is NULL" in lib.dcarl_last_error().decode()


def test_adjust_refuses_out_over_what_a_row_reads():
    from dcarl_amd import candidates
    s, n = torch.zeros(2, 32), 2 * 32
    buf = torch.zeros(3 * n)
    out = buf[:n].view(2, 32)
    for kw in (dict(bias=buf[n - 1:n + 31]), dict(bias=buf[:32]), dict(bias=buf[32:96].view(2, 32)), dict(bias=buf[:32].expand(2, 32)), dict(frequency=buf[10:12]),
               dict(presence=buf[62:64]), dict(given=buf.view(torch.int32)[:2]), dict(allowed=buf.view(torch.int32)[63:64]),
               dict(taken=buf.view(torch.int32)[60:70], taken_off=[0, 1, 2]), dict(taken=torch.zeros(4, dtype=torch.int32), taken_off=buf.view(torch.int64)[30:33])):
        with pytest.raises(ValueError, match="out lies"):
            candidates.adjust(s, out=out, **kw)
    wide = torch.zeros(2, 70)
    for kw in (dict(bias=buf[n:n + 32]), dict(bias=out), dict(bias=wide[:, 33:65], out=wide[:, :32]), dict(presence=buf[64:66])):
        with pytest.raises(_lib.DcarlError, match="no CPU path"):         # (past the checks)
            candidates.adjust(s, **{"out": out, **kw})


def test_c_abi_recurrence_beyond_a_launch_is_refused():
    if torch.cuda.is_available():
        pytest.skip("fake addresses: only where nothing can run")
    lib = load_library()
    one, null = C.c_void_p(16), C.c_void_p(None)
    for N, D, t in (((1 << 31) - 2, 17, 3), (1 << 25, 16400, 2)):
        r = C.byref(_lib.CRecurrence(N=N, D=D, E=1, ep_off=16, x=16, ldx=D, gate=16, ldg=1, gate_kind=1, type=t))
        for rc in (lib.dcarl_recurrence_forward(r, null, one, one, null, null), lib.dcarl_recurrence_backward(r, one, one, one, D, null, one, one, null, null)):
            assert rc == -1 and "more than one call takes" in lib.dcarl_last_error().decode()
