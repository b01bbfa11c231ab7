"""The sequence operators on the GPU against their definitions in float64 (oracle/sequence_oracle.py).

Bounds.  u = half a step of the type sums are held in (2^-24 for f32, 2^-53 for f64), uT half a step of the storage type.
* recurrence: every term that reaches h_t passes at most L gates (L: its episode's steps so far), each a product and a sum of relative error <= u,
  and a scan in blocks adds products of the same gates: at most 2 L + 40 roundings on a path (40: the joins of up to ten levels, four each).
  |error| <= (2 L + 40) u M_t with M the recurrence of the magnitudes, + uT |h_t| for the result's rounding.  Gradients: the same for d; a product d h
  has both errors, (4 L + 90) u, and a sum over D channels D more.
* sums of n rows: (n + 10) u times the sum of magnitudes, + uT.  Whole numbers below 2^24 add up exactly, in any order: compared for equality.
* scores: at most six roundings in f32 of values no larger than M, + uT.
Subnormal results of f16 round by at most 2^-25 absolutely."""
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
TYPES = [torch.float64, torch.float32, torch.bfloat16, torch.float16]


def half_step(t):
    return torch.finfo(t).eps / 2


def sum_step(t):
    return 2.0 ** -53 if t == torch.float64 else 2.0 ** -24


def tiny(t):
    return 2.0 ** -25 if t == torch.float16 else 0.0


@pytest.fixture(scope="module")
def dc():
    import dcarl_amd
    dcarl_amd.require_gpu()
    return dcarl_amd


def n64(t):
    return t.detach().double().cpu().numpy()


def ragged(lengths):
    return [0] + list(np.cumsum(lengths))


def inputs(N, D, E, t, kind, seed, h0=True, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(N, D, generator=gen).to(t)
    gate = {"full": torch.sigmoid(3 + 2 * torch.randn(N, D, generator=gen)), "step": torch.sigmoid(3 + 2 * torch.randn(N, generator=gen)) * spread}.get(kind)
    gate = 0.9375 if gate is None else gate.to(t)
    return x, gate, torch.randn(E, D, generator=gen).to(t) if h0 else None, torch.randn(N, D, generator=gen).to(t), torch.randn(E, D, generator=gen).to(t)


def check(got, want, bound, what):
    got, bound = n64(got), np.broadcast_to(bound, np.shape(want))
    off = np.abs(got - want)
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(off / np.maximum(bound, 1e-300)):.2f} times the bound, first at {np.argwhere(bad)[0]}"


def check_recurrence(dc, x, gate, off, h0, dh, dl, reverse, t, use_last=True):
    dev = torch.device("cuda")
    leaf = [v.to(dev).requires_grad_() if isinstance(v, torch.Tensor) else v for v in (x, gate, h0)]
    h, last = dc.episodes.gated_recurrence(leaf[0], leaf[1], torch.tensor(off, device=dev), leaf[2], reverse=reverse, want_last=True)
    (h2,) = (dc.episodes.gated_recurrence(leaf[0].detach(), leaf[1].detach() if isinstance(leaf[1], torch.Tensor) else leaf[1], off,
                                         None if h0 is None else leaf[2].detach(), reverse=reverse),)
    assert torch.equal(h, h2)                                            # with and without a gradient: the same numbers
    wanted = [v for v in leaf if isinstance(v, torch.Tensor)]
    outs, cots = ([h, last], [dh.to(dev), dl.to(dev)]) if use_last else ([h], [dh.to(dev)])
    grads = dict(zip([i for i, v in enumerate(leaf) if isinstance(v, torch.Tensor)], torch.autograd.grad(outs, wanted, cots)))

    N, D = x.shape
    n = off[-1]
    u, uT = sum_step(t), half_step(t)
    L = max([b - a for a, b in zip(off, off[1:])] + [0])
    g = gate if not isinstance(gate, torch.Tensor) else n64(gate).reshape(N, D if gate.dim() == 2 else 1)
    w_h, prev, w_last = so.recurrence(n64(x), g, off, None if h0 is None else n64(h0), reverse)
    m_h, m_prev, m_last = so.recurrence(np.abs(n64(x)), np.abs(g), off, None if h0 is None else np.abs(n64(h0)), reverse)
    path = (2 * L + 40) * u
    check(h, w_h, path * m_h + uT * np.abs(w_h) + tiny(t), "h")
    check(last, w_last, path * m_last + uT * np.abs(w_last) + tiny(t), "last")
    dlast = n64(dl) if use_last else None
    dhz = n64(dh).copy()
    dhz[n:] = 0
    wx, wg, w0 = so.recurrence_gradients(dhz, g, prev, off, dlast, reverse)
    mx, mg, m0 = so.recurrence_gradients(np.abs(dhz), np.abs(g), m_prev, off, None if dlast is None else np.abs(dlast), reverse)
    check(grads[0], wx, path * mx + uT * np.abs(wx) + tiny(t), "dx")
    if 1 in grads:
        more = (4 * L + 90) * u
        if gate.dim() == 1:
            wg, mg, more = wg.sum(1), mg.sum(1), more + D * u
        check(grads[1], wg, more * mg + uT * np.abs(wg) + tiny(t), "dgate")
    if 2 in grads:
        check(grads[2], w0, path * m0 + uT * np.abs(w0) + tiny(t), "dh0")


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("kind", ["full", "step", "number"])
@pytest.mark.parametrize("t", TYPES)
def test_recurrence_types_and_gates(dc, t, kind, reverse):
    off = ragged([5, 0, 1, 70, 0, 0, 33, 128, 1, 1])
    x, gate, h0, dh, dl = inputs(off[-1], 37, len(off) - 1, t, kind, 1)
    check_recurrence(dc, x, gate, off, h0, dh, dl, reverse, t)


@pytest.mark.parametrize("D", [1, 2, 7, 8, 16, 31, 33, 63, 64, 65, 130, 256, 260, 517])
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_recurrence_widths(dc, t, D):
    off = ragged([64, 3, 100, 17, 0, 63])
    x, gate, h0, dh, dl = inputs(off[-1], D, len(off) - 1, t, "full" if D % 2 else "step", D)
    check_recurrence(dc, x, gate, off, h0, dh, dl, D % 3 == 0, t)


@pytest.mark.parametrize("lengths", [[1], [2], [0], [0, 0, 0], [1] * 300, [4097], [700, 1, 2000], [0] * 50 + [9] + [0] * 50, [31, 33] * 20, list(range(60)), [1023, 1025, 511, 513]],
                         ids=lambda v: f"{len(v)}x{max(v)}")
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_recurrence_lengths(dc, t, lengths):
    off = ragged(lengths)
    for D, kind in ((40, "full"), (1, "number"), (3, "step"), (130, "step")):
        x, gate, h0, dh, dl = inputs(off[-1], D, len(lengths), t, kind, len(lengths) + D)
        check_recurrence(dc, x, gate, off, h0, dh, dl, D == 3, t)


def test_recurrence_many_steps_in_parts(dc):
    # long enough that the time axis is cut between workgroups: episodes that cross the cuts, one that spans many, some that end at them
    lengths = [3000, 1, 4096, 96, 0, 9000, 37, 2048, 64, 64, 1500]
    off = ragged(lengths)
    for D, kind, t in ((24, "full", torch.float32), (70, "step", torch.float32), (1, "number", torch.float64), (5, "full", torch.bfloat16)):
        for reverse in (False, True):
            x, gate, h0, dh, dl = inputs(off[-1], D, len(lengths), t, kind, D)
            check_recurrence(dc, x, gate, off, h0, dh, dl, reverse, t)


@pytest.mark.parametrize("D, t", [(1, torch.float32), (1, torch.float64), (1, torch.bfloat16), (3, torch.float32), (20, torch.float32), (18, torch.float64), (70, torch.bfloat16), (130, torch.float16), (9, torch.float32)])
@pytest.mark.parametrize("reverse", [False, True])
def test_recurrence_whole_numbers_across_tiles_are_exact(dc, D, t, reverse):
    """Gates of +1 and -1 and small whole numbers: nothing fades, so what passes between tiles and groups of tiles has to be right, and every sum is a
    whole number that f32 holds, in any order of joining: the results are the definition's, rounded once to the type."""
    gen = torch.Generator().manual_seed(D)
    off = ragged([1, 700, 0, 23000, 130, 2048, 4000])                     # 23000 steps: tens of tiles for every width, more than four groups of them
    N, E = off[-1], len(off) - 1
    x, dh = (torch.randint(-1, 2, (N, D), generator=gen).to(t) for _ in range(2))
    h0, dl = (torch.randint(-3, 4, (E, D), generator=gen).to(t) for _ in range(2))
    for kind in ("full", "step"):
        gate = (torch.randint(0, 2, (N, D) if kind == "full" else (N,), generator=gen) * 2 - 1).to(t)
        leaf = [v.cuda().requires_grad_() for v in (x, gate, h0)]
        h, last = dc.episodes.gated_recurrence(leaf[0], leaf[1], off, leaf[2], reverse=reverse, want_last=True)
        grads = torch.autograd.grad([h, last], leaf, [dh.cuda(), dl.cuda()])
        w_h, prev, w_last = so.recurrence(n64(x), n64(gate).reshape(N, -1), off, n64(h0), reverse)
        wx, wg, w0 = so.recurrence_gradients(n64(dh), n64(gate).reshape(N, -1), prev, off, n64(dl), reverse)
        wg = wg if kind == "full" else wg.sum(1)
        assert max(np.abs(v).max() for v in (w_h, wx, wg)) < 2 ** 24      # (f16 holds 65504: what lies beyond is infinite in both)
        for got, want, what in zip([h, last, *grads], [w_h, w_last, wx, wg, w0], ["h", "last", "dx", "dgate", "dh0"]):
            assert torch.equal(got.detach().cpu(), torch.from_numpy(want).to(t)), (kind, what)


def test_recurrence_side_by_side_on_two_streams(dc):
    """Two long calls at once, each waiting for its own tiles only."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    off = torch.tensor([0, 60000, 60001, 131072], device="cuda")
    args = [(torch.randn(131072, D, device="cuda", generator=gen), torch.rand(131072, D, device="cuda", generator=gen) * 0.1 + 0.899) for D in (192, 5)]
    want = [dc.episodes.gated_recurrence(x, g, off, validate=False) for x, g in args]
    streams = [torch.cuda.Stream() for _ in args]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for k, (x, g) in enumerate(args):
            with torch.cuda.stream(streams[k]):
                got[k].append(dc.episodes.gated_recurrence(x, g, off, validate=False))
    torch.cuda.synchronize()
    assert all(torch.equal(w, a) for w, many in zip(want, got) for a in many)


def test_recurrence_rows_behind_and_no_h0(dc):
    off = [0, 6, 40]
    x, gate, _, dh, dl = inputs(90, 20, 2, torch.float32, "full", 3)
    x[40:], gate[40:], dh[40:] = math.nan, math.inf, math.nan             # padding is not read
    check_recurrence(dc, x, gate, off, None, dh, dl, False, torch.float32, use_last=False)
    check_recurrence(dc, x, gate, off, None, dh, dl, True, torch.float32)
    h = dc.episodes.gated_recurrence(x.cuda(), gate.cuda(), [0])
    assert torch.equal(h, torch.zeros_like(h))                            # no episode at all


def test_recurrence_layouts(dc):
    """Row strides, odd alignment, an expanded row, channels that are not contiguous, a (N,) stream with a stride."""
    N, D, off = 77, 20, [0, 30, 77]
    wide = torch.randn(N, 3 * D + 1, device="cuda", dtype=torch.bfloat16)
    x, gate = wide[:, 1:1 + D], torch.sigmoid(wide[:, D + 2:2 * D + 2].float()).to(torch.bfloat16)
    want = dc.episodes.gated_recurrence(x.contiguous(), gate.contiguous(), off)
    g_wide = torch.zeros(N, D + 3, device="cuda", dtype=torch.bfloat16)
    g_wide[:, 3:] = gate
    assert torch.equal(dc.episodes.gated_recurrence(x, g_wide[:, 3:], off), want)
    assert torch.equal(dc.episodes.gated_recurrence(x.t().contiguous().t(), gate, off), want)
    one = torch.randn(1, D, device="cuda", dtype=torch.bfloat16)
    assert torch.equal(dc.episodes.gated_recurrence(one.expand(N, D), gate, off), dc.episodes.gated_recurrence(one.repeat(N, 1), gate, off))
    s = torch.rand(2 * N, device="cuda")[::2]
    g = torch.rand(3 * N, device="cuda")[::3]
    for reverse in (False, True):
        a = dc.episodes.gated_recurrence(s, g, off, reverse=reverse)
        assert a.shape == (N,) and torch.equal(a, dc.episodes.gated_recurrence(s.contiguous(), g.contiguous(), off, reverse=reverse))
        b = dc.episodes.gated_recurrence(x.float(), g, off, reverse=reverse)
        assert torch.equal(b, dc.episodes.gated_recurrence(x.float(), g.contiguous(), off, reverse=reverse))
    # a gradient with strides of its own (an expanded one)
    leaf = x.float().detach().requires_grad_()
    h = dc.episodes.gated_recurrence(leaf, gate.float(), off)
    ga, = torch.autograd.grad(h.sum(), leaf, retain_graph=True)
    gb, = torch.autograd.grad(h, leaf, torch.ones_like(h))
    assert torch.equal(ga, gb)


def test_recurrence_episodes_do_not_touch(dc):
    """NaN and infinity in one episode's inputs, gates or start reach no other episode, forward or backward."""
    off = ragged([40, 300, 90, 500, 70])
    for D in (1, 12, 200):
        x, gate, h0, dh, dl = (v.cuda() for v in inputs(off[-1], D, 5, torch.float32, "full", 9))

        def both(x, gate, h0, dh):
            leaf = [v.clone().requires_grad_() for v in (x, gate, h0)]
            h = dc.episodes.gated_recurrence(leaf[0], leaf[1], off, leaf[2])
            return (h.detach(), *torch.autograd.grad(h, leaf, dh))
        clean = both(x, gate, h0, dh)
        for bad in (math.nan, math.inf):
            x2, g2, h2, d2 = x.clone(), gate.clone(), h0.clone(), dh.clone()
            x2[100], g2[339], h2[3], d2[600] = bad, bad, bad, bad         # in episodes 1 and 3
            got = both(x2, g2, h2, d2)
            for a, b in zip(clean[:3], got[:3]):
                for e in (0, 2, 4):
                    assert torch.equal(a[off[e]:off[e + 1]], b[off[e]:off[e + 1]])
            assert torch.equal(clean[3][[0, 2, 4]], got[3][[0, 2, 4]])


def test_recurrence_odd_calls(dc):
    off = [0, 3, 5]
    x, g = torch.randn(5, 4, device="cuda", requires_grad=True), torch.rand(5, device="cuda", requires_grad=True)
    h = dc.episodes.gated_recurrence(x, g, off)
    d, = torch.autograd.grad((h * h).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        d.sum().backward()
    h = dc.episodes.gated_recurrence(x, g, off)
    a = torch.autograd.grad(h.sum(), (x, g), retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(a, torch.autograd.grad(h.sum(), (x, g))))        # twice through one graph
    assert torch.equal(a[0], torch.autograd.grad(dc.episodes.gated_recurrence(x, g.detach(), off).sum(), x)[0])
    assert torch.equal(a[1], torch.autograd.grad(dc.episodes.gated_recurrence(x.detach(), g, off).sum(), g)[0])
    h = dc.episodes.gated_recurrence(x, g, off)
    with torch.no_grad():
        g.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        h.sum().backward()
    none = torch.zeros(5, 0, device="cuda")
    leaf = torch.ones(5, device="cuda", requires_grad=True)
    h, last = dc.episodes.gated_recurrence(none, leaf, off, torch.zeros(2, 0, device="cuda"), want_last=True)
    assert h.shape == (5, 0) and last.shape == (2, 0) and not torch.autograd.grad(h.sum() + last.sum(), leaf)[0].any()
    # only the last states are used, and h of steps that nothing depends on
    x2 = torch.randn(5, 4, device="cuda", requires_grad=True)
    _, last = dc.episodes.gated_recurrence(x2, 0.5, off, want_last=True)
    dx, = torch.autograd.grad(last.sum(), x2)
    assert torch.equal(dx[:, 0].cpu(), torch.tensor([0.25, 0.5, 1.0, 0.5, 1.0]))


def test_recurrence_gradcheck(dc):
    off = ragged([3, 0, 5, 1])
    for kind in ("full", "step"):
        x, gate, h0, _, _ = inputs(9, 3, 4, torch.float64, kind, 5)
        leaf = [v.cuda().requires_grad_() for v in (x, gate, h0)]
        for reverse in (False, True):
            assert torch.autograd.gradcheck(lambda a, b, c: dc.episodes.gated_recurrence(a, b, off, c, reverse=reverse, want_last=True), leaf)


def test_recurrence_one_step_at_a_time_is_the_whole(dc):
    """Serving: E live episodes fed a step at a time carry what the whole pass computes."""
    E, T, D = 6, 9, 48
    x, gate = torch.randn(E, T, D, device="cuda"), torch.rand(E, T, D, device="cuda")
    whole, last = dc.episodes.gated_recurrence(x.reshape(-1, D), gate.reshape(-1, D), torch.arange(E + 1) * T, want_last=True)
    one = torch.arange(E + 1, device="cuda")
    s = None
    for k in range(T):
        s = dc.episodes.gated_recurrence(x[:, k], gate[:, k], one, s, validate=False)
        # T steps of two roundings each on either side
        assert (s - whole.view(E, T, D)[:, k]).abs().max() <= 2 * 2 * T * 2.0 ** -24 * float(x.abs().max()) * T
    assert torch.allclose(s, last, rtol=0, atol=4 * T * T * 2.0 ** -24 * float(x.abs().max()))


def test_discounted_returns(dc):
    rng = np.random.default_rng(4)
    lengths = rng.integers(0, 400, 200)
    off = ragged(lengths)
    r = rng.normal(size=off[-1])
    want, _, _ = so.recurrence(r[:, None], 0.95, off, reverse=True)
    m, _, _ = so.recurrence(np.abs(r)[:, None], 0.95, off, reverse=True)
    for t in (torch.float64, torch.float32):
        rt = torch.tensor(r, dtype=t, device="cuda")
        got = dc.episodes.discounted_returns(rt, off, 0.95)
        # 0.95 itself is rounded for f32: one more relative u per gate passed
        bound = (3 * max(lengths) + 40) * sum_step(t) * m + 2 * half_step(t) * m
        check(got.view(-1, 1), want, bound, "returns")
    assert torch.equal(dc.episodes.discounted_returns(r, off, 0.95), dc.episodes.discounted_returns(torch.tensor(r, device="cuda"), off, 0.95))


# ---- rows ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("N, S, D", [(1, 1, 1), (7, 3, 5), (64, 20, 33), (300, 1000, 64), (513, 2, 130), (4097, 70000, 3), (5000, 257, 257), (20000, 3, 8), (9000, 1, 40), (100, 5, 1500)])
def test_lookup_and_gradient(dc, t, N, S, D):
    gen = torch.Generator().manual_seed(N)
    ids = torch.randint(-1, S, (N,), generator=gen)
    if N > 1000:
        ids[torch.rand(N, generator=gen) < 0.4] = S // 2                  # a long run
    table = torch.randn(S, D, generator=gen).to(t)
    dout = torch.randn(N, D, generator=gen).to(t)
    for dtype in (torch.int32, torch.int64):
        leaf = table.cuda().requires_grad_()
        out = dc.tables.lookup(leaf, ids.to(dtype).cuda(), 1.75)
        grad, = torch.autograd.grad(out, leaf, dout.cuda())
        want = so.rows(n64(table), ids.numpy(), 1.75)
        check(out, want, (half_step(t) + sum_step(t)) * np.abs(want) + tiny(t), "rows")
        want, mag, n = so.rows_gradient(n64(dout), ids.numpy(), S, 1.75)
        check(grad, want, (n[:, None] + 10) * sum_step(t) * mag + half_step(t) * np.abs(want) + tiny(t), "gradient")
        assert torch.equal(grad, dc.tables.lookup_gradient(dout.cuda(), ids.to(dtype).cuda(), S, 1.75))
        assert not grad[torch.tensor(n == 0, device="cuda")].any()


@pytest.mark.parametrize("N, S", [(1, 1), (63, 9), (3000, 300000), (4095, 1 << 24), (4096, 4096), (4097, 300), (16384, 300), (16385, 300), (70001, 65536), (200000, 300000), (130000, 17)])
def test_gradient_of_whole_numbers_is_exact(dc, N, S):
    gen = torch.Generator(device="cuda").manual_seed(N)
    ids = torch.randint(-1, S, (N,), generator=gen, device="cuda")
    ids[torch.rand(N, generator=gen, device="cuda") < 0.5] = S - 1
    dout = torch.randint(-8, 9, (N, 6), generator=gen, device="cuda").float()           # sums stay below 2^24: exact in any order
    want = torch.zeros(S + 1, 6, dtype=torch.float64).index_add_(0, torch.where(ids < 0, S, ids).cpu(), dout.double().cpu())[:S]
    assert torch.equal(dc.tables.lookup_gradient(dout, ids, S).cpu().double(), want)


def test_lookup_edges(dc):
    t = torch.randn(5, 6, device="cuda")
    assert dc.tables.lookup(t, torch.zeros(0, dtype=torch.int64)).shape == (0, 6)
    assert dc.tables.lookup(t, torch.zeros(2, 0, 3, dtype=torch.int32)).shape == (2, 0, 3, 6)
    ids = torch.tensor([[0, 4], [-1, 2]])
    assert torch.equal(dc.tables.lookup(t, ids), torch.stack([torch.stack([t[0], t[4]]), torch.stack([t[0] * 0, t[2]])]))
    assert not dc.tables.lookup_gradient(torch.zeros(0, 6, device="cuda"), torch.zeros(0, dtype=torch.int64), 5).any()
    assert dc.tables.lookup_gradient(torch.ones(1, 6, device="cuda"), [-1], 0).shape == (0, 6)
    # without the check, ids outside the table count as -1, far ones included
    far = torch.tensor([5, -2, 1 << 40, -(1 << 40), (1 << 32) + 1, 1], device="cuda")
    out = dc.tables.lookup(t, far, validate=False)
    assert not out[:5].any() and torch.equal(out[5], t[1])
    g = dc.tables.lookup_gradient(torch.ones(6, 6, device="cuda"), far, 5, validate=False)
    assert torch.equal(g.sum(1).cpu(), torch.tensor([0.0, 6, 0, 0, 0]))
    with pytest.raises(IndexError):
        dc.tables.lookup(t, far)
    # table rows at a distance, an unaligned one, an expanded one; a gradient with strides
    wide = torch.randn(5, 13, device="cuda", dtype=torch.float16)
    ids = torch.tensor([4, 1, 1], device="cuda")
    assert torch.equal(dc.tables.lookup(wide[:, 3:12], ids), wide[:, 3:12].contiguous()[ids])
    assert torch.equal(dc.tables.lookup(wide[:1, :9].expand(5, 9), ids), wide[:1, :9].repeat(3, 1))
    assert torch.equal(dc.tables.lookup(wide.t(), ids[1:]), wide.t().contiguous()[ids[1:]])
    d = torch.randn(3, 20, device="cuda")
    assert torch.equal(dc.tables.lookup_gradient(d[:, 5:11], ids, 5), dc.tables.lookup_gradient(d[:, 5:11].contiguous(), ids, 5))
    # NaN and infinity stay in their rows
    d = torch.ones(4, 3, device="cuda")
    d[1], d[2] = math.nan, math.inf
    g = dc.tables.lookup_gradient(d, [0, 1, 2, 3], 5)
    assert torch.equal(g[[0, 3, 4]].sum(1).cpu(), torch.tensor([3.0, 3.0, 0.0])) and g[1].isnan().all() and g[2].isinf().all()


def test_lookup_gradcheck(dc):
    t = torch.randn(4, 3, device="cuda", dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda a: dc.tables.lookup(a, [[3, 0, 3], [1, -1, 3]], 0.7), [t])


# ---- scores --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B, V, H", [(1, 1, 3), (3, 11, 5), (2, 33, 0), (5, 300, 40), (1, 4097, 200), (70, 65, 9), (2, 8200, 64)])
def test_adjust(dc, t, B, V, H):
    gen = torch.Generator().manual_seed(B + V)
    s = (3 * torch.randn(B, V, generator=gen)).to(t)
    lengths = torch.randint(0, 2 * H + 1, (B,), generator=gen)
    off = torch.cat([torch.zeros(1, dtype=torch.int64), lengths.cumsum(0)])
    taken = torch.randint(-1, min(V, 50) + 1, (int(off[-1]),), generator=gen)          # -1 and V or 50: V counts nowhere
    given = lengths.div(3, rounding_mode="floor").to(torch.int32)
    strengths = [1 + torch.rand(B, generator=gen), torch.rand(B, generator=gen), torch.rand(B, generator=gen)]
    mask = torch.rand(B, V, generator=gen) < 0.6
    if B > 1:
        mask[1] = False
    cu = lambda v: v.cuda() if isinstance(v, torch.Tensor) else v      # noqa: E731
    for bias, allowed, dtype in ((None, None, torch.int32), (torch.randn(V, generator=gen), mask[0], torch.int64), (torch.randn(B, V, generator=gen), mask, torch.int32)):
        for strong in (strengths, [1.25, 0.5, 0.25]):
            kw = dict(repetition=strong[0], frequency=strong[1], presence=strong[2])
            got = dc.candidates.adjust(s.cuda(), taken.to(dtype).cuda(), off.cuda(), given=given.cuda(), bias=cu(bias),
                                       allowed=None if allowed is None else dc.candidates.pack_allowed(allowed.cuda()), **{k: cu(v) for k, v in kw.items()})
            want, mag = so.adjust(n64(s), taken.numpy(), off.tolist(), given.numpy(), bias=None if bias is None else n64(bias),
                                  allowed=None if allowed is None else allowed.numpy(), **{k: n64(v) if isinstance(v, torch.Tensor) else v for k, v in kw.items()})
            fin = np.isfinite(want)
            assert (np.isneginf(n64(got)) == ~fin).all()
            check(got[torch.tensor(fin, device="cuda")], want[fin], (6 * 2.0 ** -24 * mag + half_step(t) * np.abs(want) + tiny(t))[fin], "scores")


def test_adjust_edges(dc):
    inf, nan = math.inf, math.nan
    s = torch.tensor([[1.0, -1.0, inf, -inf, nan, 0.0, 5.0]], device="cuda")
    low = torch.finfo(torch.float32).min
    z = dc.candidates.adjust(s, torch.arange(7, device="cuda"), torch.tensor([0, 7], device="cuda"), given=torch.tensor([7], dtype=torch.int32, device="cuda"),
                             repetition=2.0, frequency=9.0, presence=9.0)
    assert z[0, [0, 1, 2, 3, 5, 6]].tolist() == [0.5, -2.0, inf, -inf, 0.0, 2.5] and z[0, 4].isnan()
    z = dc.candidates.adjust(s, allowed=dc.candidates.pack_allowed(torch.tensor([False, True, False, True, False, False, False])).cuda())
    assert z[0].tolist() == [-inf, -1.0, -inf, -inf, -inf, -inf, -inf]      # a NaN that is not allowed is no NaN
    assert dc.candidates.adjust(s, allowed=torch.zeros(1, dtype=torch.int32, device="cuda")).isneginf().all()
    # bias of the type's lowest value and of -inf are ordinary biases
    z = dc.candidates.adjust(torch.zeros(1, 3, device="cuda"), bias=torch.tensor([low, -inf, 1.0], device="cuda"))
    assert z[0].tolist() == [low, -inf, 1.0]
    z = dc.candidates.adjust(torch.zeros(1, 2, device="cuda", dtype=torch.float16), bias=torch.tensor([low, 1.0], device="cuda"))
    assert z[0].tolist() == [-inf, 1.0]                                   # below what f16 holds
    # in place, strided rows; what lies between the rows stays
    wide = torch.randn(3, 50, device="cuda")
    before = wide.clone()
    taken, off = torch.tensor([3, 3, 8], dtype=torch.int32, device="cuda"), torch.tensor([0, 1, 1, 3], device="cuda")
    want = dc.candidates.adjust(wide[:, 5:45], taken, off, frequency=0.5, presence=1.0)
    view = wide[:, 5:45]
    assert dc.candidates.adjust(view, taken, off, frequency=0.5, presence=1.0, out=view).data_ptr() == view.data_ptr()
    assert torch.equal(view, want) and torch.equal(wide[:, :5], before[:, :5]) and torch.equal(wide[:, 45:], before[:, 45:])
    assert torch.equal((want != before[:, 5:45]).nonzero().cpu(), torch.tensor([[0, 3], [2, 3], [2, 8]]))
    # one history entry many times; offsets outside the history are held to it
    many = torch.zeros(100_000, dtype=torch.int64, device="cuda")
    z = dc.candidates.adjust(torch.zeros(1, 2, device="cuda"), many, torch.tensor([-5, 1 << 40], device="cuda"), frequency=0.5)
    assert z[0].tolist() == [-50000.0, 0.0]
    assert dc.candidates.adjust(torch.zeros(0, 5, device="cuda")).shape == (0, 5) and dc.candidates.adjust(torch.zeros(5, 0, device="cuda")).shape == (5, 0)
    # `given` beyond the history and below zero
    z = dc.candidates.adjust(torch.ones(2, 2, device="cuda"), torch.tensor([0, 0], device="cuda"), torch.tensor([0, 1, 2], device="cuda"),
                             given=torch.tensor([9, -9], dtype=torch.int32, device="cuda"), repetition=2.0, presence=0.25)
    assert z.tolist() == [[0.5, 1.0], [0.25, 1.0]]


def test_adjust_many_rows(dc):
    B, V = 70_001, 9                                                      # more rows than one grid axis holds
    s = torch.randn(B, V, device="cuda")
    off = torch.arange(B + 1, device="cuda")
    taken = torch.arange(B, device="cuda") % V
    z = dc.candidates.adjust(s, taken, off, presence=0.5)
    want = s.clone()
    want[torch.arange(B, device="cuda"), taken] -= 0.5
    assert torch.equal(z, want)


# ---- how they are called: twice, on streams, in graphs, on large tensors -----------------------------------------------------
def policy(dc, p, ids, off, taken, taken_off, allowed):
    """State ids -> rows -> memory along each episode -> scores -> what may be answered."""
    x = dc.tables.lookup(p["rows"], ids, 2.0, validate=False)
    g = torch.sigmoid(dc.tables.lookup(p["gates"], ids, validate=False))
    h, last = dc.episodes.gated_recurrence(x, g, off, p["start"], want_last=True, validate=False)
    scores = last @ p["out"]
    z = dc.candidates.adjust(scores.detach(), taken, taken_off, repetition=1.5, frequency=0.25, presence=0.125, allowed=allowed)
    return h, scores, z


def policy_inputs(seed=0, S=40, D=24, V=70):
    gen = torch.Generator().manual_seed(seed)
    off = torch.tensor(ragged([30, 0, 7, 150, 1]))
    ids = torch.randint(-1, S, (int(off[-1]),), generator=gen)
    p = dict(rows=torch.randn(S, D, generator=gen), gates=torch.randn(S, D, generator=gen) + 2, start=torch.randn(5, D, generator=gen), out=torch.randn(D, V, generator=gen))
    taken_off = torch.tensor(ragged([4, 0, 3, 9, 1]))
    taken = torch.randint(0, V, (17,), generator=gen)
    allowed = torch.rand(5, V, generator=gen) < 0.5
    allowed[2] = False
    return p, ids, off, taken, taken_off, allowed


def test_policy_of_all_three(dc):
    p, ids, off, taken, taken_off, allowed = policy_inputs()
    leaf = {k: v.cuda().requires_grad_() for k, v in p.items()}
    h, scores, z = policy(dc, leaf, ids.cuda(), off.cuda(), taken.cuda(), taken_off.cuda(), dc.candidates.pack_allowed(allowed.cuda()))
    w = torch.randn(h.shape, generator=torch.Generator().manual_seed(1)), torch.randn(scores.shape, generator=torch.Generator().manual_seed(2))
    grads = torch.autograd.grad([h, scores], list(leaf.values()), [v.cuda() for v in w])

    ref = {k: v.double().requires_grad_() for k, v in p.items()}
    pad = lambda t: torch.cat([t, torch.zeros_like(t[:1])])      # noqa: E731
    x, g = 2.0 * pad(ref["rows"])[ids], torch.sigmoid(pad(ref["gates"])[ids])
    hs, lasts = [], []
    for e in range(5):
        s = ref["start"][e]
        for i in range(int(off[e]), int(off[e + 1])):
            s = g[i] * s + x[i]
            hs.append(s)
        lasts.append(s)
    h64, s64 = torch.stack(hs), torch.stack(lasts) @ ref["out"]
    want = torch.autograd.grad([h64, s64], list(ref.values()), [v.double() for v in w])
    # f32 throughout, up to 150 gates in a row and sums of up to 24 and of a few hundred terms: 700 roundings of 2^-24, relative to each tensor's largest
    for a, b in zip([h, scores, *grads], [h64, s64, *want]):
        assert (a.double().cpu() - b).abs().max() <= 700 * 2.0 ** -24 * 8 * b.abs().max()
    zz, _ = so.adjust(s64.detach().numpy(), taken.numpy(), taken_off.tolist(), repetition=1.5, frequency=0.25, presence=0.125, allowed=allowed.numpy())
    assert (np.isneginf(n64(z)) == np.isneginf(zz)).all() and np.isneginf(zz[2]).all()
    for e in (0, 1, 3, 4):                                                # the answers: the gap to the runner-up is far above the rounding here
        top = np.sort(zz[e])[::-1]
        assert top[0] - top[1] > 1e-3 and int(z[e].argmax()) == int(np.argmax(zz[e]))


def test_same_call_twice_is_the_same(dc):
    gen = torch.Generator(device="cuda").manual_seed(0)
    off = torch.tensor(ragged([5000, 300, 9000, 1, 40]), device="cuda")
    N, D = int(off[-1]), 96
    x, dh = (torch.randn(N, D, device="cuda", generator=gen).bfloat16() for _ in range(2))
    g = torch.sigmoid(3 + torch.randn(N, device="cuda", generator=gen)).bfloat16()
    ids = torch.randint(-1, 50, (N,), device="cuda", generator=gen)

    def once():
        leaf = [x.clone().requires_grad_(), g.clone().requires_grad_()]
        h = dc.episodes.gated_recurrence(leaf[0], leaf[1], off, validate=False)
        return [h.detach(), *torch.autograd.grad(h, leaf, dh), dc.tables.lookup_gradient(dh, ids, 50, validate=False)]
    first = once()
    for _ in range(3):
        torch.empty(64 << 20, dtype=torch.uint8, device="cuda").fill_(255)             # other contents where workspaces will lie
        assert all(torch.equal(a, b) for a, b in zip(first, once()))


def test_on_a_stream_of_their_own(dc):
    p, ids, off, taken, taken_off, allowed = policy_inputs(3)
    p = {k: v.cuda() for k, v in p.items()}
    args = [v.cuda() for v in (ids, off, taken, taken_off)] + [dc.candidates.pack_allowed(allowed.cuda())]
    want = policy(dc, p, *args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        busy = torch.randn(2000, 2000, device="cuda")
        for _ in range(5):
            busy = busy @ busy
        got = policy(dc, p, *args)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_captured_and_replayed(dc):
    """The whole policy with its gradients in one graph: inputs change in place, every replay is checked against the eager result."""
    p, ids, off, taken, taken_off, allowed = policy_inputs(4)
    static = {k: v.cuda() for k, v in p.items()}
    ids, off, taken, taken_off = (v.cuda() for v in (ids, off, taken, taken_off))
    bits = dc.candidates.pack_allowed(allowed.cuda())
    w = torch.randn(ids.numel(), 24, device="cuda")

    def step():
        x = dc.tables.lookup(static["rows"], ids, 2.0, validate=False)
        g = dc.tables.lookup(static["gates"], ids, 0.1, validate=False)
        leaf = [v.detach().requires_grad_() for v in (x, g, static["start"])]
        h = dc.episodes.gated_recurrence(leaf[0], leaf[1], off, leaf[2], validate=False)
        dx, dg, d0 = torch.autograd.grad(h, leaf, w)
        drows = dc.tables.lookup_gradient(dx, ids, 40, 2.0, validate=False)
        z = dc.candidates.adjust(h.detach()[:5], taken, taken_off, frequency=0.5, allowed=None)
        return h.detach(), dg, d0, drows, z
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):                                                    # two graphs of the same operators live side by side
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for k in range(4):
        for v in (static["rows"], static["gates"], static["start"], w):
            v.normal_()
        ids.copy_(torch.randint(-1, 40, ids.shape, device="cuda"))
        off[1:5] = torch.randint(0, ids.numel(), (4,), device="cuda").sort().values    # other episodes of the same number
        for graph, _ in graphs:
            graph.replay()
        want = step()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want)), k
    with pytest.raises(ValueError, match="captured"):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            static["rows"].mul(1.0)
            dc.tables.lookup(static["rows"], ids)
    torch.cuda.synchronize()
    assert bits.shape == (5, 3)
    leaf = static["rows"].detach().requires_grad_()
    eager = dc.episodes.gated_recurrence(leaf, 0.5, torch.tensor([0, 40], device="cuda"), validate=False)
    grad = torch.ones_like(eager)
    torch.cuda.synchronize()
    with pytest.raises(ValueError, match="outside of the graph"):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            static["rows"].mul(1.0)
            dc.episodes._Recurrence.backward(eager.grad_fn, grad)
    torch.cuda.synchronize()


def test_offsets_beyond_32_bits(dc):
    D = 1024
    S = (1 << 31) // D + 5000                                             # elements of the table pass 2^31
    table = torch.zeros(S, D, dtype=torch.bfloat16, device="cuda")
    table[-3:] = torch.randn(3, D, device="cuda").bfloat16()
    ids = torch.tensor([S - 1, 0, S - 3, S - 2], device="cuda")
    assert torch.equal(dc.tables.lookup(table, ids), table[ids])
    g = dc.tables.lookup_gradient(torch.ones(4, D, device="cuda", dtype=torch.bfloat16), ids, S)
    assert bool((g[ids] == 1).all()) and int((g.view(-1).view(torch.int16) != 0).sum(dtype=torch.int64)) == 4 * D
    del g
    # the same memory as steps: the last episode starts behind element 2^31
    off = torch.tensor([0, S - 300, S], device="cuda")
    h = dc.episodes.gated_recurrence(table, 0.5, off)
    tail = dc.episodes.gated_recurrence(table[-300:].clone(), 0.5, [0, 300])
    assert torch.equal(h[-300:], tail) and not h[:1000].any()
    del h
    # one row of gradients gathered from behind 2^31
    ids = torch.full((S,), -1, dtype=torch.int32, device="cuda")
    ids[-3:] = 1
    g = dc.tables.lookup_gradient(table, ids, 2)
    want = table[-3:].float().sum(0)
    assert not g[0].any() and bool(((g[1].float() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -22 * table[-3:].float().abs().sum(0)).all())


def test_scores_beyond_32_bits(dc):
    B, V = 2200, 1_000_003
    s = torch.zeros(B, V, dtype=torch.bfloat16, device="cuda")
    off = torch.zeros(B + 1, dtype=torch.int64, device="cuda")
    off[-1] = 2
    z = dc.candidates.adjust(s, torch.tensor([V - 1, 4], device="cuda"), off, presence=1.0, out=s)
    assert z[-1, V - 1] == -1 and z[-1, 4] == -1 and int((z[-1] != 0).sum()) == 2 and not z[0].any() and not z[1100].any()


@pytest.mark.parametrize("D", [1, 5, 64])
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_recurrence_gates_above_one_leave_zeros_alone(dc, t, D):
    """The product of the gates overflows long before the first value arrives; nothing is rounded: powers of two alone."""
    lengths = [300, 5000, 70000]
    off = ragged(lengths)
    N = off[-1]
    x, dh = torch.zeros(N, D), torch.zeros(N, D)
    for b, e in zip(off, off[1:]):
        x[e - 4], x[e - 2] = 1.0, 2.0
        dh[b + 1], dh[b + 3] = 1.0, 2.0
    h = torch.zeros(N, D)
    dx = torch.zeros(N, D)
    for b, e in zip(off, off[1:]):
        h[e - 4:e] = torch.tensor([1.0, 4.0, 18.0, 72.0])[:, None]
        dx[b:b + 4] = torch.tensor([132.0, 33.0, 8.0, 2.0])[:, None]
    leaf = [x.to("cuda", t).requires_grad_(), torch.full((N, D), 4.0, device="cuda", dtype=t, requires_grad=True)]
    got = dc.episodes.gated_recurrence(*leaf, off)
    assert torch.equal(got.detach().cpu().float(), h)
    gx, gg = torch.autograd.grad(got, leaf, dh.to("cuda", t))
    assert torch.equal(gx.cpu().float(), dx) and not gg.any()
    back = dc.episodes.gated_recurrence(x.flip(0).to("cuda", t), 4.0, [N - v for v in reversed(off)], reverse=True)
    assert torch.equal(back.cpu().float(), h.flip(0))


def test_adjust_extreme_repetition(dc):
    """r whose inverse overflows f32 or is subnormal: still z / r, of two roundings at most (2^-24 each; results here are normal)."""
    r = torch.tensor([2.0 ** -149, 5 * 2.0 ** -149, 2.0 ** -128, 2.0 ** 126, 3 * 2.0 ** 126, 2.0 ** 125, 1.75 * 2.0 ** 127], dtype=torch.float32)
    z = torch.tensor([2.0 ** -30, 3 * 2.0 ** -30, 7 * 2.0 ** -30, 7.0, 11.0, 13.0, 23.0], dtype=torch.float32).repeat(7, 1)
    z[3:] = z[3:] * 2.0 ** 40
    z[:3, 3:] = 2.0 ** -28
    ids, off = torch.arange(7, device="cuda").repeat(7), torch.arange(8, device="cuda") * 7
    got = dc.candidates.adjust(z.cuda(), ids, off, repetition=r.cuda())
    want = z.double() / r.double()[:, None]
    assert want.min() > 2.0 ** -126 and want.max() < 2.0 ** 127 * 1.9
    check(got, want.numpy(), 2 * 2.0 ** -24 * want.numpy(), "z / r")
    got = dc.candidates.adjust(torch.tensor([[5.0, math.inf, -1.0]], device="cuda"), torch.arange(3, device="cuda"), torch.tensor([0, 3], device="cuda"), repetition=math.inf)
    assert got[0, 0] == 0 and got[0, 1].isnan() and got[0, 2] == -math.inf
    one = dc.candidates.adjust(z[4:5].cuda(), ids[:7], off[:2], repetition=float(r[4]))      # a number for all rows
    check(one, want[4:5].numpy(), 2 * 2.0 ** -24 * want[4:5].numpy(), "z / r")


@pytest.mark.parametrize("scale", [math.inf, math.nan, -0.0])
def test_gradient_rows_without_an_id_are_zero_whatever_the_scale(dc, scale):
    ids = torch.tensor([3, -1, 3, 9], device="cuda")
    grad = dc.tables.lookup_gradient(torch.ones(4, 5, device="cuda"), ids, 300, scale)
    named = torch.zeros(300, dtype=torch.bool, device="cuda")
    named[[3, 9]] = True
    assert not grad[~named].any()
    assert torch.equal(grad[named].cpu(), torch.tensor([[2.0], [1.0]]).expand(2, 5) * scale) or math.isnan(scale) and grad[named].isnan().all()


def test_gradient_of_more_chunks_and_rows_than_one_grid_axis_takes(dc):
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GB")
    N = (1 << 28) + 1000                                                  # chunks of 64 ids
    ids = torch.arange(N, device="cuda", dtype=torch.int32) % 3
    dout = torch.zeros(N, 1, device="cuda", dtype=torch.float16)
    places = torch.cat([torch.randint(0, N, (900,), generator=torch.Generator().manual_seed(1)), torch.arange(N - 300, N)]).unique()
    dout[places.cuda()] = 1.0
    grad = dc.tables.lookup_gradient(dout, ids, 3, validate=False)
    assert torch.equal(grad.flatten().cpu().long(), torch.bincount(places % 3))
    del ids, dout
    S, D = (1 << 24) + 77, 1032                                           # a workgroup takes four rows of this width
    ids = torch.tensor([0, S - 1, (1 << 24) - 1, 1 << 24, 12345, S - 1], device="cuda")
    dout = torch.arange(6, device="cuda", dtype=torch.float16)[:, None].expand(6, D) + 1
    grad = dc.tables.lookup_gradient(dout, ids, S)
    assert torch.equal(grad[ids].cpu(), torch.tensor([1.0, 8, 3, 4, 5, 8], dtype=torch.float16)[:, None].expand(6, D))
    assert sum(int((grad[a:a + (1 << 21)] != 0).any(1).sum()) for a in range(0, S, 1 << 21)) == 5


@pytest.mark.parametrize("kind", ["full", "step", "number"])
@pytest.mark.parametrize("t, D", [(torch.float64, 1), (torch.float64, 7), (torch.float32, 3), (torch.float32, 65), (torch.bfloat16, 4), (torch.bfloat16, 770), (torch.float16, 2), (torch.float16, 33)])
def test_recurrence_of_about_a_step_each(dc, t, D, kind):
    """Few steps of many episodes: all of them, some, two or three steps, all in one episode; rows behind the last."""
    for i, (lengths, behind) in enumerate((([1], 0), ([1] * 48, 0), ([0, 1, 0, 0, 2, 1, 0], 3), ([2] * 20 + [1, 0], 0), ([0] * 63 + [64], 0), ([100] + [0] * 63 + [28], 0), ([0] * 5, 9), ([1] * 300, 0))):
        off = ragged(lengths)
        x, gate, h0, dh, dl = inputs(off[-1] + behind, D, len(lengths), t, kind, i)
        if behind:
            x[off[-1]:] = math.nan
            dh[off[-1]:] = math.nan
        for reverse in (False, True):
            check_recurrence(dc, x, gate, off, h0 if i != 3 else None, dh, dl, reverse, t)


def test_lookup_and_its_gradient_captured(dc):
    table = torch.randn(70, 40, device="cuda")
    ids = torch.randint(-1, 70, (9000,), device="cuda")
    w = torch.randn(9000, 40, device="cuda")

    def step():
        leaf = table.detach().requires_grad_()
        rows = dc.tables.lookup(leaf, ids, 0.5, validate=False)
        return rows.detach(), torch.autograd.grad(rows, leaf, w)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        table.normal_()
        w.normal_()
        ids.copy_(torch.randint(-1, 70, ids.shape, device="cuda"))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    eager = dc.tables.lookup(table.detach().requires_grad_(), ids, validate=False)
    torch.cuda.synchronize()
    with pytest.raises(ValueError, match="outside of the graph"):
        other = torch.cuda.CUDAGraph()
        with torch.cuda.graph(other):
            table.mul(1.0)
            dc.tables._Lookup.backward(eager.grad_fn, w)
    torch.cuda.synchronize()


def test_steps_of_live_episodes_captured(dc):
    """Serving: a row per live episode, a step of each, scores and what may be answered, in one graph that keeps its states in place."""
    E, S, D, V = 30, 50, 24, 70
    gen = torch.Generator().manual_seed(2)
    table, out = torch.randn(S, D, generator=gen).cuda(), torch.randn(D, V, generator=gen).cuda()
    ids, taken = torch.zeros(E, dtype=torch.int64, device="cuda"), torch.zeros(E, dtype=torch.int64, device="cuda")
    one = torch.arange(E + 1, device="cuda")
    gate = torch.rand(E, D, generator=gen).cuda()
    state = torch.zeros(E, D, device="cuda")
    z = torch.zeros(E, V, device="cuda")

    def step(state):
        h = dc.episodes.gated_recurrence(dc.tables.lookup(table, ids, validate=False), gate, one, state, validate=False)
        dc.candidates.adjust(h @ out, taken, one, presence=0.5, out=z)
        return h
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(state)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        state.copy_(step(state))
    state.zero_()
    want = torch.zeros_like(state)
    for _ in range(5):
        ids.copy_(torch.randint(-1, S, (E,), generator=gen))
        taken.copy_(torch.randint(0, V, (E,), generator=gen))
        graph.replay()
        got = z.clone()
        want = step(want)
        torch.cuda.synchronize()
        assert torch.equal(state, want) and torch.equal(got, z)
