"""What the sequence operators' longer paths compute: the state that passes between groups of tiles for few channels, and long histories of scores.

Whole numbers are exact in any order of joining (compared for equality); scores take at most six roundings in f32 of values no larger than M, + half a step
of the type."""
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


def walk(x, g, before):
    """h_t = g_t h_{t-1} + x_t for gates of +1 and -1: with P the running product of the gates, which is its own inverse, h = P (before + sum of x P)."""
    P = np.cumprod(g, axis=0)
    return P * (before + np.cumsum(x * P, axis=0))


def definition(x, g, off, h0, dh, dl, reverse):
    """h, last, dx, dgate, dh0 in whole numbers of 64 bits, episode by episode."""
    h, dx, dg = np.zeros_like(x), np.zeros_like(x), np.zeros_like(x)
    last, dh0 = h0.copy(), dl.copy()
    for e, (b, z) in enumerate(zip(off, off[1:])):
        if z == b:
            continue
        s = slice(b, z)
        turn = (lambda v: v[::-1]) if reverse else (lambda v: v)
        xe, ge, de = turn(x[s]), np.broadcast_to(turn(g[s]), x[s].shape), turn(dh[s])
        he = walk(xe, ge, h0[e])
        d = walk(de[::-1], np.concatenate([np.ones_like(ge[:1]), ge[:0:-1]]), dl[e])[::-1]
        h[s], dx[s], dg[s] = turn(he), turn(d), turn(d * np.concatenate([h0[e][None], he[:-1]]))
        last[e], dh0[e] = he[-1], ge[0] * d[0]
    return h, last, dx, dg, dh0


def test_the_definition_here_is_the_oracles():
    rng = np.random.default_rng(0)
    off = [0, 4, 4, 5, 30]
    x, dh = rng.integers(-1, 2, (2, 30, 2))
    g, h0, dl = rng.integers(0, 2, (30, 2)) * 2 - 1, *rng.integers(-3, 4, (2, 4, 2))
    for reverse in (False, True):
        h, prev, last = so.recurrence(x.astype(float), g.astype(float), off, h0.astype(float), reverse)
        want = (h, last, *so.recurrence_gradients(dh.astype(float), g.astype(float), prev, off, dl.astype(float), reverse))
        for a, b in zip(definition(x, g, off, h0, dh, dl, reverse), want):
            assert np.array_equal(a, b)


@pytest.mark.parametrize("D, t, tile", [(1, torch.float32, 4096), (1, torch.float64, 2048), (1, torch.bfloat16, 4096), (1, torch.float16, 4096), (2, torch.float16, 512),
                                        (3, torch.float32, 512), (9, torch.float32, 512), (8, torch.float64, 256), (16, torch.bfloat16, 512), (17, torch.bfloat16, 128)])
@pytest.mark.parametrize("reverse", [False, True])
def test_whole_numbers_across_groups_of_tiles(dc, D, t, tile, reverse):
    """Nothing fades under gates of +1 and -1.  One episode spans six groups of sixteen tiles and more, so that a state is handed on past the four groups whose
    maps are joined; one spans two to three groups; others lie in one tile or end at a border."""
    lengths = [1, 700, 0, 99 * tile + 77, 130, 40 * tile, 0, tile, 2048, 4000]
    off = [0] + list(np.cumsum(lengths))
    N, E = off[-1], len(lengths)
    up16 = lambda b: (b + 15) // 16 * 16      # noqa: E731
    # (the tiles are as small as this test takes them to be: a word for each of from, till and the states is in the plan)
    code = {torch.float64: 0, torch.float32: 1, torch.bfloat16: 2, torch.float16: 3}[t]
    words = dc.load_library().dcarl_recurrence_states_bytes(N, D, E, code, 2) - up16(N + 16) - up16(4 * N)
    assert words >= (N // tile) * (8 + D * (8 if code == 0 else 4))
    rng = np.random.default_rng(D)
    x, dh = rng.integers(-1, 2, (2, N, D))
    h0, dl = rng.integers(-3, 4, (2, E, D))
    for kind in ("full", "step"):
        g = rng.integers(0, 2, (N, D) if kind == "full" else (N, 1)) * 2 - 1
        want = list(definition(x, g, off, h0, dh, dl, reverse))
        want[3] = want[3] if kind == "full" else want[3].sum(1)
        assert max(np.abs(v).max() for v in want) < 2 ** 24
        leaf = [torch.from_numpy(v).to("cuda", t).requires_grad_() for v in (x, g if kind == "full" else g[:, 0], h0)]
        h, last = dc.episodes.gated_recurrence(leaf[0], leaf[1], off, leaf[2], reverse=reverse, want_last=True)
        grads = torch.autograd.grad([h, last], leaf, [torch.from_numpy(v).to("cuda", t) for v in (dh, dl)])
        for got, w, what in zip([h, last, *grads], want, ["h", "last", "dx", "dgate", "dh0"]):
            assert torch.equal(got.detach().cpu(), torch.from_numpy(w.astype(np.float64)).to(t)), (kind, what)


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("lengths, behind", [([20011, 9001, 5, 16387], 0), ([8193, 0, 4097], 0), ([1536, 1536, 1536], 0), ([1536, 1536, 1535], 0), ([5003, 0, 1, 77], 0), ([9, 4099], 40_000),
                                             ([12_345], 0), ([8], 1528), ([8], 1527)], ids=lambda v: "-".join(map(str, v)) if isinstance(v, list) else str(v))
def test_adjust_long_histories(dc, t, wide, lengths, behind):
    """On both sides of 1536 entries per row, where the workgroups change size: several tiles of candidates with an odd rest, histories that start at any entry."""
    B, V = len(lengths), 3 * 4096 + 77
    gen = torch.Generator().manual_seed(sum(lengths) + behind)
    s = (3 * torch.randn(B, V, generator=gen)).to(t)
    off = torch.tensor([0] + list(np.cumsum(lengths)))
    n = int(off[-1]) + behind
    taken = (torch.rand(n, generator=gen) ** 3 * (V + 40)).long() - 20          # many times the same few; below 0 and from V on: nowhere
    taken[::97] = V - 1
    taken[1::89] = 4095
    taken[2::83] = 4096
    if wide:
        taken[3::71] += 1 << 32
    given = torch.tensor([v // 3 for v in lengths], dtype=torch.int32)
    mask = torch.rand(B, V, generator=gen) < 0.7
    kw = dict(repetition=1 + torch.rand(B, generator=gen), frequency=torch.rand(B, generator=gen) / 64, presence=torch.rand(B, generator=gen))
    n64 = lambda v: v.double().cpu().numpy()      # noqa: E731
    for bias, allowed in ((torch.randn(B, V, generator=gen), mask), (torch.randn(V, generator=gen), None)):
        got = dc.candidates.adjust(s.cuda(), taken.to(torch.int64 if wide else torch.int32).cuda(), off.cuda(), given=given.cuda(), bias=bias.cuda(),
                                   allowed=None if allowed is None else dc.candidates.pack_allowed(allowed.cuda()), **{k: v.cuda() for k, v in kw.items()})
        want, mag = so.adjust(n64(s), taken.numpy(), off.tolist(), given.numpy(), bias=n64(bias), allowed=None if allowed is None else allowed.numpy(),
                              **{k: n64(v) for k, v in kw.items()})
        fin = np.isfinite(want)
        assert (np.isneginf(n64(got)) == ~fin).all()
        off_by = np.abs(n64(got)[fin] - want[fin])
        bound = (6 * 2.0 ** -24 * mag + torch.finfo(t).eps / 2 * np.abs(want) + (2.0 ** -25 if t == torch.float16 else 0))[fin]
        assert (off_by <= bound).all(), (off_by / bound).max()
