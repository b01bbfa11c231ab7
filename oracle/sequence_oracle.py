"""CPU restatement of the sequence operators in float64 — TEST INFRASTRUCTURE ONLY.

``dcarl_amd.episodes.gated_recurrence``, ``dcarl_amd.tables.lookup`` and ``dcarl_amd.candidates.adjust`` have no counterpart in the reference:
these are their definitions, step by step, with the magnitudes the tests' error bounds are made of."""
import numpy as np


def recurrence(x, gate, ep_off, h0=None, reverse=False):
    """x (N, D), gate (N, D), (N, 1) or a number -> (h (N, D), previous states (N, D), last (E, D))."""
    x = np.asarray(x, dtype=np.float64)
    N, D = x.shape
    E = len(ep_off) - 1
    g = np.broadcast_to(np.asarray(gate, dtype=np.float64), (N, D)) if np.ndim(gate) else np.full((N, D), float(gate))
    h, prev, last = np.zeros((N, D)), np.zeros((N, D)), np.zeros((E, D))
    for e in range(E):
        s = np.zeros(D) if h0 is None else np.array(h0[e], dtype=np.float64)
        steps = range(ep_off[e], ep_off[e + 1])
        for t in (reversed(steps) if reverse else steps):
            prev[t] = s
            s = g[t] * s + x[t]
            h[t] = s
        last[e] = s
    return h, prev, last


def recurrence_gradients(dh, gate, prev, ep_off, dlast=None, reverse=False):
    """-> (dx (N, D), dgate (N, D): per channel, dh0 (E, D))."""
    dh = np.asarray(dh, dtype=np.float64)
    N, D = dh.shape
    E = len(ep_off) - 1
    g = np.broadcast_to(np.asarray(gate, dtype=np.float64), (N, D)) if np.ndim(gate) else np.full((N, D), float(gate))
    dx, dg, dh0 = np.zeros((N, D)), np.zeros((N, D)), np.zeros((E, D))
    for e in range(E):
        c = np.zeros(D) if dlast is None else np.array(dlast[e], dtype=np.float64)
        steps = range(ep_off[e], ep_off[e + 1])
        for t in (steps if reverse else reversed(steps)):
            d = dh[t] + c
            dx[t], dg[t] = d, d * prev[t]
            c = g[t] * d
        dh0[e] = c
    return dx, dg, dh0


def rows(table, ids, scale):
    table, ids = np.asarray(table, dtype=np.float64), np.asarray(ids)
    out = np.zeros((len(ids), table.shape[1]))
    for n, s in enumerate(ids):
        if 0 <= s < len(table):
            out[n] = scale * table[s]
    return out


def rows_gradient(dout, ids, n_rows, scale):
    """-> (gradient, the same sums over magnitudes, terms per row)."""
    dout, ids = np.asarray(dout, dtype=np.float64), np.asarray(ids)
    g, m, n = np.zeros((n_rows, dout.shape[1])), np.zeros((n_rows, dout.shape[1])), np.zeros(n_rows, dtype=np.int64)
    for i, s in enumerate(ids):
        if 0 <= s < n_rows:
            g[s] += dout[i]
            m[s] += np.abs(dout[i])
            n[s] += 1
    return scale * g, abs(scale) * m, n


def adjust(scores, taken=None, taken_off=None, given=None, repetition=1.0, frequency=0.0, presence=0.0, bias=None, allowed=None):
    """-> (adjusted scores, the largest magnitude met on the way).  allowed: truth values (B, V) or (V,)."""
    z = np.array(scores, dtype=np.float64)
    B, V = z.shape
    per_row = lambda v: np.broadcast_to(np.asarray(v, dtype=np.float64), (B,))      # noqa: E731
    r, f, p = per_row(repetition), per_row(frequency), per_row(presence)
    mag = np.abs(z)
    for b in range(B):
        if taken is not None:
            ids = np.asarray(taken[taken_off[b]:taken_off[b + 1]])
            first = int(given[b]) if given is not None else 0
            for v in range(V):
                n_all, n = int((ids == v).sum()), int((ids[first:] == v).sum())
                if n_all:
                    z[b, v] = z[b, v] / r[b] if z[b, v] > 0 else z[b, v] * r[b]
                    mag[b, v] = max(mag[b, v], abs(z[b, v]))
                if n:
                    z[b, v] -= f[b] * n + p[b]
                    mag[b, v] += abs(f[b] * n) + abs(p[b])
    if bias is not None:
        z = z + np.asarray(bias, dtype=np.float64)
        mag = mag + np.abs(np.broadcast_to(np.asarray(bias, dtype=np.float64), z.shape))
    if allowed is not None:
        z = np.where(np.broadcast_to(allowed, z.shape), z, -np.inf)
    return z, mag
