"""What the sequence operators of dcarl_amd are measured on: cases, their inputs, one pass, its floor.

Three operators: the gated linear recurrence along ragged episodes (``episodes.gated_recurrence``, ``episodes.discounted_returns``),
rows of a table by id with the gradient by sorted ids (``tables.lookup``), and the adjustment of candidate scores by what was taken
already, biases and masks (``candidates.adjust``).  ``own`` False: their plain form in elementary torch operations."""
import math

import torch

own = False

TYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one step of every live episode of a policy server: latency
        dict(name="recurrence step", op="recurrence", N=48, E=48, D=1024, type="bf16", gate="full", h0=True, reverse=False, train=False),
        # the value column of a record table: discounted returns of a reward stream, an ordinary collection run
        dict(name="returns", op="returns", N=400_000, E=700, type="f64"),
        # a packed training batch of episodes of different lengths
        dict(name="recurrence packed", op="recurrence", N=16384, E=24, D=1024, type="bf16", gate="full", h0=True, reverse=False, train=True),
        # few very long streams: the time axis is all the parallelism there is
        dict(name="recurrence long", op="recurrence", N=65536, E=2, D=2048, type="bf16", gate="full", h0=False, reverse=False, train=True),
        # a gate per step shared by all channels, reversed, odd sizes
        dict(name="recurrence shared gate", op="recurrence", N=10007, E=9, D=999, type="f32", gate="step", h0=True, reverse=True, train=True),
        # many short episodes, odd width, evaluation only
        dict(name="recurrence short f16", op="recurrence", N=5003, E=130, D=130, type="f16", gate="full", h0=False, reverse=False, train=False),
        # the rows of a handful of states: latency
        dict(name="rows few", op="rows", N=16, S=32000, D=2048, type="bf16", skew=0.0, train=False),
        # a training batch on a table much larger than the batch: most gradient rows are zeros
        dict(name="rows train", op="rows", N=16384, S=50000, D=1024, type="bf16", skew=0.05, train=True),
        # a few states dominate (a vehicle that waits): long runs of one id
        dict(name="rows skewed", op="rows", N=131071, S=8000, D=257, type="f32", skew=0.6, train=True),
        # one answer over a few thousand candidates: latency
        dict(name="scores few", op="scores", B=4, V=20011, type="bf16", history=64, bias="none", mask=True),
        # a serving batch
        dict(name="scores batch", op="scores", B=64, V=128000, type="bf16", history=2000, bias="shared", mask=True),
        # the largest batch, long histories, a bias of every row's own
        dict(name="scores large", op="scores", B=256, V=151643, type="f32", history=8000, bias="rows", mask=True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["recurrence", "recurrence", "returns", "rows", "rows", "scores", "scores"])
    if op == "returns":
        N = _log(rng, 1, 4_000_000)
        return dict(op=op, N=N, E=_log(rng, 1, max(1, N // 50)), type=rng.choice(["f64", "f32"]))
    if op == "recurrence":
        D = _log(rng, 1, 4096)
        N = _log(rng, 1, max(1, min(65536, 65536 * 2048 // (2 * D))))
        return dict(op=op, N=N, E=_log(rng, 1, max(1, N // 8)), D=D, type=rng.choice(["bf16", "bf16", "f16", "f32"]), gate=rng.choice(["full", "full", "step", "number"]),
                    h0=rng.random() < 0.5, reverse=rng.random() < 0.5, train=rng.random() < 0.6)
    if op == "rows":
        D = _log(rng, 1, 4096)
        S = _log(rng, 20, min(200_000, 100_000_000 // D))
        return dict(op=op, N=_log(rng, 1, min(200_000, 50_000_000 // D)), S=S, D=D, type=rng.choice(["bf16", "f16", "f32"]), skew=rng.choice([0.0, 0.05, 0.5]),
                    train=rng.random() < 0.7)
    B, V = _log(rng, 1, 256), _log(rng, 11, 151_000)
    return dict(op=op, B=B, V=V, type=rng.choice(["bf16", "f16", "f32"]), history=_log(rng, 1, 8000), bias=rng.choice(["none", "shared", "rows"]),
                mask=rng.random() < 0.7)


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _offsets(N, E, gen):
    """E episodes of different lengths, some of them empty, that fill N steps; one step each where N == E."""
    if N == E:
        return torch.arange(N + 1)
    cuts = torch.randint(0, N + 1, (E - 1,), generator=gen).sort().values
    return torch.cat([torch.zeros(1, dtype=torch.int64), cuts, torch.full((1,), N, dtype=torch.int64)])


def prepare(case, seed):
    dev = torch.device("cuda")
    gen, cpu = torch.Generator(device=dev).manual_seed(seed), torch.Generator().manual_seed(seed)
    t = TYPES[case["type"]]
    st = dict(case=case)

    def normal(*shape, dtype=t):
        return torch.randn(*shape, device=dev, generator=gen).to(dtype)

    if case["op"] in ("recurrence", "returns"):
        off = _offsets(case["N"], case["E"], cpu)
        length = off[1:] - off[:-1]
        st.update(ep_off=off.to(dev), longest=int(length.max()), held=torch.nonzero(length > 0).flatten().to(dev))
        # rows at which an episode of at least one step begins and ends, which the plain form wants
        st.update(first=st["ep_off"][:-1][st["held"]], last=st["ep_off"][1:][st["held"]] - 1)
    if case["op"] == "returns":
        # step rewards 0.1 sqrt(v), a collision now and then
        r = 0.1 * torch.rand(case["N"], device=dev, generator=gen, dtype=torch.float64).mul(14.0).sqrt()
        r[torch.rand(case["N"], device=dev, generator=gen) < 0.002] = -100.0
        st.update(reward=r.to(t), gamma=0.95)
    elif case["op"] == "recurrence":
        N, D, E = case["N"], case["D"], case["E"]
        st.update(x=normal(N, D), h0=normal(E, D) if case["h0"] else None)
        if case["gate"] == "number":
            st.update(gate=0.97)
        else:  # memories of a few to a few hundred steps
            st.update(gate=torch.sigmoid(3.0 + 1.5 * torch.randn((N, D) if case["gate"] == "full" else (N,), device=dev, generator=gen)).to(t))
        if case["train"]:
            st.update(dh=normal(N, D))
    elif case["op"] == "rows":
        N, S, D = case["N"], case["S"], case["D"]
        ids = torch.randint(0, S, (N,), device=dev, generator=gen)
        u = torch.rand(N, device=dev, generator=gen)
        ids = torch.where(u < case["skew"], S // 3, ids)                       # the state that dominates
        ids = torch.where((u > 0.6) & (u < 0.75), (ids.double() / S).pow(4).mul(S).long(), ids)  # and a long tail
        ids = torch.where(u > 0.99, -1, ids)                                   # dropped visits
        st.update(table=normal(S, D), ids=ids.to(torch.int32) if N % 2 else ids, scale=math.sqrt(D))
        if case["train"]:
            st.update(dout=normal(N, D))
    else:
        B, V, H = case["B"], case["V"], case["history"]
        length = torch.randint(0, 2 * H + 1, (B,), generator=cpu)
        off = torch.cat([torch.zeros(1, dtype=torch.int64), length.cumsum(0)])
        n = int(off[-1])
        taken = torch.rand(n, device=dev, generator=gen).pow(3).mul(V).long().clamp_(0, V - 1)
        st.update(scores=normal(B, V, dtype=torch.float32).mul_(3.0).to(t), taken=taken.to(torch.int32), taken_off=off.to(dev), row=torch.repeat_interleave(torch.arange(B), length).to(dev),
                  given=(length // 3).to(torch.int32).to(dev), repetition=1.0 + 0.5 * torch.rand(B, device=dev, generator=gen),
                  frequency=0.3 * torch.rand(B, device=dev, generator=gen), presence=0.5 * torch.rand(B, device=dev, generator=gen))
        st.update(bias=None if case["bias"] == "none" else normal(*((V,) if case["bias"] == "shared" else (B, V)), dtype=torch.float32))
        allowed = torch.rand(B, V, device=dev, generator=gen) < 0.3 if case["mask"] else None
        if allowed is not None and B > 2:
            allowed[1] = False                                                 # a row whose mask leaves nothing
        st.update(allowed=None if allowed is None else _pack(allowed))
    return st


def _pack(allowed):
    """[B][V] truth values -> [B][ceil(V/32)] int32 words, candidate v in bit v % 32 of word v // 32."""
    B, V = allowed.shape
    bits = torch.nn.functional.pad(allowed, (0, -V % 32)).view(B, -1, 32).to(torch.int64)
    words = (bits << torch.arange(32, device=allowed.device)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


# ---- the plain forms -------------------------------------------------------------------------------------------------
def _scan(x, g, longest):
    """h_t = g_t h_{t-1} + x_t along the first axis by doubling; g is 0 where an episode begins."""
    k = 1
    while k < longest:
        x = torch.cat([x[:k], x[k:] + g[k:] * x[:-k]])
        g = torch.cat([g[:k] * 0, g[k:] * g[:-k]])
        k *= 2
    return x


def _plain_recurrence(st):
    c, t = st["case"], st["x"].dtype
    wide = torch.float64 if t == torch.float64 else torch.float32
    x, g = st["x"].to(wide), st["gate"]
    N = x.shape[0]
    g = torch.full((N, 1), g, dtype=wide, device=x.device) if isinstance(g, float) else g.to(wide).view(N, -1)
    begin, end = st["first"], st["last"]
    if c["reverse"]:
        x, g, begin, end = x.flip(0), g.flip(0), N - 1 - end, N - 1 - begin
    h0 = torch.zeros(c["E"], x.shape[1], dtype=wide, device=x.device) if st["h0"] is None else st["h0"].to(wide)
    before = h0[st["held"]]
    x = x.index_add(0, begin, g[begin] * before)
    h = _scan(x, g.index_fill(0, begin, 0.0), st["longest"])
    out = dict(h=h.flip(0) if c["reverse"] else h)
    if c["train"]:
        dh = st["dh"].to(wide)
        dh = dh.flip(0) if c["reverse"] else dh
        later = torch.cat([g[1:], g[:1] * 0]).index_fill(0, end, 0.0)           # the gate of the step behind
        d = _scan(dh.flip(0), later.flip(0), st["longest"]).flip(0)
        out.update(dx=d.flip(0) if c["reverse"] else d)
        if not isinstance(st["gate"], float):
            prev = torch.cat([h[:1] * 0, h[:-1]]).index_copy(0, begin, before)
            dg = d * prev
            dg = dg if c["gate"] == "full" else dg.sum(1)
            out.update(dgate=dg.flip(0) if c["reverse"] else dg)
        if st["h0"] is not None:
            out.update(dh0=torch.zeros_like(h0).index_copy(0, st["held"], g[begin] * d[begin]))
    return {k: v.to(t) for k, v in out.items()}


def _plain_returns(st):
    wide = st["reward"].to(torch.float64).flip(0)
    N = wide.shape[0]
    g = torch.full((N,), st["gamma"], dtype=torch.float64, device=wide.device).index_fill(0, N - 1 - st["last"], 0.0)
    return _scan(wide, g, st["longest"]).flip(0).to(st["reward"].dtype)


def _plain_rows(st):
    table, ids = st["table"], st["ids"].long()
    kept = (ids >= 0).view(-1, 1)
    at = ids.clamp(min=0)
    out = dict(out=torch.where(kept, table[at].float() * st["scale"], 0.0).to(table.dtype))
    if "dout" in st:
        # the gradient of a row: the sum over the run of its id in sorted order, a difference of running sums in 64 bits
        key, order = ids.sort(stable=True)
        total = st["dout"].double()[order].cumsum(0)
        total = torch.cat([torch.zeros_like(total[:1]), total])
        every = torch.arange(table.shape[0], device=key.device)
        grad = total[torch.searchsorted(key, every, right=True)] - total[torch.searchsorted(key, every)]
        out.update(dtable=(grad * st["scale"]).to(table.dtype))
    return out


def _plain_scores(st):
    s, B, V = st["scores"], st["case"]["B"], st["case"]["V"]
    z = s.float()
    place = st["row"] * V + st["taken"]
    here = torch.arange(place.shape[0], device=z.device) - st["taken_off"][st["row"]]
    chosen = (here >= st["given"][st["row"]]).float()
    seen = torch.zeros(B * V, device=z.device).index_fill_(0, place, 1.0).view(B, V) > 0
    n = torch.zeros(B * V, device=z.device).index_add_(0, place, chosen).view(B, V)
    r = st["repetition"].view(B, 1)
    z = torch.where(seen, torch.where(z > 0, z / r, z * r), z)
    z = z - st["frequency"].view(B, 1) * n - st["presence"].view(B, 1) * (n > 0)
    z = z if st["bias"] is None else z + st["bias"]
    if st["allowed"] is not None:
        bit = torch.arange(V, device=z.device)
        z = torch.where((st["allowed"][:, bit // 32] >> (bit % 32)) & 1 > 0, z, -math.inf)
    return z.to(s.dtype)


def run(st):
    op = st["case"]["op"]
    if not own:
        return {"recurrence": _plain_recurrence, "returns": _plain_returns, "rows": _plain_rows, "scores": _plain_scores}[op](st)
    from dcarl_amd import candidates, episodes, tables
    if op == "returns":
        return episodes.discounted_returns(st["reward"], st["ep_off"], st["gamma"], validate=False)
    if op == "scores":
        return candidates.adjust(st["scores"], st["taken"], st["taken_off"], given=st["given"], repetition=st["repetition"], frequency=st["frequency"],
                                 presence=st["presence"], bias=st["bias"], allowed=st["allowed"])
    if op == "rows":
        if "dout" not in st:
            return dict(out=tables.lookup(st["table"], st["ids"], st["scale"], validate=False))
        table = st["table"].detach().requires_grad_()
        out = tables.lookup(table, st["ids"], st["scale"], validate=False)
        return dict(out=out.detach(), dtable=torch.autograd.grad(out, table, st["dout"])[0])
    if "dh" not in st:
        return dict(h=episodes.gated_recurrence(st["x"], st["gate"], st["ep_off"], st["h0"], reverse=st["case"]["reverse"], validate=False))
    leaf = {k: st[k].detach().requires_grad_() for k in ("x", "gate", "h0") if isinstance(st[k], torch.Tensor)}
    h = episodes.gated_recurrence(leaf["x"], leaf.get("gate", st["gate"]), st["ep_off"], leaf.get("h0"), reverse=st["case"]["reverse"], validate=False)
    grads = torch.autograd.grad(h, list(leaf.values()), st["dh"])
    return dict(zip(["d" + k for k in leaf], grads), h=h.detach())


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------
def _steps(off, reverse):
    """Rows of the t-th step of every episode that has one, with those episodes; the longest first, so that they stay a prefix."""
    length = off[1:] - off[:-1]
    order = length.argsort(descending=True, stable=True)
    n = length[order]
    start = torch.where(torch.tensor(reverse, device=off.device), off[1:][order] - 1, off[:-1][order])
    alive = torch.searchsorted(-n, -torch.arange(int(n[0]) if len(n) else 0, device=off.device), right=False).tolist()
    for t, m in enumerate(alive):
        yield start[:m] + (-t if reverse else t), order[:m], m


def _exact_recurrence(st):
    c, x = st["case"], st["x"].double()
    N, D, E = c["N"], c["D"], c["E"]
    gate = st["gate"]
    g = torch.full((N, 1), gate, dtype=torch.float64, device=x.device) if isinstance(gate, float) else gate.double().view(N, -1)
    h0 = torch.zeros(E, D, dtype=torch.float64, device=x.device) if st["h0"] is None else st["h0"].double()
    h, prev = torch.empty_like(x), torch.empty_like(x) if c["train"] else None
    state = None
    for rows, eps, m in _steps(st["ep_off"], c["reverse"]):
        state = h0[eps] if state is None else state[:m]
        if prev is not None:
            prev[rows] = state
        state = g[rows] * state + x[rows]
        h[rows] = state
    out = dict(h=h)
    if not c["train"]:
        return out
    dh, dx, dg, dh0 = st["dh"].double(), torch.empty_like(x), torch.empty_like(g), torch.zeros_like(h0)
    for rows, eps, m in reversed(list(_steps(st["ep_off"], c["reverse"]))):
        d = dh[rows] + dh0[eps]                                                # dh0 holds what comes back from the step behind
        dx[rows] = d
        dg[rows] = d * prev[rows] if c["gate"] == "full" else (d * prev[rows]).sum(1, keepdim=True)
        dh0[eps] = g[rows] * d
    out.update(dx=dx)
    if not isinstance(gate, float):
        out.update(dgate=dg.view(gate.shape))
    if st["h0"] is not None:
        out.update(dh0=dh0)
    return out


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op in ("recurrence", "returns") and st["longest"] > 100_000:
        return None
    if op == "recurrence":
        return _exact_recurrence(st)
    if op == "returns":
        r = st["reward"].double()
        out = torch.empty_like(r)
        state = None
        for rows, _, m in _steps(st["ep_off"], True):
            state = r[rows] if state is None else r[rows] + st["gamma"] * state[:m]
            out[rows] = state
        return out
    if op == "rows":
        ids, table = st["ids"].long(), st["table"].double()
        padded = torch.cat([table * st["scale"], torch.zeros_like(table[:1])])     # row -1
        out = dict(out=padded[ids])
        if "dout" in st:
            # row by row on the host: many rows of one id are a long queue of atomics on the device
            keep = ids >= 0
            grad = torch.zeros(table.shape, dtype=torch.float64).index_add_(0, ids[keep].cpu(), st["dout"][keep].cpu().double())
            out.update(dtable=grad.to(table.device) * st["scale"])
        return out
    B, V, dev = case["B"], case["V"], st["scores"].device
    z = torch.empty(B, V, dtype=torch.float64, device=dev)
    for b, (lo, hi) in enumerate(zip(st["taken_off"].tolist()[:-1], st["taken_off"].tolist()[1:])):
        ids, given = st["taken"][lo:hi].long(), int(st["given"][b])
        s = st["scores"][b].double()
        all_n, new_n = torch.bincount(ids, minlength=V), torch.bincount(ids[given:], minlength=V)
        r, f, p = (st[k][b].double() for k in ("repetition", "frequency", "presence"))
        s = torch.where(all_n > 0, s * torch.where(s > 0, 1 / r, r), s) - f * new_n - p * (new_n > 0)
        if st["bias"] is not None:
            s = s + (st["bias"] if st["bias"].dim() == 1 else st["bias"][b]).double()
        if st["allowed"] is not None:
            bits = (st["allowed"][b].view(-1, 1) >> torch.arange(32, device=dev)) & 1
            s = s.masked_fill(bits.flatten()[:V] == 0, -math.inf)
        z[b] = s
    return z


def work(case):
    b = torch.finfo(TYPES[case["type"]]).bits // 8
    if case["op"] == "returns":
        return dict(bytes=2 * case["N"] * b + 8 * case["E"], flops=2 * case["N"])
    if case["op"] == "recurrence":
        N, D, E = case["N"], case["D"], case["E"]
        gate = {"full": N * D * b, "step": N * b, "number": 0}[case["gate"]]
        state = E * D * b if case["h0"] else 0
        once = 2 * N * D * b + gate + state + 8 * E
        return dict(bytes=once + (2 * N * D * b + gate + state if case["train"] else 0), flops=(2 + (5 if case["train"] else 0)) * N * D)
    if case["op"] == "rows":
        N, S, D = case["N"], case["S"], case["D"]
        once = (min(N, S) + N) * D * b + 4 * N
        return dict(bytes=once + (N + S) * D * b if case["train"] else once, flops=N * D * (2 if case["train"] else 1))
    B, V = case["B"], case["V"]
    bias = {"none": 0, "shared": 4 * V, "rows": 4 * B * V}[case["bias"]]
    return dict(bytes=2 * B * V * b + bias + (B * V // 8 if case["mask"] else 0) + 4 * B * case["history"], flops=4 * B * V)
