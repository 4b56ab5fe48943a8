"""Decay attention on the GPU against the 64-bit reference (tests/decay_reference.py).

Every result is a sum of products of inputs, so the same reference on the inputs' magnitudes gives M, the sum of the terms'
magnitudes, and an error is bounded entry by entry:
  * a result of type t is rounded once at the end: half a step, eps(t) / 2 * |value|;
  * float32 sums of K terms in any order: K 2^-24 M.  An entry passes through a sum over Dk or Dv (<= 128), one over the rows of
    a sequence (T) and a few roundings of weights and products (32, weights g^e by exp2 of a rounded exponent among them);
  * bfloat16 inputs: scores and states enter a product as the sum of two bfloat16 terms at least, 2^-17 of each, twice in a
    chain: 2^-16 M; results in float32 carry three terms, 2^-24 each, which the 32 above holds;
  * weights below 2^-126 may be zero: each takes at most 2^-126 times four inputs (below 2^3 each) from at most 2^7 x 2^9 terms: 2^-98.
"""
import pytest
import torch

import decay_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    return torch.device("cuda:0")


def _inputs(seed, lead, n, H, Hq, Hk, Hv, Dk, Dv, dtype, state, decay=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = dict(q=r(*lead, Hq, Dk).to(dtype), k=r(*lead, Hk, Dk).to(dtype), v=r(*lead, Hv, Dv).to(dtype),
             log_decay=-torch.exp(torch.rand(H, generator=g) * 7 - 6) if decay is None else torch.tensor(decay, dtype=F32))
    x["grad_o"] = r(*lead, H, Dv).to(dtype)
    x["state"], x["grad_state"] = (r(n, H, Dk, Dv), r(n, H, Dk, Dv)) if state else (None, None)
    return x


def _close(name, got, want, size, T, D):
    """got within the bound of the module's docstring of want, size: the same from the inputs' magnitudes."""
    assert got.shape == want.shape, (name, got.shape, want.shape)
    got, want, size = got.cpu(), want.detach(), size.detach()
    assert torch.isfinite(got.float()).all(), name
    room = 2.0 ** -98 + (T + D + 32) * 2.0 ** -24 * size + (2.0 ** -8 * want.abs() + 2.0 ** -16 * size if got.dtype == BF16 else 2.0 ** -24 * want.abs())
    off = (got.double() - want).abs()
    worst = ((off - room).max() if off.numel() else torch.tensor(-1.0)).item()
    assert worst <= 0, f"{name}: {off.max().item():.3g} off, {worst:.3g} more than the bound"


def _check(x, dev, offsets=None, longest=None, scale=None):
    from timediff_amd.decay_attention import decay_attention
    T = longest if longest is not None else x["q"].shape[1]
    D = max(x["q"].shape[-1], x["v"].shape[-1])
    kw = dict(scale=scale, offsets=offsets)
    size = {n: None if t is None else t.abs() if n != "log_decay" else t for n, t in x.items()}
    want, big = (ref.decay_attention(y["q"], y["k"], y["v"], y["log_decay"], state=y["state"], **kw) for y in (x, size))
    dwant, dbig = (ref.gradients(y["q"], y["k"], y["v"], y["log_decay"], y["grad_o"], y["grad_state"], state=y["state"], **kw) for y in (x, size))
    names = ["q", "k", "v", "log_decay"] + (["state"] if x["state"] is not None else [])
    leaf = {n: x[n].to(dev).requires_grad_() for n in names}
    got = decay_attention(leaf["q"], leaf["k"], leaf["v"], leaf["log_decay"], scale=scale, offsets=None if offsets is None else offsets.to(dev),
                          initial_state=leaf.get("state"), return_state=True)
    outs, grads = ([got[0], got[1]], [x["grad_o"].to(dev), x["grad_state"].to(dev)]) if x["state"] is not None else ([got[0]], [x["grad_o"].to(dev)])
    d = dict(zip(names, torch.autograd.grad(outs, [leaf[n] for n in names], grads)))
    assert got[0].dtype == x["q"].dtype and got[1].dtype == F32
    _close("o", got[0], want[0], big[0], T, D)
    _close("state", got[1], want[1], big[1], T, D)
    for n in names:
        assert d[n].dtype == leaf[n].dtype
        _close("grad " + n, d[n], dwant[n], dbig[n], T * (x["q"].shape[0] if n == "log_decay" else 1) + 2 * T, D)
    return got, d


SHAPES = [  # B, T, H, Hq, Hk, Hv, Dk, Dv, state
    (1, 1, 1, 1, 1, 1, 1, 1, True), (3, 1, 2, 2, 2, 2, 16, 16, False), (2, 0, 2, 2, 2, 2, 8, 8, True), (2, 2, 3, 3, 3, 3, 5, 7, True),
    (2, 63, 2, 2, 2, 2, 64, 64, False), (2, 64, 2, 2, 2, 2, 64, 64, True), (2, 65, 2, 2, 2, 2, 64, 64, True), (1, 272, 4, 4, 4, 4, 64, 64, False),
    (2, 24, 4, 4, 4, 4, 23, 23, True), (1, 129, 4, 2, 1, 4, 32, 48, True), (1, 200, 6, 3, 2, 1, 128, 128, True), (1, 100, 2, 1, 1, 1, 128, 24, True),
    (1, 100, 2, 2, 2, 1, 33, 127, False), (1, 513, 1, 1, 1, 1, 80, 96, True)]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=["-".join(map(str, s)) for s in SHAPES])
def test_sequences(shape, dtype, dev):
    B, T, H, Hq, Hk, Hv, Dk, Dv, state = shape
    _check(_inputs(T + Dk, (B, T), B, H, Hq, Hk, Hv, Dk, Dv, dtype, state), dev)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("lengths, before, behind", [((0, 5, 0, 70, 1, 0), 0, 0), ((130, 3), 0, 9), ((64, 64, 0), 4, 2), ((0,), 0, 3), ((300, 1, 33), 0, 0)])
def test_packed(lengths, before, behind, dtype, dev):
    """Empty sequences, rows before the first and behind the last: those come back as zeros and take no gradient."""
    off = torch.tensor([before + sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32)
    rows = before + sum(lengths) + behind
    x = _inputs(rows, (rows,), len(lengths), 4, 2, 4, 1, 24, 40, dtype, True)
    for n in ("q", "k", "v", "grad_o"):      # what stands in rows of no sequence is not read
        x[n][:before], x[n][before + sum(lengths):] = float("nan"), float("inf")
    clean = {n: t if t is None else torch.where(torch.isfinite(t), t, torch.zeros_like(t)) for n, t in x.items()}
    from timediff_amd.decay_attention import decay_attention
    got, d = _check(clean, dev, offsets=off, longest=max(lengths) * len(lengths))
    leaf = {n: x[n].to(dev).requires_grad_() for n in ("q", "k", "v", "log_decay", "state")}
    o, s = decay_attention(leaf["q"], leaf["k"], leaf["v"], leaf["log_decay"], offsets=off.to(dev), initial_state=leaf["state"], return_state=True)
    again = torch.autograd.grad([o, s], list(leaf.values()), [x["grad_o"].to(dev), x["grad_state"].to(dev)])
    assert torch.equal(o, got[0]) and torch.equal(s, got[1])
    for (n, g) in zip(leaf, again):
        assert torch.equal(g, d[n]), n
        if n in "qkv":
            assert (g[:before] == 0).all() and (g[before + sum(lengths):] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("decay", [(0.0, -1e-4), (-20.0, -200.0), (-0.7, -3e38), (0.01, -0.05)], ids=["none", "fast", "lowest", "growing"])
def test_decays(decay, dtype, dev):
    """No decay, one that forgets within a row, the type's lowest value, one that grows."""
    _check(_inputs(11, (2, 150), 2, 2, 2, 2, 2, 32, 16, dtype, True, decay), dev)


def test_no_memory(dev):
    """log_decay = -inf: o_t = scale (q_t . k_t) v_t, and an entering state is forgotten."""
    from timediff_amd.decay_attention import decay_attention, decay_attention_step
    x = _inputs(5, (2, 70), 2, 2, 2, 2, 2, 16, 16, F32, True, (float("-inf"), float("-inf")))
    o, s = decay_attention(*(x[n].to(dev) for n in ("q", "k", "v", "log_decay")), initial_state=x["state"].to(dev), return_state=True)
    q, k, v = (x[n].double() for n in "qkv")
    _close("o", o, 0.25 * (q * k).sum(-1, keepdim=True) * v, 0.25 * (q * k).abs().sum(-1, keepdim=True) * v.abs(), 70, 16)
    _close("state", s, k[:, -1, :, :, None] * v[:, -1, :, None, :], (k[:, -1, :, :, None] * v[:, -1, :, None, :]).abs(), 70, 16)
    st = x["state"].to(dev)
    decay_attention_step(*(x[n][:, 0].to(dev) for n in "qkv"), x["log_decay"].to(dev), st)
    assert torch.isfinite(st).all()


def _strided(t, dev, how):
    """The same values behind other strides: a slice of a wider tensor, rows before sequences, or an odd alignment."""
    t = t.to(dev)
    if how == "slice":
        w = torch.full((*t.shape[:-1], t.shape[-1] + 9), float("nan"), dtype=t.dtype, device=dev)
        w[..., 3:3 + t.shape[-1]] = t
        return w[..., 3:3 + t.shape[-1]]
    if how == "time first":
        return t.transpose(0, 1).contiguous().transpose(0, 1)
    if how == "heads first":
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    return t.transpose(-1, -2).contiguous().transpose(-1, -2)      # last dimension not contiguous: copied


@pytest.mark.parametrize("how", ["slice", "time first", "heads first", "columns"])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_strides(how, dtype, dev):
    from timediff_amd.decay_attention import decay_attention
    x = _inputs(7, (3, 70), 3, 2, 2, 1, 2, 32, 64, dtype, False)
    res = []
    for f in (lambda t: t.to(dev), lambda t: _strided(t, dev, how)):
        leaf = [f(x[n]).detach().requires_grad_() for n in "qkv"] + [x["log_decay"].to(dev).requires_grad_()]
        o = decay_attention(*leaf)
        res.append([o, *torch.autograd.grad(o, leaf, f(x["grad_o"]))])
    for a, b in zip(*res):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("B, H, Hq, Hk, Hv, Dk, Dv", [(1, 1, 1, 1, 1, 1, 1), (3, 4, 2, 1, 4, 23, 23), (17, 2, 2, 2, 2, 64, 64), (2, 8, 2, 2, 8, 128, 128),
                                                      (5, 3, 3, 3, 1, 100, 33)])
def test_step(B, H, Hq, Hk, Hv, Dk, Dv, dtype, dev):
    """Against one row of the reference, from strided inputs; the state is updated where it is."""
    from timediff_amd.decay_attention import decay_attention_step
    x = _inputs(B + Dk, (B, 1), B, H, Hq, Hk, Hv, Dk, Dv, dtype, True)
    want, big = (ref.decay_attention(*(f(x[n]) for n in "qkv"), x["log_decay"], state=f(x["state"])) for f in (lambda t: t, torch.abs))
    state = x["state"].to(dev)
    o = decay_attention_step(*(_strided(x[n], dev, "slice")[:, 0] for n in "qkv"), x["log_decay"].to(dev), state)
    _close("o", o, want[0][:, 0], big[0][:, 0], 1, Dk)
    _close("state", state, want[1], big[1], 1, Dk)


def test_prompt_then_steps(dev):
    """The state that the sequence form leaves, continued row by row, is the longer sequence."""
    from timediff_amd.decay_attention import decay_attention, decay_attention_step
    x = _inputs(23, (2, 90), 2, 4, 2, 2, 4, 64, 32, BF16, False)
    want, big = (ref.decay_attention(f(x["q"]), f(x["k"]), f(x["v"]), x["log_decay"]) for f in (lambda t: t, torch.abs))
    q, k, v, ld = (x[n].to(dev) for n in ("q", "k", "v", "log_decay"))
    o, s = decay_attention(q[:, :77], k[:, :77], v[:, :77], ld, return_state=True)
    rows = [o] + [decay_attention_step(q[:, t], k[:, t], v[:, t], ld, s)[:, None] for t in range(77, 90)]
    _close("o", torch.cat(rows, 1), want[0], big[0], 90, 64)
    _close("state", s, want[1], big[1], 90, 64)


def test_gradient_against_differences(dev):
    """o is linear in each of q, k, v and the entering state: sum((o(x + d) - o(x)) grad_o) = sum(grad_x d) up to rounding, K 2^-24 of
    the sum of magnitudes on each side (twice).  For log_decay the central difference is off by h^2 / 6 times the third derivative,
    at most T^3 times the sum of magnitudes (weights d^3 g^d)."""
    from timediff_amd.decay_attention import decay_attention
    T = 12
    x = _inputs(31, (2, T), 2, 2, 1, 2, 1, 16, 8, F32, True)
    names = ["q", "k", "v", "log_decay", "state"]
    leaf = {n: x[n].to(dev).requires_grad_() for n in names}
    go, gs = x["grad_o"].to(dev).double(), x["grad_state"].to(dev).double()

    def loss(a):
        o, s = decay_attention(a["q"], a["k"], a["v"], a["log_decay"], initial_state=a["state"], return_state=True)
        return (o.double() * go).sum() + (s.double() * gs).sum(), o, s
    _, o, s = loss(leaf)
    d = dict(zip(names, torch.autograd.grad([o, s], list(leaf.values()), [go.float(), gs.float()])))
    plain = {n: t.detach() for n, t in leaf.items()}
    bo, bs = ref.decay_attention(*(x[n].abs() for n in "qkv"), x["log_decay"], state=x["state"].abs())
    M = ((bo * x["grad_o"].abs()).sum() + (bs * x["grad_state"].abs()).sum()).item()
    g = torch.Generator().manual_seed(9)
    for n in names:
        way = torch.randn(x[n].shape, generator=g).to(dev).clamp(-1, 1)
        room = 8 * (T + 16 + 32) * 2.0 ** -24 * M * 4
        if n == "log_decay":
            h = 1e-2
            up, down = (loss(dict(plain, log_decay=plain[n] + a * h * way))[0] for a in (1, -1))
            diff, room = (up - down) / (2 * h), room / h + h * h / 6 * T ** 3 * M * 1.2
        else:
            diff = loss(dict(plain, **{n: plain[n] + way}))[0] - loss(plain)[0]
        assert abs((diff - (d[n].double() * way).sum()).item()) <= room, n


def test_only_wanted_gradients(dev):
    from timediff_amd.decay_attention import decay_attention
    x = _inputs(2, (2, 40), 2, 2, 2, 2, 2, 16, 16, F32, True)
    full = {n: x[n].to(dev).requires_grad_() for n in ("q", "k", "v", "log_decay", "state")}
    def run(leaf):
        return decay_attention(leaf["q"], leaf["k"], leaf["v"], leaf["log_decay"], initial_state=leaf["state"], return_state=True)
    want = dict(zip(full, torch.autograd.grad(run(full)[0].sum(), list(full.values()))))
    for n in full:
        one = {m: t.detach().requires_grad_(m == n) for m, t in full.items()}
        assert torch.equal(torch.autograd.grad(run(one)[0].sum(), one[n])[0], want[n]), n
    # a loss of the state alone
    only = {m: t.detach().requires_grad_() for m, t in full.items()}
    g = torch.autograd.grad(run(only)[1].sum(), [only["k"], only["v"], only["q"], only["state"]])
    big = ref.gradients(*(x[n] for n in ("q", "k", "v", "log_decay")), torch.zeros(2, 40, 2, 16), torch.ones(2, 2, 16, 16), state=x["state"])
    for got, n in zip(g, ("k", "v", "q", "state")):
        assert torch.allclose(got.cpu().double(), big[n], rtol=1e-4, atol=1e-4), n


def test_repeatable_and_streams(dev):
    """The same bits twice, on another stream than the inputs', and with two calls at once."""
    from timediff_amd.decay_attention import decay_attention
    x = _inputs(13, (4, 300), 4, 4, 2, 2, 4, 64, 64, BF16, False)
    def both():
        leaf = [x[n].to(dev).requires_grad_() for n in ("q", "k", "v", "log_decay")]
        o = decay_attention(*leaf)
        return [o, *torch.autograd.grad(o, leaf, x["grad_o"].to(dev))]
    want = both()
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for s in side:
        with torch.cuda.stream(s):
            got.append(both())
    torch.cuda.synchronize()
    for res in got:
        for a, b in zip(res, want):
            assert torch.equal(a, b)


def test_captured(dev):
    """Forward, backward and single rows in one graph, replayed with other inputs and other offsets; eager work between."""
    from timediff_amd.decay_attention import decay_attention, decay_attention_step
    n, rows = 3, 200
    def fresh(seed, cuts):
        x = _inputs(seed, (rows,), n, 2, 1, 2, 2, 32, 32, BF16, True)
        x["offsets"] = torch.tensor(cuts, dtype=torch.int32)
        return {k: t.to(dev) for k, t in x.items()}
    def work(x, state):
        leaf = {k: x[k].detach().requires_grad_() for k in ("q", "k", "v", "log_decay", "state")}
        o, s = decay_attention(leaf["q"], leaf["k"], leaf["v"], leaf["log_decay"], offsets=x["offsets"], initial_state=leaf["state"], return_state=True)
        d = torch.autograd.grad([o, s], list(leaf.values()), [x["grad_o"], x["grad_state"]])
        with torch.no_grad():
            y = decay_attention_step(x["q"][:n], x["k"][:n], x["v"][:n], x["log_decay"], state)
        return [o.detach(), s.detach(), *d, y, state]
    hold = fresh(1, [0, 50, 50, 190])
    state = hold["state"].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(hold, state)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work(hold, state)
    for seed, cuts in ((2, [0, 70, 130, 200]), (3, [0, 0, 199, 199]), (4, [5, 60, 61, 180])):
        x = fresh(seed, cuts)
        for k in hold:
            hold[k].copy_(x[k])
        state.copy_(x["state"])
        want = work(x, x["state"].clone())
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_long_offsets(dev):
    """Rows whose element offsets pass 32 bits: a view of a wide tensor, against the same rows side by side."""
    from timediff_amd.decay_attention import decay_attention
    T, wide = 70, 2 ** 25 + 64
    g = torch.Generator(device=dev).manual_seed(1)
    big = torch.zeros(T, wide, dtype=BF16, device=dev)       # 4.4 GiB
    small = torch.randn(T, 96, generator=g, device=dev).to(BF16)
    big[:, -96:] = small
    def cut(t):
        return [x.unflatten(-1, (1, 32))[None] for x in t[:, -96:].split(32, -1)]
    ld = torch.tensor([-0.05], device=dev)
    assert torch.equal(decay_attention(*cut(big), ld), decay_attention(*cut(small.contiguous()), ld))


def test_empty_batch(dev):
    from timediff_amd.decay_attention import decay_attention, decay_attention_step
    e = lambda *s: torch.zeros(*s, device=dev, requires_grad=True)  # noqa: E731
    q, k, v, ld, s0 = e(0, 5, 2, 8), e(0, 5, 2, 8), e(0, 5, 2, 4), e(2), e(0, 2, 8, 4)
    o, s = decay_attention(q, k, v, ld, initial_state=s0, return_state=True)
    assert o.shape == (0, 5, 2, 4) and s.shape == (0, 2, 8, 4)
    d = torch.autograd.grad(o.sum() + s.sum(), [q, ld, s0])
    assert d[0].shape == q.shape and (d[1] == 0).all()
    with torch.no_grad():
        assert decay_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s0).shape == (0, 2, 4)


@pytest.mark.parametrize("packed", [False, True], ids=["dense", "packed"])
def test_long_rows_of_many_heads(packed, dev):
    """Enough heads for the chip and more than 4096 rows: the backward pass alone is cut into segments.  An entry is a sum over its
    own head, so three heads are held against the reference."""
    from timediff_amd.decay_attention import decay_attention
    T, H, D, pick = 4400, 640, 4, [0, 3, 639]
    cuts = [0, 4300, T] if packed else None
    x = _inputs(41, (T,) if packed else (1, T), 2 if packed else 1, H, H, H, H, D, D, BF16, True)
    off = torch.tensor(cuts, dtype=torch.int32) if packed else None
    names = ("q", "k", "v", "log_decay", "state")
    leaf = {n: x[n].to(dev).requires_grad_() for n in names}
    o, s = decay_attention(*(leaf[n] for n in names[:4]), offsets=None if off is None else off.to(dev), initial_state=leaf["state"], return_state=True)
    d = dict(zip(names, torch.autograd.grad([o, s], [leaf[n] for n in names], [x["grad_o"].to(dev), x["grad_state"].to(dev)])))
    few = lambda n, t: t[pick] if n == "log_decay" else t[:, pick] if "state" in n else t[..., pick, :]  # noqa: E731
    y = {n: few(n, t) for n, t in x.items()}
    size = {n: t.abs() if n != "log_decay" else t for n, t in y.items()}
    want, big = (ref.gradients(z["q"], z["k"], z["v"], z["log_decay"], z["grad_o"], z["grad_state"], state=z["state"], offsets=off) for z in (y, size))
    for n in names:
        _close("grad " + n, few(n, d[n]), want[n], big[n], 3 * T, D)


def test_written_state_is_noticed(dev):
    """A state that a graph saved and a step then changed: the backward pass is refused, as for torch's own writes in place."""
    from timediff_amd.decay_attention import decay_attention, decay_attention_step
    x = {n: None if t is None else t.to(dev) for n, t in _inputs(3, (2, 9), 2, 2, 2, 2, 2, 8, 8, F32, True).items()}
    o = decay_attention(x["q"].requires_grad_(), x["k"], x["v"], x["log_decay"], initial_state=x["state"])
    with torch.no_grad():
        decay_attention_step(x["q"][:, 0], x["k"][:, 0], x["v"][:, 0], x["log_decay"], x["state"])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()
    with torch.inference_mode():               # no such count there
        state = x["state"].clone()
        decay_attention_step(x["q"][:, 0], x["k"][:, 0], x["v"][:, 0], x["log_decay"], state)


def test_captured_beside_an_eager_graph(dev):
    """While an eager graph of the same leaves lives a capture is refused; once it is gone the same leaves are captured and replayed."""
    from timediff_amd.decay_attention import decay_attention
    x = _inputs(19, (2, 70), 2, 2, 2, 2, 2, 16, 16, F32, False)
    leaf = [x[n].to(dev).requires_grad_() for n in ("q", "k", "v", "log_decay")]
    go = x["grad_o"].to(dev)
    eager = decay_attention(*leaf)
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            decay_attention(*leaf)
    want = torch.autograd.grad(eager, leaf, go)
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(decay_attention(*leaf), leaf, go)
    for _ in range(3):
        for g in got:
            g.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T", [1, 17, 40, 64, 100, 129])
@pytest.mark.parametrize("Dk, Dv", [(64, 128), (128, 48), (41, 101), (101, 41)])
def test_rectangles(Dk, Dv, T, dtype, dev):
    """States wider than high and the other way round, at every number of row tiles that the last rows of a sequence can have."""
    _check(_inputs(T + Dk, (2, T), 2, 2, 1, 2, 2, Dk, Dv, dtype, True), dev)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("B, T, H, D", [(100, 530, 2, 40), (3, 1100, 2, 72), (2, 700, 2, 16)], ids=["whole", "wide cut", "narrow cut"])
def test_cut_or_whole(B, T, H, D, dtype, dev):
    """Sequences long enough to be cut into segments, enough of them to be left whole, and states that are cut differently backward."""
    x = _inputs(T, (B, T), B, H, H, H, H, D, D, dtype, True)
    from timediff_amd.decay_attention import decay_attention
    names = ["q", "k", "v", "log_decay", "state"]
    leaf = {n: x[n].to(dev).requires_grad_() for n in names}
    o, s = decay_attention(*(leaf[n] for n in names[:4]), initial_state=leaf["state"], return_state=True)
    d = dict(zip(names, torch.autograd.grad([o, s], list(leaf.values()), [x["grad_o"].to(dev), x["grad_state"].to(dev)])))
    few = slice(0, 2)             # a sequence's results are its own; log_decay's gradient sums over all of them
    y = {n: t if n == "log_decay" else t[few] for n, t in x.items()}
    size = {n: t.abs() if n != "log_decay" else t for n, t in y.items()}
    want, big = (ref.decay_attention(z["q"], z["k"], z["v"], z["log_decay"], state=z["state"]) for z in (y, size))
    _close("o", o[few], want[0], big[0], T, D)
    _close("state", s[few], want[1], big[1], T, D)
    dwant, dbig = (ref.gradients(z["q"], z["k"], z["v"], z["log_decay"], z["grad_o"], z["grad_state"], state=z["state"]) for z in (y, size))
    for n in names:
        if n != "log_decay" or B == 2:
            _close("grad " + n, d[n] if n == "log_decay" else d[n][few], dwant[n], dbig[n], 3 * T * (B if n == "log_decay" else 1), D)


@pytest.mark.parametrize("B, H, Dk, Dv", [(200, 3, 40, 72), (300, 2, 7, 16), (171, 3, 128, 30), (3, 1, 128, 32), (4, 2, 120, 50), (2, 3, 50, 120)])
def test_step_forms(B, H, Dk, Dv, dev):
    """Few and many states, narrow and wide: every number of threads and of columns of the single row."""
    from timediff_amd.decay_attention import decay_attention_step
    x = _inputs(B + Dk, (B, 1), B, H, H, H, H, Dk, Dv, F32, True)
    want, big = (ref.decay_attention(*(f(x[n]) for n in "qkv"), x["log_decay"], state=f(x["state"])) for f in (lambda t: t, torch.abs))
    state = x["state"].to(dev)
    o = decay_attention_step(*(x[n][:, 0].to(dev) for n in "qkv"), x["log_decay"].to(dev), state)
    _close("o", o, want[0][:, 0], big[0][:, 0], 1, Dk)
    _close("state", state, want[1], big[1], 1, Dk)
