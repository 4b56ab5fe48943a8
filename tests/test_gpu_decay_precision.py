"""How exact decay attention is: bfloat16 results are the float32 results rounded once.

One row of each sequence (many sequences) has a closed form, with x . y the sum over D entries and S, dS the entering state and the
gradient of the state left behind:
    o = c (q . k) v + c g S^T q         dq = c (v . do) k + c g S do         state = g S + k v^T
    dk = c (v . do) q + dS v            dv = c (q . k) do + dS^T k           dstate = g (dS + c q do^T)
Float32 computes each with sums of D products (of bfloat16 values: exact), D roundings of 2^-24 each, and at most 12 more: the
weight g by exp2 (2) of a rounded exponent (|log2 g| <= 1: 2), the scale, a product carried as three bfloat16 terms (2^-24 once, and its
three products added: 3), the products with weight and scale (3), the sum of the two parts (1).  Then one rounding to bfloat16: half
a step at the result."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    return torch.device("cuda:0")


def _half_step(x):
    """Half the distance between bfloat16 neighbours at x (float64 holding bfloat16 values)."""
    return torch.ldexp(torch.ones_like(x), torch.frexp(x).exponent - 9)


@pytest.mark.parametrize("D", [4, 40, 72, 128])
@pytest.mark.parametrize("state", [False, True], ids=["alone", "with a state"])
@pytest.mark.parametrize("slope", [False, True], ids=["fixed decay", "learned decay"])
def test_one_row(D, state, slope, dev):
    from timediff_amd.decay_attention import decay_attention
    B, H, c = 4096 if D == 4 else 512, 2, 0.37
    g = torch.Generator(device=dev).manual_seed(D)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    q, k, v, do = (r(B, 1, H, D).to(BF16) for _ in range(4))
    S, dS = (r(B, H, D, D), r(B, H, D, D)) if state else (None, None)
    ld = torch.tensor([-0.01, -0.6], device=dev)
    leaf = [t.clone().requires_grad_() for t in (q, k, v)] + ([S.clone().requires_grad_()] if state else [])
    o, s = decay_attention(*leaf[:3], ld.clone().requires_grad_(slope), scale=c, initial_state=leaf[3] if state else None, return_state=True)
    d = torch.autograd.grad([o, s] if state else [o], leaf, [do, dS] if state else [do])
    got = dict(zip(("o", "dq", "dk", "dv", "dS"), [o.detach(), *d]))
    c32 = float(torch.tensor(c, dtype=F32))

    def formula(mag):
        f = (lambda t: t.double().abs()) if mag else (lambda t: t.double())  # noqa: E731
        Q, K, V, DO = (f(t)[:, 0] for t in (q, k, v, do))
        w = ld.double().exp()[:, None]
        qk, vo = (Q * K).sum(-1, keepdim=True), (V * DO).sum(-1, keepdim=True)
        res = dict(o=c32 * qk * V, dq=c32 * vo * K, dk=c32 * vo * Q, dv=c32 * qk * DO)
        if state:
            left, right = (lambda M, x: (M * x[..., None, :]).sum(-1)), (lambda M, x: (M * x[..., :, None]).sum(-2))
            E, dE = f(S), f(dS)
            res["o"] = res["o"] + c32 * w * right(E, Q)
            res["dq"] = res["dq"] + c32 * w * left(E, DO)
            res["dk"] = res["dk"] + left(dE, V)
            res["dv"] = res["dv"] + right(dE, K)
            res["dS"] = w[..., None] * (dE + c32 * Q[..., :, None] * DO[..., None, :])
        return res
    want, size = formula(False), formula(True)
    for n, w in want.items():
        x = got[n].double()
        x = x if n == "dS" else x[:, 0]
        room = (D + 12) * 2.0 ** -24 * size[n] + (2.0 ** -24 * w.abs() if n == "dS" else _half_step(x))
        off = (x - w).abs() - room
        assert (off <= 0).all(), f"{n}: {(off > 0).sum().item()} of {off.numel()} further off than float32 and one rounding allow, by {off.max().item():.3g}"


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("Dk, Dv", [(16, 16), (64, 64), (64, 128), (128, 64), (128, 128), (41, 101)])
def test_gradients_do_not_depend_on_what_else_is_wanted(Dk, Dv, dtype, dev):
    """q's, k's and v's gradients are the same bits with learned and with fixed decays."""
    from timediff_amd.decay_attention import decay_attention
    g = torch.Generator().manual_seed(5)
    q, k, v, do = (torch.randn(2, 150, 2, d, generator=g).to(dtype).to(dev) for d in (Dk, Dk, Dv, Dv))
    res = []
    for slope in (True, False):
        leaf = [t.clone().requires_grad_() for t in (q, k, v)]
        o = decay_attention(*leaf, torch.tensor([-0.02, -0.4], device=dev, requires_grad=slope))
        res.append(torch.autograd.grad(o, leaf, do))
    for a, b in zip(*res):
        assert torch.equal(a, b)


@pytest.mark.parametrize("log_decay", [-0.01, -0.3, -0.6])
def test_weights(log_decay, dev):
    """One row's reach: with k_0 alone nonzero o_t = g^t, with grad_o's last row alone nonzero grad_v_j = g^(T-1-j), a single weight each, down
    to 2^-111.  A weight is 2^x (one unit in the last place: 2 roundings), a first-order correction (2), and itself rounded (1), 3 more for the
    products around it: 8 within a chunk of 64.  Across a border three weights (8 each), their products (6), and 2 for every chunk's decay."""
    from timediff_amd.decay_attention import decay_attention
    T = 128
    one = torch.ones(1, T, 1, 1, device=dev)
    k, do = torch.zeros_like(one), torch.zeros_like(one)
    k[:, 0], do[:, -1] = 1, 1
    ld = torch.tensor([log_decay], device=dev)
    t = torch.arange(T, device=dev)
    exact = torch.exp(ld.double() * t)
    room = torch.where(t < 64, 8, 30 + 4) * 2.0 ** -24 * exact
    o = decay_attention(one, k, one, ld, scale=1.0)[0, :, 0, 0].double()
    v = one.clone().requires_grad_()
    dv = torch.autograd.grad(decay_attention(one, one, v, ld, scale=1.0), v, do)[0][0, :, 0, 0].double().flip(0)
    for name, x in (("o", o), ("dv", dv)):
        off = (x - exact).abs() - room
        assert (off <= 0).all(), f"{name}: {((x - exact).abs() / exact).max().item() * 2 ** 24:.1f} roundings at most, {(off > 0).nonzero().flatten().tolist()[:5]} ..."


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("D", [16, 48, 100])
@pytest.mark.parametrize("T, log_decay", [(1, 6.0), (5, 3.0), (20, 2.9), (40, 1.5), (50, 1.45)])
def test_growing_states_of_short_sequences(T, log_decay, D, dtype, dev):
    """Decays above zero whose g^T is far from overflowing, while g^32 or g^64 would: every result is finite, log_decay's gradient too, and as
    near the 64-bit one as float32's sums of T and D terms, 32 roundings beside, and a rounding to the result's type allow."""
    import decay_reference as ref
    from timediff_amd.decay_attention import decay_attention
    g = torch.Generator().manual_seed(T)
    x = {n: torch.randn(2, T, 2, D, generator=g).to(dtype) for n in ("q", "k", "v", "do")}
    x["S"], x["dS"] = torch.randn(2, 2, D, D, generator=g), torch.randn(2, 2, D, D, generator=g)
    x["ld"] = torch.tensor([log_decay, 0.5])
    names = ["q", "k", "v", "ld", "S"]
    leaf = {n: x[n].to(dev).requires_grad_() for n in names}
    o, s = decay_attention(*(leaf[n] for n in names[:4]), initial_state=leaf["S"], return_state=True)
    got = torch.autograd.grad([o, s], [leaf[n] for n in names], [x["do"].to(dev), x["dS"].to(dev)])
    want, size = (ref.gradients(f(x["q"]), f(x["k"]), f(x["v"]), x["ld"], f(x["do"]), f(x["dS"]), state=f(x["S"])) for f in (lambda t: t, torch.abs))
    for n, d in zip(("q", "k", "v", "log_decay", "state"), got):
        d = d.cpu().double()
        assert torch.isfinite(d).all(), n
        room = ((4 if n == "log_decay" else 1) * T + 2 * D + 32) * 2.0 ** -24 * size[n] + (2.0 ** -8 if dtype is BF16 and n in "qkv" else 2.0 ** -24) * want[n].abs()
        assert ((d - want[n]).abs() <= room).all(), n


def test_states_of_long_sequences(dev):
    """float32 states of 16384 rows in one piece, with positive inputs and hardly any decay, so that they grow evenly: every chunk of 64 rows
    rounds them three times (the decay and two sums of 32 rows), by 2^-24 at most and in independent directions.  The state at a rounding is t / T of the
    last, so the norm of what they leave is at most sqrt(3 x 256 / 3) 2^-24 of the state's."""
    from timediff_amd.decay_attention import decay_attention
    B, T, D = 192, 16384, 40
    g = torch.Generator(device=dev).manual_seed(2)
    q, k, v = (torch.rand(B, T, 1, D, generator=g, device=dev) for _ in range(3))
    ld = torch.tensor([-1e-6], device=dev)
    _, s = decay_attention(q, k, v, ld, return_state=True)
    w = torch.exp(ld.double() * torch.arange(T - 1, -1, -1, device=dev))[:, None]
    for b in (0, 1, 100, 191):
        exact = (k[b, :, 0].double() * w).t() @ v[b, :, 0].double()
        assert (s[b, 0].double() - exact).norm() <= 16 * 2.0 ** -24 * exact.norm(), b
