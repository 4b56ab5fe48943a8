"""Decay attention where counts come near 32 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    return torch.device("cuda:0")


def test_rows_near_two_to_the_31(dev):
    """One sequence of 2^31 - 8192 rows, cut into segments (the inputs are one value expanded; the output is 4.3 GB).  o_t = (1 - g^(t+1)) /
    (1 - g); the state's 3 roundings a chunk of 64 decay with it: 3 x 2^-24 / (1 - g^64) of it, 2.8 %, and half a step of the result, 0.4 %."""
    from timediff_amd.decay_attention import decay_attention
    T = 2 ** 31 - 8192
    one = torch.ones(1, dtype=BF16, device=dev).expand(1, T, 1, 1)
    ld = torch.tensor([-1e-7], device=dev)
    o = decay_attention(one, one, one, ld, scale=1.0).view(-1)
    t = torch.linspace(0, T - 1, 4001, dtype=torch.float64, device=dev).long()
    ld = ld.double()
    want = torch.expm1(ld * (t + 1).double()) / torch.expm1(ld)
    room = (3 * 2.0 ** -24 / -torch.expm1(64 * ld) + 2.0 ** -8) * want
    assert ((o[t].double() - want).abs() <= room).all()


def test_more_workgroups_than_one_launch_takes(dev):
    """A launch holds fewer than 2^32 threads: 2^24 and a few states step with 256 each, 2^25 and a few sequences run with 128 each.  One
    row and 1 x 1 states: o = c (g S + k v) q in float32 (10 roundings), rounded to bfloat16 (half a step)."""
    from timediff_amd.decay_attention import decay_attention, decay_attention_step
    g = torch.Generator(device=dev).manual_seed(1)
    for n, step in ((2 ** 24 + 3, True), (2 ** 25 + 3, False)):
        q, k, v = (torch.randn(n, 1, 1, generator=g, device=dev).to(BF16) for _ in range(3))
        S, ld = torch.randn(n, 1, 1, 1, generator=g, device=dev), torch.tensor([-0.3], device=dev)
        new = ld.double().exp() * S.double().view(-1) + k.double().view(-1) * v.double().view(-1)
        size = S.double().view(-1).abs() + (k.double() * v.double()).view(-1).abs()
        want = 0.5 * new * q.double().view(-1)
        if step:
            state = S.clone()
            o = decay_attention_step(q, k, v, ld, state, scale=0.5)
        else:
            o, state = decay_attention(*(t[:, None] for t in (q, k, v)), ld, scale=0.5, initial_state=S, return_state=True)
        assert ((state.view(-1).double() - new).abs() <= 10 * 2.0 ** -24 * size).all()
        assert ((o.view(-1).double() - want).abs() <= 2.0 ** -8 * want.abs() + 20 * 2.0 ** -24 * size * q.double().view(-1).abs()).all()


@pytest.mark.parametrize("B, T, H", [(1, 70, 1), (3, 100, 2), (9, 300, 4)])
def test_odd_addresses_with_even_strides(B, T, H, dev):
    """Strides that suit 16-byte reads and addresses that do not take another kernel.  The same results as from aligned tensors: sums of up to T D products in another order, 2^-24
    each of the sums of magnitudes on both sides, and a bfloat16 step where that crosses a border."""
    import decay_reference as ref
    from timediff_amd.decay_attention import decay_attention
    Dk, Dv = 8, 72
    g = torch.Generator().manual_seed(T)
    x = [torch.randn(B, T, H, d, generator=g).to(BF16) for d in (Dk, Dk, Dv, Dv)]
    ld = -torch.exp(torch.rand(H, generator=g) * 6 - 6)

    def odd(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=dev)
        flat[1:] = t.to(dev).view(-1)
        return flat[1:].view(t.shape)
    res = []
    for f in (lambda t: t.to(dev), odd):
        leaf = [f(t).requires_grad_() for t in x[:3]] + [ld.to(dev).requires_grad_()]
        o = decay_attention(*leaf)
        res.append([o.detach(), *torch.autograd.grad(o, leaf, f(x[3]))])
    size = ref.gradients(*(t.abs() for t in x[:3]), ld, x[3].abs())
    size["o"] = ref.decay_attention(*(t.abs() for t in x[:3]), ld)[0]
    for n, a, b in zip(("o", "q", "k", "v", "log_decay"), *res):
        terms = T * (B if n == "log_decay" else 1) + T + Dv + 32
        a, b = a.cpu().double(), b.cpu().double()
        assert ((a - b).abs() <= (2.0 ** -7 if n != "log_decay" else 2.0 ** -23) * a.abs() + 2 * terms * 2.0 ** -24 * size[n]).all(), n
