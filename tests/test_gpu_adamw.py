"""AdamW over tensor lists on the GPU against its formula in 64 bits, entry by entry.

Tolerances: every float32 operation is off by at most 2^-24 of its result.  m and v are two products and a sum, their factors
rounded too: 4 x 2^-24 of the magnitudes added.  The parameter carries 3 roundings of its own size, and the step 8 of its size
beside what m's error makes of it.  An 8-bit moment is a choice between two neighbours at t + u; float32 has t within 16 x 6 x 2^-24 and the sum
within 2^-20, together below 2^-17: further than that from a whole number the codes are equal, nearer they are neighbours."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

SIZES = [1, 3, 255, 256, 257, 0, 1000, 4096, 100003]


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    return torch.device("cuda:0")


def _apart(t, by):
    """A copy that begins `by` elements behind an aligned address."""
    return torch.cat([t.new_zeros(by), t.reshape(-1)])[by:].view(t.shape) if t.dtype != torch.float8_e4m3fn else _apart(t.view(torch.uint8), by).view(t.dtype)


def _lists(seed, dev, sizes, grad=torch.float32, bits=32, apart=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda n: torch.randn(n, generator=g)  # noqa: E731
    f = lambda t: _apart(t, apart).to(dev) if apart == 0 else _apart(t.to(dev), apart)  # noqa: E731
    x = dict(params=[f(r(n)) for n in sizes], grads=[f((r(n) * 1e-2).to(grad)) for n in sizes])
    if bits == 32:
        x.update(exp_avgs=[f(r(n) * 1e-2) for n in sizes], exp_avg_sqs=[f((r(n) * 1e-2) ** 2) for n in sizes])
    else:
        blocks = [-(-n // 256) for n in sizes]
        code = lambda n, hi: torch.rand(n, generator=g) * hi  # noqa: E731
        x.update(exp_avgs=[f(((code(n, 2) - 1) * 448).to(torch.float8_e4m3fn)) for n in sizes], exp_avg_sqs=[f((code(n, 448)).to(torch.float8_e4m3fn)) for n in sizes],
                 scales=[((torch.rand(b, 2, generator=g) + 0.1) * 1e-4).to(dev) for b in blocks],
                 random=[f(torch.randint(-2 ** 31, 2 ** 31, (n,), generator=g, dtype=torch.int32)) for n in sizes])
    return x


def _clone(x):
    return {k: [t.clone() for t in v] for k, v in x.items()}


def _cpu(x):
    return {k: [t.cpu().float().double() if t.is_floating_point() else t.cpu() for t in v] for k, v in x.items()}


def _formula(p, g, m, v, lr, betas, eps, weight_decay, step, gs):
    g = g * gs
    mm, vv = betas[0] * m + (1 - betas[0]) * g, betas[1] * v + (1 - betas[1]) * g * g
    em = 2.0 ** -22 * (betas[0] * m.abs() + (1 - betas[0]) * g.abs())
    k = lr / (1 - betas[0] ** step)
    down = vv.sqrt() / math.sqrt(1 - betas[1] ** step) + eps
    new = p * (1 - lr * weight_decay) - k * mm / down
    return new, mm, vv, 2.0 ** -24 * (3 * p.abs() + 8 * (k * mm / down).abs()) + k * em / down, em, 2.0 ** -22 * vv


HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05, step=5)


@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("apart", [0, 1, 2])
@pytest.mark.parametrize("scaled", [False, True])
def test_32_bits(grad, apart, scaled, dev):
    from timediff_amd.optim import adamw_
    x = _lists(3, dev, SIZES * 6, grad, apart=apart)          # 54 tensors: two launches
    before = _cpu(x)
    adamw_(**x, **HYPER, grad_scale=torch.tensor([0.37], device=dev) if scaled else None)
    after = _cpu(x)
    gs = float(np.float32(0.37)) if scaled else 1.0
    for i in range(len(x["params"])):
        p, m, v, ep, em, ev = _formula(*(before[k][i] for k in ("params", "grads", "exp_avgs", "exp_avg_sqs")), gs=gs, **HYPER)
        for name, want, room in (("params", p, ep), ("exp_avgs", m, em), ("exp_avg_sqs", v, ev)):
            assert ((after[name][i] - want).abs() <= room).all(), (name, i)
        assert torch.equal(after["grads"][i], before["grads"][i])


def _codes(x, u, n, positive):
    """The formula's codes (values in units of the scale), scales, and which choices are within 2^-17 of falling the other way."""
    top = torch.zeros(-(-n // 256) * 256, dtype=torch.float64)
    top[:n] = x.abs()
    top = top.view(-1, 256).amax(1)
    y = x.abs() / top.repeat_interleave(256)[:n] * 448
    gap = 2.0 ** (torch.floor(torch.log2(y.clamp(min=2.0 ** -6))) - 3)
    s = y / gap + u
    low = torch.floor(s) * gap
    if positive:
        low = torch.where(x > 0, low.clamp(min=2.0 ** -9), low)
    return low * torch.sign(x), top / 448, (s - torch.round(s)).abs() < 2.0 ** -17, gap


@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("apart", [0, 1])
def test_8_bits(grad, apart, dev):
    from timediff_amd.optim import adamw_
    x = _lists(4, dev, SIZES * 6, grad, bits=8, apart=apart)
    before = _cpu(x)
    adamw_(**x, **HYPER)
    after = _cpu(x)
    for i, n in enumerate(SIZES * 6):
        sc = before["scales"][i].repeat_interleave(256, 0)[:n]
        m0, r0 = before["exp_avgs"][i] * sc[:, 0], before["exp_avg_sqs"][i] * sc[:, 1]
        p, m, v, ep, em, ev = _formula(before["params"][i], before["grads"][i], m0, r0 * r0, gs=1.0, **HYPER)
        assert ((after["params"][i] - p).abs() <= ep + 2.0 ** -22 * (p - before["params"][i]).abs()).all(), i   # decoding: 3 roundings more
        bits = before["random"][i].long() & 0xFFFFFFFF
        for name, val, word, col in (("exp_avgs", m, bits % 65536, 0), ("exp_avg_sqs", v.sqrt(), bits // 65536, 1)):
            want, scale, near, gap = _codes(val, (word.double() + 0.5) / 65536, n, col == 1)
            off = (after[name][i] - want).abs()
            # m is a difference where its terms have other signs: its error counts in units of the gap, which at worst makes it a neighbour
            loose = near | (col == 0) * ((em / scale.repeat_interleave(256)[:n]) / gap > 2.0 ** -18)
            assert (off[~loose] == 0).all() and (off <= 2 * gap).all(), (name, i)
            assert ((after["scales"][i][:, col] - scale).abs() <= 2.0 ** -21 * scale + 1e-12 * (col == 0)).all(), (name, i)


def _philox(i, position, step, seed):
    """Word i % 4 of the Philox4x32-10 block of counter (i / 4, position, step), key `seed`."""
    i = np.arange(i, dtype=np.uint64)
    c = [(i // 4) & 0xFFFFFFFF, (i // 4) >> np.uint64(32), np.full_like(i, position), np.full_like(i, step)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    M = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        p0, p1 = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), p1 & M, (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), p0 & M]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.choose((i % np.uint64(4)).astype(int), c).astype(np.uint32).view(np.int32)


def test_own_random_numbers(dev):
    """Without `random` the words are Philox's of (seed, position, index, step): the same result as with them given, from aligned
    and from unaligned tensors."""
    from timediff_amd.optim import adamw_
    sizes = [700, 0, 513, 4096]
    x = _lists(6, dev, sizes, bits=8)
    seed = 0x1234567890ABCDEF
    x["random"] = [torch.from_numpy(_philox(n, i, HYPER["step"], seed)).to(dev) for i, n in enumerate(sizes)]
    given, own = _clone(x), _clone(x)
    own.pop("random")
    odd = {k: v if k == "scales" else [_apart(t, 1) for t in v] for k, v in _clone(own).items()}
    other = _clone(own)
    adamw_(**given, **HYPER)
    adamw_(**own, **HYPER, seed=seed)
    adamw_(**odd, **HYPER, seed=seed)
    adamw_(**other, **HYPER, seed=seed + 1)
    for k in ("params", "exp_avgs", "exp_avg_sqs", "scales"):
        for a, b, c in zip(given[k], own[k], odd[k]):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)) and torch.equal(a.view(torch.uint8), c.view(torch.uint8)), k
    assert any((a.view(torch.uint8) != b.view(torch.uint8)).any() for a, b in zip(own["exp_avgs"], other["exp_avgs"]))


def test_rounding_is_unbiased(dev):
    """All 65536 values of a half word once: the mean of the codes is the value, within 2^-15 of the neighbours' distance (the
    mean of floor(t + u) is within 2^-16 of t, and t within 2^-17)."""
    from timediff_amd.optim import adamw_
    blocks = 258                                       # the first value of a block is its largest, the others are all alike
    n = blocks * 256
    words = torch.zeros(blocks, 256, dtype=torch.int64)
    free = torch.arange(blocks * 255) % 65536
    words[:, 1:] = (free + (65535 - free) * 65536).view(blocks, 255)
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32).view(-1)
    for value in (0.7003, 0.0211, 0.51, 1.3e-5):
        g = torch.full((blocks, 256), value)
        g[:, 0] = 1.0
        z8 = torch.zeros(n, device=dev).to(torch.float8_e4m3fn)
        m8, r8, sc = z8.clone(), z8.clone(), torch.zeros(blocks, 2, device=dev)
        adamw_([torch.zeros(n, device=dev)], [g.view(-1).to(dev)], [m8], [r8], [sc], lr=0.0, betas=(0.0, 0.0), eps=1.0, weight_decay=0.0, step=1,
               random=[words.to(dev)])
        for codes, col in ((m8, 0), (r8, 1)):
            got = (codes.float().view(blocks, 256) * sc[:, col:col + 1])[:, 1:].cpu().double().reshape(-1)[:65536]
            y = float(np.float32(value)) * 448
            gap = 2.0 ** (max(math.floor(math.log2(y)), -6) - 3) / 448
            if col == 1 and y < 2.0 ** -9:
                continue                                # a second moment above zero is never stored as zero: biased upwards there
            assert abs(got.mean().item() - value) <= 2.0 ** -15 * gap + 2.0 ** -22 * value, (value, col)


def test_blocks_of_zeros_and_tiny_values(dev):
    from timediff_amd.optim import adamw_
    n = 1024
    g = torch.zeros(n)
    g[256:512] = 1e-30            # m: 1e-31, below 2^-100; sqrt(v): 1e-31
    g[512:768] = 1e-20
    g[768] = 1.0
    g[769:] = 1e-12               # far below the block's largest: m may be zero, sqrt(v) must not
    z8 = torch.zeros(n, device=dev).to(torch.float8_e4m3fn)
    m8, r8, sc, p = z8.clone(), z8.clone(), torch.full((4, 2), 7.0, device=dev), torch.ones(n, device=dev)
    adamw_([p], [g.to(dev)], [m8], [r8], [sc], lr=1e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.0, step=1)
    assert torch.isfinite(p).all() and (p[:256] == 1).all()
    assert (sc[0] == 0).all() and sc[1, 0] == 0 and (sc[2:] > 0).all()
    assert (m8.float()[:512] == 0).all() and (r8.float()[768:] > 0).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_gradient_that_is_not_finite(bad, dev):
    """32 bits: that value alone; 8 bits: its parameter, and the moments of its block."""
    from timediff_amd.optim import adamw_
    for bits in (32, 8):
        x = _lists(8, dev, [1024], bits=bits)
        y = _clone(x)
        x["grads"][0][300] = bad
        for z in (x, y):
            adamw_(**z, **HYPER)
        hit = torch.arange(1024, device=dev) == 300
        assert not torch.isfinite(x["params"][0][300]) and torch.equal(x["params"][0][~hit], y["params"][0][~hit])
        if bits == 8:
            block = torch.arange(1024, device=dev) // 256 == 1
            m = x["exp_avgs"][0].float() * x["scales"][0][:, 0].repeat_interleave(256)
            assert not torch.isfinite(m[block]).any() and torch.equal(x["exp_avgs"][0].view(torch.uint8)[~block], y["exp_avgs"][0].view(torch.uint8)[~block])


def _params(dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*s, generator=g).to(dev).requires_grad_() for s in ((40, 30), (7,), (300,), (3, 3, 3))]


def _grads(step, i, shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(100 * step + i)) * 0.1


def test_optimizer_is_torchs(dev):
    """Two groups, a param that gets its first gradient later, another without one now and then: torch.optim.AdamW in 64 bits, each
    step's rounding (a few 2^-24 of the values) carried along, 6 steps."""
    from timediff_amd.optim import AdamW
    mine = _params(dev)
    theirs = [p.detach().cpu().double().requires_grad_() for p in mine]
    groups = lambda ps: [dict(params=ps[:2], lr=1e-2), dict(params=ps[2:], weight_decay=0.3, betas=(0.8, 0.99))]  # noqa: E731
    a, b = AdamW(groups(mine), lr=3e-3), torch.optim.AdamW(groups(theirs), lr=3e-3)
    for step in range(6):
        for i, (p, q) in enumerate(zip(mine, theirs)):
            live = not (i == 1 and step < 2) and not (i == 2 and step % 2)
            g = _grads(step, i, p.shape)
            p.grad, q.grad = (g.to(dev), g.double()) if live else (None, None)
        a.step()
        b.step()
    for p, q in zip(mine, theirs):
        assert ((p.cpu().double() - q).abs() <= 6 * 2.0 ** -22 * (q.abs() + 6 * 1e-2)).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_round_trip(bits, dev, tmp_path):
    """A saved and loaded optimizer goes on bit for bit."""
    from timediff_amd.optim import AdamW
    ps = _params(dev)
    opt = AdamW(ps, state_bits=bits, seed=5)
    def feed(params, o, steps):
        for step in steps:
            for i, p in enumerate(params):
                p.grad = _grads(step, i, p.shape).to(dev)
            o.step()
    feed(ps, opt, range(3))
    torch.save(opt.state_dict(), tmp_path / "opt.pt")
    copy = [p.detach().clone().requires_grad_() for p in ps]
    again = AdamW(copy, state_bits=bits, seed=5)
    again.load_state_dict(torch.load(tmp_path / "opt.pt", weights_only=True))
    feed(ps, opt, range(3, 5))
    feed(copy, again, range(3, 5))
    for p, q in zip(ps, copy):
        assert torch.equal(p, q)
        for k, t in opt.state[p].items():
            assert k == "step" and again.state[q][k] == t == 5 or torch.equal(again.state[q][k].view(torch.uint8), t.view(torch.uint8)) and again.state[q][k].dtype == t.dtype


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps(bits, dev):
    """A replayed step with advance() before each replay is the eager step, learning rate changes included; without capturable, a
    capture is refused."""
    from timediff_amd.optim import AdamW
    ps, qs = _params(dev), _params(dev)
    a, b = AdamW(ps, state_bits=bits, seed=1), AdamW([dict(params=qs)], state_bits=bits, seed=1, capturable=True)
    for i, (p, q) in enumerate(zip(ps, qs)):
        p.grad, q.grad = (_grads(0, i, p.shape).to(dev) for _ in range(2))
    a.step()
    b.step()
    plain = AdamW(_params(dev))
    for p in plain.param_groups[0]["params"]:
        p.grad = torch.zeros_like(p)
    graph, scale = torch.cuda.CUDAGraph(), torch.ones(1, device=dev)
    refused = []
    with torch.cuda.graph(graph):
        b.step(grad_scale=scale)
        try:
            plain.step()
        except RuntimeError as e:
            refused.append(str(e))
    assert refused and "capturable" in refused[0]
    for step in range(1, 5):
        for i, (p, q) in enumerate(zip(ps, qs)):
            g = _grads(step, i, p.shape).to(dev)
            p.grad.copy_(g)
            q.grad.copy_(g)
        scale.fill_(1.0 / step)
        for o in (a, b):
            o.param_groups[0]["lr"] = 1e-3 * step
        a.step(grad_scale=scale)
        b.advance()
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(ps, qs):
            assert torch.equal(p, q), step


def test_classifier_update_is_what_it_was(dev):
    """The classifier's AdamW step is one call of adamw_: bit for bit the multiplication and td_clip_adam_ema that it replaces."""
    import ctypes as C

    from timediff_amd import _lib
    from timediff_amd._lib import check, lib, ptr
    from timediff_amd.classifier import RNN, nnTimeSeriesClassifier
    g = torch.Generator().manual_seed(2)
    X, y = torch.randn(96, 5, 12, generator=g), (torch.rand(96, generator=g) > 0.5).long()
    y[:2] = torch.tensor([0, 1])
    torch.manual_seed(0)
    c = nnTimeSeriesClassifier(lambda in_channels: RNN(in_channels, hidden_dim=24), X, y, bsz=32)
    for _ in range(4):
        old = [t.clone() for t in (c.flat, c.exp_avg, c.exp_avg_sq)]
        c.train_step()
        old[0].mul_(1.0 - c.lr * c.weight_decay)
        check(lib().td_clip_adam_ema(ptr(old[0]), ptr(c.flat_grad), ptr(old[1]), ptr(old[2]), None, c.flat.numel(), None, 0.0, c.lr, c.betas[0],
                                     c.betas[1], c.eps, c.step, 0, 0.0, C.c_void_p(torch.cuda.current_stream().cuda_stream)))
        for a, b in zip((c.flat, c.exp_avg, c.exp_avg_sq), old):
            assert torch.equal(a, b)


@pytest.mark.parametrize("bits", [32, 8])
def test_mixer_trained_and_streamed(bits, dev):
    """The operators together: projections around decay attention with learned decays, trained for three steps with AdamW over all
    of its tensors, then run row by row from the state that a prompt leaves.  Gradients against the 64-bit reference at each step's
    own weights; the stream against the sequence form."""
    import decay_reference as ref
    from timediff_amd.decay_attention import decay_attention, decay_attention_step
    from timediff_amd.optim import AdamW
    torch.manual_seed(1)
    C_, H, D, T = 6, 4, 16, 50
    qkv, out = torch.nn.Linear(C_, 3 * H * D).to(dev), torch.nn.Linear(H * D, C_).to(dev)
    ld = torch.nn.Parameter(-torch.tensor([0.01, 0.05, 0.2, 1.0], device=dev))
    ps = [*qkv.parameters(), *out.parameters(), ld]
    opt = AdamW(ps, lr=1e-2, state_bits=bits)
    x, want = torch.randn(4, T, C_, device=dev), torch.randn(4, T, C_, device=dev)

    def mix(x, params, attend):
        w, b, wo, bo, decay = params
        q, k, v = torch.nn.functional.linear(x, w, b).unflatten(-1, (3, H, D)).unbind(-3)
        return torch.nn.functional.linear(attend(q, k, v, decay).flatten(-2), wo, bo)
    for _ in range(3):
        opt.zero_grad()
        ((mix(x, ps, decay_attention) - want) ** 2).mean().backward()
        exact = [p.detach().cpu().double().requires_grad_() for p in ps]
        ((mix(x.cpu().double(), exact, lambda *a: ref.decay_attention(*a)[0]) - want.cpu().double()) ** 2).mean().backward()
        for p, e in zip(ps, exact):
            # float32 through two projections (torch's) and the recurrence: sums of up to 200 x 192 terms, 2^-24 each, against the largest entry
            assert ((p.grad.cpu().double() - e.grad).abs() <= 4e-4 * e.grad.abs().max()).all()
        old = [p.detach().clone() for p in ps]
        opt.step()
        assert all((a != b).any() for a, b in zip(old, ps))
    with torch.no_grad():
        full = mix(x, ps, decay_attention)
        keep = {}
        def prompt(*a):
            o, keep["s"] = decay_attention(*a, return_state=True)
            return o
        rows = [mix(x[:, :20], ps, prompt)] + [mix(x[:, t], ps, lambda *a: decay_attention_step(*a, keep["s"]))[:, None] for t in range(20, T)]
        assert ((torch.cat(rows, 1) - full).abs() <= 1e-4 * full.abs().max()).all()


def test_written_params_are_noticed(dev):
    """A param that a graph saved and a step then changed: the backward pass is refused, as for torch's own writes in place."""
    from timediff_amd.optim import adamw_
    w = torch.ones(300, device=dev, requires_grad=True)
    loss = (w * w).sum()
    zeros = [torch.zeros(300, device=dev) for _ in range(2)]
    kw = dict(lr=0.1, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, step=1)
    adamw_([w], [torch.ones(300, device=dev)], zeros[:1], zeros[1:], **kw)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():               # no such count there
        p = torch.ones(300, device=dev)
        adamw_([p, w], [torch.ones(300, device=dev) for _ in range(2)], *([torch.zeros(300, device=dev) for _ in range(2)] for _ in range(2)), **kw)
    assert (p < 1).all()


def test_record_of_another_device(dev):
    """A record in host memory would be read by the kernel: refused."""
    from timediff_amd.optim import adamw_
    x = _lists(1, dev, [300])
    with pytest.raises(ValueError, match="record must be on the params' device"):
        adamw_(**x, **HYPER, record=torch.zeros(32, dtype=torch.uint8))


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_with_a_param_left_out(bits, dev):
    """Eager steps with a late gradient, then a graph that steps all params but one, replayed with advance(), then eager steps of all: the bits of
    the optimizer without capturable."""
    from timediff_amd.optim import AdamW
    ps, qs = _params(dev), _params(dev)
    a, b = AdamW(ps, state_bits=bits, seed=1), AdamW(qs, state_bits=bits, seed=1, capturable=True)

    def feed(step, skip=()):
        for i, (p, q) in enumerate(zip(ps, qs)):
            g = _grads(step, i, p.shape).to(dev)
            if i in skip:
                p.grad = q.grad = None
            else:
                p.grad = g
                q.grad = g.clone() if q.grad is None else q.grad.copy_(g)
    for step in range(3):
        feed(step, skip=(1,) if step < 2 else ())
        a.step()
        b.step()
    feed(3, skip=(1,))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.step()
    for step in range(3, 6):
        feed(step, skip=(1,))
        a.step()
        b.advance()
        graph.replay()
        torch.cuda.synchronize()
    for step in range(6, 8):
        feed(step)
        a.step()
        b.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)
        assert a.state[p]["step"] == b.state[q]["step"]
