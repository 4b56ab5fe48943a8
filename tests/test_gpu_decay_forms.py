"""Every form of decay attention's kernels against the 64-bit reference (tests/decay_reference.py): packed sequences that are cut into segments, fixed
decays (a backward kernel of their own), and backward passes of more sequences and heads than workgroups.

An entry is a sum of at most K products of inputs and weights, M the sum of their magnitudes (the same reference on the inputs' magnitudes): float32
is off by at most K 2^-24 M, and 32 roundings more of M for weights, scales and the splitting of operands; then one rounding to the result's type.
K: a sum over D, one over a sequence's rows T, one over both for the products that pass through a state, and for log_decay's gradient, which sums
over all rows R and their distances in double precision, the three of its parts: D + 2 T for entries, D + 3 T for log_decay."""
import pytest
import torch

import decay_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
NAMES = ("q", "k", "v", "log_decay", "state")


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    return torch.device("cuda:0")


def _inputs(seed, lead, n, heads, Dk, Dv, dtype):
    H, Hq, Hk, Hv = heads
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return dict(q=r(*lead, Hq, Dk).to(dtype), k=r(*lead, Hk, Dk).to(dtype), v=r(*lead, Hv, Dv).to(dtype), log_decay=-torch.exp(torch.rand(H, generator=g) * 6 - 6.5),
                state=r(n, H, Dk, Dv), grad_o=r(*lead, H, Dv).to(dtype), grad_state=r(n, H, Dk, Dv))


def _run(x, dev, learned, offsets=None):
    """-> {name: result}, gradients among them, with learned or with fixed decays."""
    from timediff_amd.decay_attention import decay_attention
    leaf = {n: x[n].to(dev).requires_grad_(learned or n != "log_decay") for n in NAMES}
    o, s = decay_attention(*(leaf[n] for n in NAMES[:4]), offsets=None if offsets is None else offsets.to(dev), initial_state=leaf["state"], return_state=True)
    want = [n for n in NAMES if leaf[n].requires_grad]
    d = torch.autograd.grad([o, s], [leaf[n] for n in want], [x["grad_o"].to(dev), x["grad_state"].to(dev)])
    return {"o": o.detach(), "final": s.detach(), **{"grad " + n: t for n, t in zip(want, d)}}


def _reference(x, offsets=None):
    res = []
    for f in (lambda t: t, torch.abs):
        a = [f(x[n]) for n in "qkv"] + [x["log_decay"]]
        o, s = ref.decay_attention(*a, state=f(x["state"]), offsets=offsets)
        d = ref.gradients(*a, f(x["grad_o"]), f(x["grad_state"]), state=f(x["state"]), offsets=offsets)
        res.append({"o": o, "final": s, **{"grad " + n: d[n] for n in NAMES}})
    return res


def _close(name, got, want, size, T, D):
    got, want, size = got.cpu(), want.detach(), size.detach()
    assert got.shape == want.shape and torch.isfinite(got.float()).all(), name
    terms = D + (3 if name == "grad log_decay" else 2) * T + 32
    off = (got.double() - want).abs() - terms * 2.0 ** -24 * size - (2.0 ** -8 if got.dtype == BF16 else 2.0 ** -24) * want.abs() - 2.0 ** -98
    assert (off <= 0).all(), f"{name}: {(off > 0).sum().item()} of {off.numel()} outside, by {off.max().item():.3g} (largest {want.abs().max().item():.3g})"


SIZES = [(16, 16), (64, 64), (64, 128), (128, 64), (128, 128), (41, 101), (60, 33)]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("heads", [(2, 2, 2, 2), (4, 2, 1, 4)], ids=["own", "shared"])
@pytest.mark.parametrize("Dk, Dv", SIZES)
def test_packed_and_cut(Dk, Dv, heads, dtype, dev):
    """Segments of 256 rows in both directions: sequences of several, of one, shorter than a chunk, empty, and ends inside tiles; rows of none on
    both sides.  Fixed decays give the same bits."""
    lengths = [700, 0, 37, 256, 1, 333, 64]
    off = torch.tensor([5 + sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32)
    rows = 5 + sum(lengths) + 9
    x = _inputs(Dk + Dv, (rows,), len(lengths), heads, Dk, Dv, dtype)
    got, fixed = _run(x, dev, True, off), _run(x, dev, False, off)
    want, size = _reference(x, off)
    for n, t in got.items():
        _close(n, t, want[n], size[n], max(lengths), max(Dk, Dv))
        if n != "grad log_decay":
            assert torch.equal(t, fixed[n]), n
        if n in ("o", "grad q", "grad k", "grad v"):
            assert (t[:5] == 0).all() and (t[-9:] == 0).all(), n


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T", [1, 40, 150, 1100])
@pytest.mark.parametrize("Dk, Dv", SIZES)
def test_dense(Dk, Dv, T, dtype, dev):
    """Whole and cut (1100 rows), with learned and with fixed decays, log_decay's gradient over all sequences."""
    x = _inputs(Dk + T, (3, T), 3, (2, 1, 2, 2), Dk, Dv, dtype)
    got, fixed = _run(x, dev, True), _run(x, dev, False)
    want, size = _reference(x)
    for n, t in got.items():
        _close(n, t, want[n], size[n], T, max(Dk, Dv))
        if n != "grad log_decay":
            assert torch.equal(t, fixed[n]), n


@pytest.mark.parametrize("learned", [True, False], ids=["learned", "fixed"])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("Dk, Dv", SIZES)
def test_more_items_than_workgroups(Dk, Dv, dtype, learned, dev):
    """600 sequences of 2 heads: a workgroup of the backward pass takes several, one after another.  A sequence's results are its own: those of the first, second and
    third trips are held against the reference, and all of them against a call of a few sequences each, which has a workgroup for every one."""
    B, T = 600, 70
    x = _inputs(Dk, (B, T), B, (2, 2, 2, 2), Dk, Dv, dtype)
    got = _run(x, dev, learned)
    pick = [0, 255, 256, 300, 511, 512, 599]
    want, size = _reference({n: t if n == "log_decay" else t[pick] for n, t in x.items()})
    slope, parts = 0.0, 0.0
    for i in range(0, B, 100):
        part = _run({n: t if n == "log_decay" else t[i:i + 100] for n, t in x.items()}, dev, learned)
        for n, t in part.items():
            if n == "grad log_decay":
                slope, parts = slope + t.double(), parts + t.double().abs()
            else:
                assert torch.equal(got[n][i:i + 100], t), n
    for n, t in got.items():
        if n != "grad log_decay":
            _close(n, t[pick], want[n], size[n], T, max(Dk, Dv))
    if learned:                       # the sum is double: each part's rounding to float32, and its own
        assert ((got["grad log_decay"].double() - slope).abs() <= 2.0 ** -24 * (parts + slope.abs())).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("first, second", [("q", "k"), ("grad_o", "v")])
@pytest.mark.parametrize("Dk, Dv, T, rows", [(16, 16, 5, (1, 3)), (64, 64, 64, (0, 63)), (64, 64, 100, (70, 71)), (64, 128, 64, (17, 18)), (64, 128, 40, (2, 39)), (128, 128, 90, (5, 60)),
                                             (41, 101, 64, (30, 33))])
def test_products_of_later_rows_overflow(Dk, Dv, T, rows, first, second, dtype, dev):
    """Row a of one tensor and a later row b of its partner hold 2^70: their product overflows and belongs to no result, since b is behind a.  All
    others are finite."""
    x = _inputs(T, (2, T), 2, (2, 2, 2, 2), Dk, Dv, dtype)
    a, b = rows
    x[first][:, a, :, 0] = 2.0 ** 70
    x[second][:, b, :, 0] = 2.0 ** 70
    want, size = _reference(x)
    for learned in (True, False):
        for n, t in _run(x, dev, learned).items():
            _close(n, t, want[n], size[n], T, max(Dk, Dv))
