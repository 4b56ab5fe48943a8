"""AdamW where a list has more values than one launch takes."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_more_workgroups_than_one_launch_takes():
    """A launch holds fewer than 2^32 threads, 2^34 - 1024 values: a tensor of a little more, with 8-bit moments (138 GB), and a small one behind
    it.  From zero moments the first step is lr g / (|g| + eps)."""
    assert torch.cuda.is_available(), "these tests need the MI355X"
    dev = torch.device("cuda:0")
    n = (2 ** 24 - 1) * 1024 + 700
    if torch.cuda.mem_get_info(dev)[0] < 150 * 2 ** 30:
        pytest.skip("needs 150 GiB of device memory")
    from timediff_amd.optim import adamw_
    sizes = [n, 1000]
    z = lambda k, t: torch.zeros(k, dtype=t, device=dev)  # noqa: E731
    ps, ms, vs = ([z(k, t) for k in sizes] for t in (torch.float32, torch.uint8, torch.uint8))
    gs = [torch.full((k,), 0.25, dtype=torch.bfloat16, device=dev) for k in sizes]
    sc = [z((-(-k // 256), 2), torch.float32) for k in sizes]
    codes = lambda ts: [t.view(torch.float8_e4m3fn) for t in ts]  # noqa: E731
    lr = 2.0 ** -7
    adamw_(ps, gs, codes(ms), codes(vs), sc, lr=lr, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.0, step=1)
    # |g| = 0.25 and eps = 1e-8: off from lr by lr eps / |g| and by roundings of m, v, sqrt, the corrections and the division
    room = lr * (1e-8 / 0.25 + 8 * 2.0 ** -24)
    edge = (2 ** 24 - 1) * 1024
    for t in (ps[0][:4096], ps[0][edge - 4096:edge], ps[0][edge:], ps[1]):
        assert ((t.double() + lr).abs() <= room).all()
    assert (ps[0].amax() <= -lr + room) and (ps[0].amin() >= -lr - room)
    # every block's largest is its scale, m = 0.025 and sqrt(v) = 0.025
    for s in sc:
        assert ((s * 448 - 0.025).abs() <= 0.025 * 10 * 2.0 ** -24).all()
    assert (ms[0][edge:] == 0x7E).all() and (vs[0][edge:] == 0x7E).all()          # 448
