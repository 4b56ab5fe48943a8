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
