"""The AdamW optimizer's own bookkeeping without a GPU: the calls that reach the kernels are recorded in place of adamw_."""
import pytest
import torch

from timediff_amd import optim
from timediff_amd.optim import AdamW


class Calls(list):
    """(params, step, seed, whether a record was given) of every adamw_ call."""
    refuse = capturing = False

    def adamw_(self, params, grads, exp_avgs, exp_avg_sqs, scales=None, **kw):
        if self.refuse:
            raise TypeError("refused")
        self.append(([id(p) for p in params], kw["step"], kw["seed"], kw["record"] is not None))


@pytest.fixture
def calls(monkeypatch):
    got = Calls()
    monkeypatch.setattr(optim, "adamw_", got.adamw_)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: got.capturing)
    return got


def _params(n=3):
    return [torch.zeros(4, requires_grad=True) for _ in range(n)]


def test_a_refused_step_is_not_counted(calls):
    ps = _params(1)
    opt = AdamW(ps)
    ps[0].grad = torch.zeros(4)
    calls.refuse = True
    with pytest.raises(TypeError):
        opt.step()
    calls.refuse = False
    opt.step()
    opt.step()
    assert [c[1] for c in calls] == [1, 2] and opt.state[ps[0]]["step"] == 2


def test_params_at_neighbouring_steps(calls):
    """A param one step behind another is stepped once."""
    ps = _params(2)
    opt = AdamW(ps)
    ps[0].grad = torch.zeros(4)
    opt.step()
    ps[1].grad = torch.zeros(4)
    opt.step()
    assert [c[:2] for c in calls] == [([id(ps[0])], 1), ([id(ps[1])], 1), ([id(ps[0])], 2)]
