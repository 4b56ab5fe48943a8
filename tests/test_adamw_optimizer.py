"""The AdamW optimizer's own bookkeeping without a GPU: the calls that reach the kernels are recorded in place of adamw_."""
import copy
import io
import pickle

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
    got.records = []

    def record(self, i, step):
        self._records.setdefault(i, object())
        got.records.append((i, step))
    monkeypatch.setattr(optim, "adamw_", got.adamw_)
    monkeypatch.setattr(AdamW, "_record", record)
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


@pytest.mark.parametrize("capturable", [False, True])
def test_late_and_missing_gradients(capturable, calls):
    """A param counts the steps that it takes part in, as torch.optim.AdamW's does, with capturable and without."""
    ps = _params(3)
    theirs = _params(3)
    a, b = AdamW(ps, capturable=capturable), torch.optim.AdamW(theirs)
    for step in range(6):
        for i, (p, q) in enumerate(zip(ps, theirs)):
            live = not (i == 1 and step < 3) and not (i == 2 and step % 2)
            p.grad, q.grad = (torch.zeros(4), torch.zeros(4)) if live else (None, None)
        a.step()
        b.step()
        for p, q in zip(ps, theirs):
            assert a.state[p].get("step", 0) == (b.state[q]["step"].item() if b.state[q] else 0)
    assert not any(c[3] for c in calls)                       # an eager step takes its numbers from the host


def test_captured_steps_are_counted_for_their_params(calls):
    """Two groups; one param never has a gradient.  An advance() with no gradient about counts them all, and the capture takes back what it does not
    step; afterwards advance() counts the captured ones."""
    ps = _params(4)
    opt = AdamW([dict(params=ps[:2]), dict(params=ps[2:])], capturable=True)
    steps = lambda: [opt.state[p]["step"] for p in ps]  # noqa: E731
    opt.advance()
    assert steps() == [1, 1, 1, 1] and calls.records == [(0, 1), (1, 1)]
    for p in ps[:3]:
        p.grad = torch.zeros(4)
    calls.capturing = True
    opt.step()
    calls.capturing = False
    assert steps() == [1, 1, 1, 0] and [c[1:2] + c[3:] for c in calls] == [(1, True), (1, True)]
    ps[3].grad = torch.zeros(4)
    opt.advance()
    opt.advance()
    assert steps() == [3, 3, 3, 0] and calls.records[-2:] == [(0, 3), (1, 3)]
    opt.step()                                                # eager: each at its own step
    assert steps() == [4, 4, 4, 1] and [c[1] for c in calls[-3:]] == [4, 1, 4] and not calls[-1][3]
    calls.capturing = True
    with pytest.raises(RuntimeError, match="must be at the same step, group 1 has \\[1, 4\\]"):
        opt.step()
    calls.capturing = False
    opt.advance()                                             # the graph captured before goes on
    assert steps() == [5, 5, 5, 1]


def test_captures_that_are_refused(calls):
    ps = _params(2)
    opt = AdamW(ps[:1], capturable=True)
    ps[0].grad, ps[1].grad = torch.zeros(4), torch.zeros(4)
    calls.capturing = True
    with pytest.raises(RuntimeError, match="one step\\(\\) or advance\\(\\) before the capture"):
        opt.step()
    calls.capturing = False
    opt.step()
    opt.add_param_group(dict(params=ps[1:]))                  # a group without a record yet
    calls.capturing = True
    with pytest.raises(RuntimeError, match="one step\\(\\) or advance\\(\\) before the capture"):
        opt.step()
    assert len(calls) == 1


def _saved(opt):
    f = io.BytesIO()
    torch.save(opt, f)
    return torch.load(io.BytesIO(f.getvalue()), weights_only=False)


# (pickle alone does not take torch's float8 tensors)
@pytest.mark.parametrize("bits, way", [(32, copy.deepcopy), (8, copy.deepcopy), (32, lambda o: pickle.loads(pickle.dumps(o))), (32, _saved), (8, _saved)])
def test_copies_step(bits, way, calls):
    ps = _params(2)
    opt = AdamW([dict(params=ps[:1]), dict(params=ps[1:])], state_bits=bits, seed=7, capturable=True)
    for p in ps:
        p.grad = torch.zeros(4)
    opt.step()
    other = way(opt)
    assert (other.state_bits, other.capturable) == (bits, True) and other.param_groups[0]["params"][0] is not ps[0]
    for g in other.param_groups:
        for p in g["params"]:
            p.grad = torch.zeros(4)
    opt.step()
    other.step()
    assert [c[1:] for c in calls[-2:]] == [c[1:] for c in calls[-4:-2]] == [(2, 7, False), (2, 7 + 2 ** 32, False)]
    assert other._records.keys() == {0, 1} and other._records[0] is not opt._records[0]


def test_seed_is_saved(calls):
    """A resumed run rounds from the saved stream; a state saved without one keeps the optimizer's own."""
    ps = _params(1)
    opt = AdamW(ps, state_bits=8, seed=11)
    ps[0].grad = torch.zeros(4)
    opt.step()
    again = AdamW(ps, state_bits=8)
    again.load_state_dict(opt.state_dict())
    again.step()
    old = opt.state_dict()
    old["param_groups"] = [{k: v for k, v in g.items() if k != "seed"} for g in old["param_groups"]]
    third = AdamW(ps, state_bits=8, seed=5)
    third.load_state_dict(old)
    third.step()
    assert [c[1:3] for c in calls] == [(1, 11), (2, 11), (2, 5)]


def test_torchs_state_is_loaded(calls):
    ps, theirs = _params(2), _params(2)
    old = torch.optim.AdamW(theirs, lr=0.5)
    for q in theirs:
        q.grad = torch.ones(4)
    old.step()
    old.step()
    opt = AdamW(ps)
    opt.load_state_dict(old.state_dict())
    for p, q in zip(ps, theirs):
        p.grad = torch.ones(4)
        assert torch.equal(opt.state[p]["exp_avg"], old.state[q]["exp_avg"]) and torch.equal(opt.state[p]["exp_avg_sq"], old.state[q]["exp_avg_sq"])
    opt.step()
    assert [c[1] for c in calls] == [3] and opt.param_groups[0]["lr"] == 0.5
    for option in ("amsgrad", "maximize"):
        with pytest.raises(ValueError, match=option):
            AdamW(ps).load_state_dict(torch.optim.AdamW(theirs, **{option: True}).state_dict())
