"""AdamW over tensor lists without a GPU: what the entry points refuse."""
import ctypes as C

import pytest
import torch

from timediff_amd import _lib
from timediff_amd.optim import AdamW, adamw_

HYPER = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, step=1)


def _lists(n=300, bits=32):
    z = torch.zeros(n)
    if bits == 32:
        return dict(params=[z], grads=[z.clone()], exp_avgs=[z.clone()], exp_avg_sqs=[z.clone()])
    z8 = z.to(torch.float8_e4m3fn)
    return dict(params=[z], grads=[z.clone()], exp_avgs=[z8], exp_avg_sqs=[z8.clone()], scales=[torch.zeros(2, 2)])


@pytest.mark.parametrize("bits, bad, error, text", [
    (32, dict(params=[torch.zeros(300, dtype=torch.bfloat16)]), TypeError, "params must be torch.float32"),
    (32, dict(grads=[torch.zeros(300, dtype=torch.float16)]), TypeError, "grads must be torch.bfloat16 or torch.float32"),
    (32, dict(grads=[]), ValueError, "0 grads for 1 params"),
    (32, dict(params=[torch.zeros(600)[::2]]), ValueError, "contiguous"),
    (32, dict(exp_avgs=[torch.zeros(300).to(torch.float8_e4m3fn)]), TypeError, "exp_avgs must be torch.float32"),
    (32, dict(random=[torch.zeros(300, dtype=torch.int32)]), ValueError, "random is for 8-bit"),
    (8, dict(scales=[torch.zeros(1, 2)]), ValueError, "2 values for each 256"),
    (8, dict(exp_avgs=[torch.zeros(300)]), TypeError, "exp_avgs must be torch.float8_e4m3fn"),
    (8, dict(random=[torch.zeros(300, dtype=torch.int64)]), TypeError, "random must be torch.int32"),
    (32, {}, ValueError, "ROCm device"),
    (8, {}, ValueError, "ROCm device"),
])
def test_refusals(bits, bad, error, text):
    with pytest.raises(error, match=text):
        adamw_(**dict(_lists(bits=bits), **bad), **HYPER)


@pytest.mark.parametrize("name", ["params", "exp_avgs", "exp_avg_sqs", "scales"])
def test_same_tensor_twice(name):
    lists = {k: [t.clone() for t in v for _ in range(2)] for k, v in _lists(bits=8).items()}
    lists[name][1] = lists[name][0]
    with pytest.raises(ValueError, match=f"the same tensor twice in {name}"):
        adamw_(**lists, **HYPER)
    # empty ones share an address, and a gradient is only read
    lists = {k: [t.clone() for t in v for _ in range(2)] + [t[:0].clone() for t in v for _ in range(2)] for k, v in _lists(bits=8).items()}
    lists["grads"][1] = lists["grads"][0]
    with pytest.raises(ValueError, match="ROCm device"):
        adamw_(**lists, **HYPER)


def test_empty_list_is_no_step():
    adamw_([], [], [], [], **HYPER)


def test_optimizer_refusals():
    for kw in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            AdamW([torch.zeros(3, requires_grad=True)], **kw)
    with pytest.raises(ValueError, match="contiguous float32"):
        AdamW([torch.zeros(3, dtype=torch.bfloat16, requires_grad=True)])
    with pytest.raises(RuntimeError, match="capturable"):
        AdamW([torch.zeros(3, requires_grad=True)]).advance()
    opt = AdamW([torch.zeros(3, requires_grad=True)], state_bits=8)
    with pytest.raises(ValueError, match="32-bit moments"):
        opt.load_state_dict({"state": {0: {"step": 1, "exp_avg": torch.zeros(3), "exp_avg_sq": torch.zeros(3)}}, "param_groups": opt.state_dict()["param_groups"]})


@pytest.mark.parametrize("field, value, text", [("step", 0, b"step counts from 1"), ("beta1", 1.0, b"betas"), ("beta2", -0.1, b"betas"),
                                                ("lr", -1.0, b"must not be negative"), ("eps", -1.0, b"must not be negative"),
                                                ("weight_decay", -1.0, b"must not be negative"), ("state_bits", 16, b"state_bits"),
                                                ("beta1", float("nan"), b"betas")])
def test_library_refuses_bad_configurations(field, value, text):
    L = _lib.lib()
    cfg = _lib.AdamwConfig(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, step=1, state_bits=32)
    assert L.td_adamw(C.byref(cfg), None, 0, None) == 0            # an empty list: nothing to do
    setattr(cfg, field, value)
    assert L.td_adamw(C.byref(cfg), None, 0, None) == 1 and text in L.td_last_error()
    assert L.td_adamw_record_set(C.c_void_p(256), C.byref(cfg), None) == 1


def test_library_refuses_bad_tensors():
    L = _lib.lib()
    cfg = _lib.AdamwConfig(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, step=1, state_bits=8)
    good = dict(param=256, grad=256, exp_avg=256, exp_avg_sq=256, scales=256, n=4, grad_dtype=_lib.F32)      # addresses never used
    for bad, text in ((dict(grad=None), b"tensor 0: null pointer"), (dict(scales=None), b"need scales"), (dict(n=-1), b"bad size"),
                      (dict(grad_dtype=7), b"gradients must be"), (dict(n=2 ** 62), b"too large")):
        t = _lib.AdamwTensor(**dict(good, **bad))
        assert L.td_adamw(C.byref(cfg), C.byref(t), 1, None) == 1 and text in L.td_last_error(), bad
    assert L.td_adamw(C.byref(cfg), None, 1, None) == 1
    assert L.td_adamw_record_set(None, C.byref(cfg), None) == 1


@pytest.mark.parametrize("record", [torch.zeros(8), torch.zeros(31, dtype=torch.uint8), torch.zeros(64, dtype=torch.uint8)[::2], torch.zeros(40, dtype=torch.uint8)[1:33]])
def test_records_that_are_none(record):
    """A kernel would read a td_adamw_record there."""
    with pytest.raises(ValueError, match="record must be the 32 bytes"):
        adamw_(**_lists(), **HYPER, record=record)
    with pytest.raises(ValueError, match="ROCm device"):
        adamw_(**_lists(), **HYPER, record=torch.zeros(32, dtype=torch.uint8))
