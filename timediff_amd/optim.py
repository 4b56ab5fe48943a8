"""AdamW over many tensors at once, its moments in 32 or in 8 bits (td_adamw), beside the trainers' flat td_clip_adam_ema.

`adamw_` steps lists of tensors that the caller owns; `AdamW` is a torch.optim.Optimizer around it.  With 8-bit moments a value
costs 2 bytes of state instead of 8: exp_avg holds m and exp_avg_sq holds sqrt(v) as float8_e4m3fn, times one float32 scale
for each 256 values (a moment's value is code.float() * scale), rounded stochastically.  No counterpart in the reference.
"""
import array
import collections
import ctypes as C
import struct

import torch

from . import _lib, ops
from ._lib import ADAMW_BLOCK, AdamwConfig, AdamwRecord, check, lib, ptr


_DTYPE, _NUMEL, _ADDRESS = torch.Tensor.dtype.__get__, torch.Tensor.numel, torch.Tensor.data_ptr
_CONTIGUOUS, _DEVICE = torch.Tensor.is_contiguous, torch.Tensor.get_device
_READ = {"grads", "random"}
_F32, _GRADS, _E4M3, _WORDS = {torch.float32}, {torch.float32, torch.bfloat16}, {torch.float8_e4m3fn}, {torch.int32}


def adamw_(params, grads, exp_avgs, exp_avg_sqs, scales=None, *, lr, betas, eps, weight_decay, step, grad_scale=None, random=None,
           seed=0, record=None):
    """One AdamW step in place over lists of tensors (one launch for every 48): params float32, grads float32 or bfloat16, all
    contiguous and on one device, none that is written twice in its list and none overlapping another.
    Moments in 32 bits: exp_avgs (m) and exp_avg_sqs (v) float32.  In 8 bits, where `scales` is given: exp_avgs (m) and exp_avg_sqs
    (sqrt(v)) float8_e4m3fn, scales float32 (ceil(n / 256), 2); all zeros is the state before the first step.
    random: for 8-bit moments, int32 tensors of the params' sizes whose low and high 16 bits round m and sqrt(v); by default the
    library draws them from (seed, position in the list, index, step).  step counts from 1.  grad_scale: a float32 device scalar that
    multiplies every gradient.  record: a device td_adamw_record (AdamW's capturable mode) read instead of lr, weight_decay, step
    and seed.  A gradient that is not finite makes its values (8 bits: the moments of its block of 256) not finite."""
    if not params:
        return
    bits = 32 if scales is None else 8
    n = list(map(_NUMEL, params))
    state = _F32 if bits == 32 else _E4M3
    # (every pass over a list is one C loop: a step over hundreds of tensors is as long as these)
    lists = [("params", params, _F32, n), ("grads", grads, _GRADS, n), ("exp_avgs", exp_avgs, state, n), ("exp_avg_sqs", exp_avg_sqs, state, n)]
    if bits == 8:
        lists.append(("scales", scales, _F32, [2 * -(-k // ADAMW_BLOCK) for k in n]))
        if random is not None:
            lists.append(("random", random, _WORDS, n))
    elif random is not None:
        raise ValueError("random is for 8-bit moments")
    if record is not None and (record.dtype is not torch.uint8 or not record.is_contiguous() or record.numel() != C.sizeof(AdamwRecord) or record.data_ptr() % 8):
        raise ValueError(f"record must be the {C.sizeof(AdamwRecord)} bytes of a td_adamw_record (uint8, at a multiple of 8)")
    for name, tensors, dtypes, sizes in lists:
        if len(tensors) != len(n):
            raise ValueError(f"{len(tensors)} {name} for {len(n)} params")
        kinds = set(map(_DTYPE, tensors))
        if not kinds <= dtypes:
            raise TypeError(f"{name} must be {' or '.join(sorted(map(str, dtypes)))}, got {', '.join(sorted(map(str, kinds - dtypes)))}")
        if not all(map(_CONTIGUOUS, tensors)):
            raise ValueError(f"{name} must be contiguous")
        if name != "params" and list(map(_NUMEL, tensors)) != sizes:
            raise ValueError(f"scales must have 2 values for each {ADAMW_BLOCK} of their param" if name == "scales" else f"{name} must have their params' sizes")
    table = array.array("q", bytes(64 * len(n)))          # td_adamw_tensor is eight 64-bit words
    for word, (name, tensors, *_) in enumerate(lists):
        table[word::8] = at = array.array("q", map(_ADDRESS, tensors))
        if name not in _READ and len(set(at)) != len(n):
            at = [a for a, k in zip(at, n) if k]
            if len(set(at)) != len(at):
                raise ValueError(f"the same tensor twice in {name}")
    index = params[0].get_device()
    for name, tensors, *_ in lists:
        if index < 0 or set(map(_DEVICE, tensors)) != {index}:
            raise ValueError(f"{name} must be on one ROCm device, the params'")
    if grad_scale is not None and (grad_scale.dtype is not torch.float32 or grad_scale.numel() != 1 or grad_scale.get_device() != index):
        raise ValueError("grad_scale must be one float32 value on the params' device")
    if record is not None and record.get_device() != index:
        raise ValueError("record must be on the params' device")
    table[6::8] = array.array("q", n)
    if set(map(_DTYPE, grads)) != _F32:
        table[7::8] = array.array("q", [_lib.F32 if g.dtype is torch.float32 else _lib.BF16 for g in grads])
    cfg = _CONFIG.pack(lr, betas[0], betas[1], eps, weight_decay, step, seed & (2 ** 64 - 1), 0 if grad_scale is None else grad_scale.data_ptr(),
                       0 if record is None else record.data_ptr(), bits, 0)
    ops._written(params)
    with ops._on_device(index):
        check(lib().td_adamw(cfg, table.buffer_info()[0], len(n), ops._raw_stream(index)))


_CONFIG = struct.Struct("<5dqQQQii")            # td_adamw_config


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's formula on td_adamw, of its arguments lr, betas, eps and weight_decay (no amsgrad or maximize); params float32, grads
    float32 or bfloat16.  With 32 bits its state dicts are loaded too.
    state_bits: 32 or 8 (state: exp_avg, exp_avg_sq[, scales], step).  seed: of the 8-bit moments' stochastic rounding, saved with the groups' other
    options.
    capturable: step() may be captured in a graph, after one eager step() or advance().  A captured step() reads step count, learning
    rate, weight decay and seed from device records, one for each group: the params of a group that it steps must be at the same step.  Call
    advance() before each replay of the graph captured last, which may hold one step().  An eager step() is the same with and without it.
    load_state_dict() makes new state tensors and records, which no earlier graph knows: capture again after it."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32, seed=0, capturable=False):
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits must be 32 or 8, got {state_bits}")
        if not (lr >= 0 and eps >= 0 and weight_decay >= 0 and 0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError(f"bad lr {lr}, betas {betas}, eps {eps} or weight_decay {weight_decay}")
        self.state_bits, self.capturable = state_bits, bool(capturable)
        self._records, self._captured, self._ahead = {}, {}, {}
        # (the seed is a group's option, so that it is saved and loaded with the others)
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, seed=int(seed)))

    def __getstate__(self):
        return dict(super().__getstate__(), state_bits=self.state_bits, capturable=self.capturable)

    def __setstate__(self, state):
        # a copy has no graph: device records and what a captured step() steps stay with the original
        super().__setstate__(dict(state, _records={}, _captured={}, _ahead={}))

    def add_param_group(self, group):
        super().add_param_group(group)
        for p in self.param_groups[-1]["params"]:
            if p.dtype != torch.float32 or not p.is_contiguous():
                self.param_groups.pop()
                raise ValueError(f"params must be contiguous float32, got {p.dtype} of strides {tuple(p.stride())}")

    def _state(self, p):
        s = self.state[p]
        if not s:
            kind = torch.float32 if self.state_bits == 32 else torch.float8_e4m3fn
            s["step"] = 0
            s["exp_avg"], s["exp_avg_sq"] = (torch.zeros(p.shape, dtype=torch.float32, device=p.device).to(kind) for _ in range(2))
            if self.state_bits == 8:
                s["scales"] = torch.zeros(-(-p.numel() // ADAMW_BLOCK), 2, dtype=torch.float32, device=p.device)
        return s

    def _config(self, i, step):
        g = self.param_groups[i]
        # each group rounds from a stream of its own
        return AdamwConfig(lr=float(g["lr"]), beta1=g["betas"][0], beta2=g["betas"][1], eps=g["eps"], weight_decay=g["weight_decay"], step=step,
                           seed=(g["seed"] + (i << 32)) & (2 ** 64 - 1), state_bits=self.state_bits)

    def _record(self, i, step):
        """Writes the device record of group i for a step."""
        rec = self._records.get(i)
        if rec is None:
            rec = self._records[i] = torch.zeros(C.sizeof(AdamwRecord), dtype=torch.uint8, device=self.param_groups[i]["params"][0].device)
        with ops._on_device(rec.get_device()):
            check(lib().td_adamw_record_set(ptr(rec), C.byref(self._config(i, step)), ops._raw_stream(rec.get_device())))

    def _one_step(self, i, params):
        """The step that all of `params` are at."""
        steps = {self._state(p)["step"] for p in params}
        if len(steps) > 1:
            raise RuntimeError(f"capturable: the params of a group that a captured step() steps must be at the same step, group {i} has {sorted(steps)}")
        return steps.pop()

    def advance(self):
        """capturable: counts one step of the params that the captured step() steps (before a capture: of those that have a gradient, or of
        all where none has) and writes what changes with it (step count, lr, weight decay, seed) to the device records."""
        if not self.capturable:
            raise RuntimeError("advance() belongs to AdamW(capturable=True)")
        todo = []
        for i, g in enumerate(self.param_groups):
            if not g["params"]:
                continue
            for p in g["params"]:
                self._state(p)
            params = self._captured.get(i)
            if params is None:
                params = [p for p in g["params"] if p.grad is not None] or g["params"]
            if params:
                todo.append((i, params, self._one_step(i, params) + 1))
        for i, params, step in todo:
            for p in params:
                self.state[p]["step"] = step
            if i not in self._captured:
                self._ahead.setdefault(i, collections.Counter()).update(map(id, params))
            self._record(i, step)

    def _capture(self):
        """What a captured step() steps from now on: for each group the params with a gradient, all at the same step."""
        for i, g in enumerate(self.param_groups):
            live = [p for p in g["params"] if p.grad is not None]
            if live and (i not in self._records or any(not self.state[p] for p in live)):
                raise RuntimeError("step() under graph capture needs AdamW(capturable=True) and one step() or advance() before the capture")
            if live:
                self._one_step(i, live)
        for i, g in enumerate(self.param_groups):
            self._captured[i] = [p for p in g["params"] if p.grad is not None]
            for p in g["params"]:                # an advance() before this capture may have counted others
                if p.grad is None and i in self._ahead:
                    self.state[p]["step"] -= self._ahead[i][id(p)]
        self._ahead = {}

    @torch.no_grad()
    def step(self, closure=None, *, grad_scale=None):
        """grad_scale: a float32 device scalar that multiplies every gradient (a clipping coefficient, an inverse loss scale)."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        capturing = torch.cuda.is_current_stream_capturing()
        if capturing and not self.capturable:
            raise RuntimeError("step() under graph capture needs AdamW(capturable=True) and one step() or advance() before the capture")
        if capturing:
            self._capture()
        else:
            self._ahead = {}
        for i, group in enumerate(self.param_groups):
            live = [p for p in group["params"] if p.grad is not None]
            for p in live:
                if p.grad.is_sparse:
                    raise RuntimeError("sparse gradients are not supported")
            count = 0 if capturing else 1                    # advance() counts a captured step
            at = {}
            for p in live:
                at.setdefault(self._state(p)["step"] + count, []).append(p)
            for step, ps in sorted(at.items()):
                st = [self.state[p] for p in ps]
                cfg = self._config(i, step)
                adamw_(ps, [p.grad.contiguous() for p in ps], [s["exp_avg"] for s in st], [s["exp_avg_sq"] for s in st],
                       [s["scales"] for s in st] if self.state_bits == 8 else None, lr=cfg.lr, betas=(cfg.beta1, cfg.beta2), eps=cfg.eps,
                       weight_decay=cfg.weight_decay, step=max(step, 1), grad_scale=grad_scale, seed=cfg.seed,
                       record=self._records[i] if capturing else None)
                for s in st:
                    s["step"] = step
            if self.capturable and not capturing and group["params"]:        # what a capture finds: it makes nothing of its own
                self._record(i, max(1, *(self._state(p)["step"] for p in group["params"])))
        return loss

    def load_state_dict(self, state_dict):
        for g in state_dict["param_groups"]:
            for option in ("amsgrad", "maximize"):
                if g.get(option):
                    raise ValueError(f"the state was saved with {option}, which this optimizer does not have")
        for s in state_dict["state"].values():
            if ("scales" in s) != (self.state_bits == 8):
                raise ValueError(f"the state was saved with {8 if 'scales' in s else 32}-bit moments, this optimizer has state_bits={self.state_bits}")
        super().load_state_dict(state_dict)
        for g in self.param_groups:
            g.setdefault("seed", self.defaults["seed"])
        for s in self.state.values():
            s["step"] = int(s["step"])            # torch's own is a tensor
        if self.state_bits == 8:          # torch casts a state to its param's type: float32 holds every e4m3 value, so the way back is exact
            for s in self.state.values():
                s["exp_avg"], s["exp_avg_sq"] = s["exp_avg"].to(torch.float8_e4m3fn), s["exp_avg_sq"].to(torch.float8_e4m3fn)
