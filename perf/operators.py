"""Cases of the decay-attention and AdamW operators: their inputs, their plain form and their work.

Decay attention is the recurrence  S_t = g S_{t-1} + k_t v_t^T,  o_t = scale * S_t^T q_t  with one decay g = exp(log_decay) a
head: over whole sequences (padded or packed), with its gradients, and for single tokens.  AdamW steps a list of tensors
at once, its two moments held in 32 bits or in 8 (e4m3 with one scale for each 256 values, rounded with given random bits).

`run` computes the plain form in elementary torch operations, or, where `own` is true, calls the package's operators.
"""
import math
import random

import torch

own = False

_CHUNK = 64          # rows that the plain form takes as one product
_BLOCK = 256         # values that share a scale in an 8-bit state
_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


# -- cases --------------------------------------------------------------------------------------------------------------------
def _mixer(op, B, T, H, Dk, Dv, dtype, *, Hq=0, Hk=0, Hv=0, packed=False, state=False, fused=False, **kw):
    return dict(op=op, B=B, T=T, H=H, Hq=Hq or H, Hk=Hk or H, Hv=Hv or H, Dk=Dk, Dv=Dv, dtype=dtype, packed=packed, state=state,
                fused=fused, **kw)


def listed():
    return [
        # one token for each of 16 series that are being generated: what counts is the latency of the call
        dict(name="step 16 series", op="step", B=16, H=4, Hq=4, Hk=4, Hv=4, Dk=64, Dv=64, dtype="bfloat16"),
        # the same for a full server: 1024 series with 128 x 128 states, query and key shared by four heads
        dict(name="step 1024 series", op="step", B=1024, H=8, Hq=2, Hk=2, Hv=8, Dk=128, Dv=128, dtype="bfloat16"),
        # a MIMIC-III-shaped batch (24 steps, hidden 92 as four heads of 23) in float32, forward only
        _mixer("forward", 256, 24, 4, 23, 23, "float32", name="forward 256 x 24"),
        # one long prompt whose state is handed to the single-token form
        _mixer("forward", 1, 32768, 16, 128, 128, "bfloat16", state=True, name="prompt 32768"),
        # an eICU-shaped training batch (32 x accumulation 2, 272 steps, hidden 256 as four heads), q | k | v from one projection
        _mixer("train", 64, 272, 4, 64, 64, "bfloat16", fused=True, name="train 64 x 272"),
        # the same at a large batch
        _mixer("train", 2048, 272, 4, 64, 64, "bfloat16", name="train 2048 x 272"),
        # packed series of different lengths with state carried in and out, shared query and key heads, wider values
        _mixer("train", 40, 20011, 8, 64, 128, "bfloat16", Hq=2, Hk=2, packed=True, state=True, name="train packed 20011"),
        # float32 end to end, an odd length
        _mixer("train", 32, 271, 8, 32, 32, "float32", name="train float32 32 x 271"),
        # the time-series classifier's ten tensors: latency
        dict(name="adamw classifier", op="adamw", tensors=10, values=38529, bits=32, grad="float32"),
        # the denoiser's 34 tensors with 8-bit moments
        dict(name="adamw denoiser 8 bits", op="adamw", tensors=34, values=4130000, bits=8, grad="float32"),
        # a wide model with bfloat16 gradients
        dict(name="adamw wide 32 bits", op="adamw", tensors=400, values=64000000, bits=32, grad="bfloat16"),
        # a large one with 8-bit moments
        dict(name="adamw large 8 bits", op="adamw", tensors=120, values=160000000, bits=8, grad="float32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["step", "forward", "train", "train", "adamw"])
    if op == "adamw":
        values = _log_int(rng, 2000, 100_000_000)
        return dict(op=op, tensors=_log_int(rng, 1, 300), values=values, bits=rng.choice([32, 8]), grad=rng.choice(["float32", "bfloat16"]))
    H = rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
    shared = [h for h in range(1, H + 1) if H % h == 0]
    heads = dict(H=H, Hq=H, Hk=H, Hv=H)
    if rng.random() < 0.4:
        heads.update(Hq=rng.choice(shared), Hk=rng.choice(shared), Hv=rng.choice(shared))
    Dk = rng.choice([16, 23, 32, 48, 64, 64, 80, 100, 128])
    Dv = Dk if rng.random() < 0.6 else rng.choice([16, 24, 33, 64, 96, 128])
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    if op == "step":
        return dict(op=op, B=_log_int(rng, 1, max(2, 100_000_000 // (H * Dk * Dv))), Dk=Dk, Dv=Dv, dtype=dtype, **heads)
    packed = rng.random() < 0.4
    rows = _log_int(rng, 1, (400_000 if op == "train" else 500_000) // H)
    if packed:
        B, T = _log_int(rng, 1, max(1, min(200, rows // 4))), rows
    else:
        T = _log_int(rng, 1, min(16384, rows))
        B = max(1, rows // T)
    return dict(op=op, B=B, T=T, Dk=Dk, Dv=Dv, dtype=dtype, packed=packed, state=rng.random() < 0.5,
                fused=not packed and rng.random() < 0.4, **heads)


# -- inputs -------------------------------------------------------------------------------------------------------------------
def _lengths(case, seed):
    """Lengths of a packed case's sequences, an empty one among them; a few rows behind the last one belong to none."""
    r = random.Random(seed)
    rows, B = case["T"], case["B"]
    w = [0.0 if B > 2 and i == B // 2 else math.exp(r.gauss(0.0, 0.8)) for i in range(B)]
    used = max(1, rows - min(7, rows // 50))
    cut, run_, out = sum(w), 0.0, []
    for x in w:
        a = int(run_ / cut * used)
        run_ += x
        out.append(int(run_ / cut * used) - a)
    out[-1] += used - sum(out)
    return out


def _tensor_sizes(case):
    r = random.Random(case["tensors"] * 1000003 + case["values"])
    w = [math.exp(r.uniform(-5.0, 0.0)) for _ in range(case["tensors"])]
    sizes = [max(1, int(case["values"] * x / sum(w))) for x in w]
    sizes[0] = max(1, sizes[0] + case["values"] - sum(sizes))
    return sizes


def _prepare_adamw(case, gen, dev):
    sizes = _tensor_sizes(case)
    align = _BLOCK if case["bits"] == 8 else 1       # 32-bit moments lie next to each other, as in a trainer's flat buffers
    at, total = [], 0
    for n in sizes:
        at.append(total)
        total += -(-n // align) * align
    p = torch.randn(total, generator=gen, device=dev) * 0.05
    g = (torch.randn(total, generator=gen, device=dev) * 1e-3 * (1 + torch.arange(total, device=dev) % 7)).to(_DTYPES[case["grad"]])
    m = torch.randn(total, generator=gen, device=dev) * 1e-3
    r = torch.randn(total, generator=gen, device=dev).abs() * 1e-3 + 1e-4
    views = lambda t: [t[a:a + n] for a, n in zip(at, sizes)]  # noqa: E731
    s = dict(op="adamw", bits=case["bits"], lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, step=37, p=p,
             params=views(p), grads=views(g), grad_scale=torch.full((1,), 0.5, device=dev))
    if case["bits"] == 8:
        blocks = total // _BLOCK
        scales = torch.stack([m.view(blocks, _BLOCK).abs().amax(1), r.view(blocks, _BLOCK).amax(1)], 1) / 448
        m = (m.view(blocks, _BLOCK) / scales[:, :1]).view(-1).to(torch.float8_e4m3fn)
        r = (r.view(blocks, _BLOCK) / scales[:, 1:]).view(-1).to(torch.float8_e4m3fn)
        rnd = torch.randint(-2 ** 31, 2 ** 31, (total,), generator=gen, device=dev, dtype=torch.int32)
        s.update(m=m, v=r, scales=scales, ms=views(m), vs=views(r), random=views(rnd),
                 scale_list=[scales[a // _BLOCK:a // _BLOCK + -(-n // _BLOCK)] for a, n in zip(at, sizes)])
    else:
        v = r * r
        s.update(m=m, v=v, scales=None, ms=views(m), vs=views(v), random=None, scale_list=None)
    return s


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    if case["op"] == "adamw":
        return _prepare_adamw(case, gen, dev)
    dt = _DTYPES[case["dtype"]]
    H, Hq, Hk, Hv, Dk, Dv, B = (case[k] for k in ("H", "Hq", "Hk", "Hv", "Dk", "Dv", "B"))
    # decays from a few rows to thousands of rows
    log_decay = -torch.exp(torch.rand(H, generator=gen, device=dev) * 6.5 - 7.5)
    lead = (B,) if case["op"] == "step" else (case["T"],) if case["packed"] else (B, case["T"])
    if case.get("fused"):
        x = torch.randn(*lead, Hq * Dk + Hk * Dk + Hv * Dv, generator=gen, device=dev).to(dt)
        q, k, v = (t.unflatten(-1, (h, d)) for t, h, d in zip(x.split([Hq * Dk, Hk * Dk, Hv * Dv], -1), (Hq, Hk, Hv), (Dk, Dk, Dv)))
    else:
        q, k, v = (torch.randn(*lead, h, d, generator=gen, device=dev).to(dt) for h, d in ((Hq, Dk), (Hk, Dk), (Hv, Dv)))
    s = dict(op=case["op"], q=q, k=k, v=v, log_decay=log_decay, scale=Dk ** -0.5, offsets=None, state=None)
    if case["op"] == "step":
        s["state"] = torch.randn(B, H, Dk, Dv, generator=gen, device=dev)
        return s
    if case["packed"]:
        n = _lengths(case, seed)
        s["offsets"] = torch.tensor([sum(n[:i]) for i in range(B + 1)], dtype=torch.int32).to(dev)
        s["longest"] = max(n)
    if case["state"]:
        s["state"] = torch.randn(B, H, Dk, Dv, generator=gen, device=dev)
    if case["op"] == "train":
        s["do"] = torch.randn(*lead, H, Dv, generator=gen, device=dev).to(dt)
        s["dstate"] = torch.randn(B, H, Dk, Dv, generator=gen, device=dev) if case["state"] else None
        for name in ("q", "k", "v", "log_decay", "state"):
            if s[name] is not None:
                s[name] = s[name].detach().requires_grad_()
    return s


# -- plain form: decay attention -------------------------------------------------------------------------------------------------
def _power(log_decay, e, factor=False):
    """exp(log_decay * e) (times e) for each head and each entry of the whole-number tensor e."""
    w = torch.exp(log_decay.double().view(-1, *[1] * e.dim()) * e)
    return (w * e if factor else w).float()


def _recur(q, k, v, ld, tangent=False):
    """sum over s <= t of w(t - s) (q_t . k_s) v_s, (N, H, T, D) each, w(d) = g^d, or its derivative d g^d by log g."""
    N, H, T, _ = q.shape
    nc = -(-T // _CHUNK)
    q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, nc * _CHUNK - T)).unflatten(2, (nc, _CHUNK)) for x in (q, k, v))
    i = torch.arange(_CHUNK, device=q.device)
    far = i[:, None] - i[None, :]
    w = torch.where(far >= 0, _power(ld, far.clamp(min=0), tangent), 0.0)
    o = (q @ k.transpose(-1, -2) * w[:, None]) @ v
    if nc > 1:
        c = torch.arange(nc, device=q.device)
        apart = (c[:, None] - 1 - c[None, :]) * _CHUNK
        left = lambda f: torch.where(apart >= 0, _power(ld, apart.clamp(min=0), f), 0.0)  # noqa: E731
        sums = lambda f: ((k * _power(ld, _CHUNK - 1 - i, f)[:, None, :, None]).transpose(-1, -2) @ v).flatten(-2)  # noqa: E731
        into = lambda f: q * _power(ld, i + 1, f)[:, None, :, None]  # noqa: E731
        whole = lambda s: s.unflatten(-1, (q.shape[-1], v.shape[-1]))  # noqa: E731
        U = sums(False)
        F = left(False) @ U
        o = o + into(tangent) @ whole(F)
        if tangent:
            o = o + into(False) @ whole(left(True) @ U + left(False) @ sums(True))
    return o.flatten(2, 3)[:, :, :T]


def _padded(s):
    """Index (N, longest) of each sequence's rows and which of them exist."""
    off = s["offsets"].long()
    t = torch.arange(s["longest"], device=off.device)
    rows = off[:-1, None] + t
    return rows.clamp(max=s["q"].shape[0] - 1), rows < off[1:, None]


def _heads_first(x, heads, place):
    """(rows ..., h, D) in 32 bits as (N, heads, T, D), zero where a padded row does not exist."""
    x = x.detach().float()
    if place is not None:
        x = torch.where(place[1][:, :, None, None], x[place[0]], 0.0)
    return x.repeat_interleave(heads // x.shape[2], 2).transpose(1, 2)


def _rows_back(x, heads, like, s, place):
    """The reverse of _heads_first for an output: heads that share one are summed, rows of no sequence are zero."""
    N, H, T, D = x.shape
    x = x.unflatten(1, (heads, H // heads)).sum(2).transpose(1, 2)
    if place is not None:
        out = torch.zeros(s["q"].shape[0], heads, D, device=x.device)
        out[place[0][place[1]]] = x[place[1]]
        x = out
    return x.to(like.dtype)


def _plain_sequences(s):
    place = None if s["offsets"] is None else _padded(s)
    ld = s["log_decay"].detach()
    H = ld.numel()
    q, k, v = (_heads_first(s[n], H, place) for n in ("q", "k", "v"))
    q = q * s["scale"]
    N, _, T, _ = q.shape
    t = torch.arange(T, device=q.device)
    n = torch.full((N,), T, device=q.device) if place is None else (s["offsets"][1:] - s["offsets"][:-1]).long()
    head = _power(ld, t + 1)[:, :, None]                                    # weight of the entering state in row t
    left = (n[:, None] - 1 - t).clamp(min=0)
    tail = torch.where(t < n[:, None], _power(ld, left), 0.0).transpose(0, 1)[..., None]    # weight of row t in the state left behind
    o = _recur(q, k, v, ld)
    S0 = None if s["state"] is None else s["state"].detach()
    if S0 is not None:
        whole = _power(ld, n).t()[:, :, None, None]
        o = o + (q * head) @ S0
    out = {"o": _rows_back(o, H, s["q"], s, place)}
    if S0 is not None:
        out["state"] = whole * S0 + (k * tail).transpose(-1, -2) @ v
    if s["op"] == "forward":
        return out
    do = _heads_first(s["do"], H, place)
    flip = lambda x: x.flip(2)  # noqa: E731
    dq = _recur(do, v, k, ld)
    dk = flip(_recur(flip(v), flip(do), flip(q), ld))
    dv = flip(_recur(flip(k), flip(q), flip(do), ld))
    slope = _recur(q, k, v, ld, tangent=True)
    dld = 0.0
    if S0 is not None:
        dS = s["dstate"]
        dq = dq + (do * head) @ S0.transpose(-1, -2)
        dk = dk + (v * tail) @ dS.transpose(-1, -2)
        dv = dv + (k * tail) @ dS
        out["dstate"] = (q * head).transpose(-1, -2) @ do + whole * dS
        slope = slope + (q * _power(ld, t + 1, True)[:, :, None]) @ S0
        late = n[:, None, None, None] * whole * S0 + (k * tail * left[:, None, :, None]).transpose(-1, -2) @ v
        dld = (dS * late).sum((0, 2, 3), dtype=torch.float64)
    out["dlog_decay"] = (dld + (do * slope).sum((0, 2, 3), dtype=torch.float64)).float()
    out.update(dq=_rows_back(dq * s["scale"], s["q"].shape[-2], s["q"], s, place), dk=_rows_back(dk, s["k"].shape[-2], s["k"], s, place),
               dv=_rows_back(dv, s["v"].shape[-2], s["v"], s, place))
    return out


def _plain_step(s):
    state, ld = s["state"], s["log_decay"]
    H = ld.numel()
    q, k, v = (s[n].float().repeat_interleave(H // s[n].shape[1], 1) for n in ("q", "k", "v"))
    state.mul_(torch.exp(ld)[:, None, None]).add_(k[..., :, None] * v[..., None, :])
    return {"o": ((q * s["scale"])[..., None, :] @ state).squeeze(-2).to(s["q"].dtype), "state": state}


# -- plain form: AdamW ---------------------------------------------------------------------------------------------------------------
def _round8(x, u, positive):
    """x (blocks, 256) as e4m3 codes and a scale each: the largest magnitude is 448, and a value goes to one of its two
    neighbours as the given u in (0, 1) says.  `positive`: nothing above zero becomes zero."""
    top = x.abs().amax(1, keepdim=True)
    some = top >= 2.0 ** -100
    y = torch.where(some, x.abs() * (448 / top), 0.0).clamp(max=448)
    step = torch.ldexp(torch.ones_like(y), (torch.frexp(y).exponent - 1).clamp(min=-6) - 3)
    c = torch.floor(y / step + u) * step
    if positive:
        c = torch.where((x > 0) & some, c.clamp(min=2.0 ** -9), c)
    return torch.copysign(c, x).to(torch.float8_e4m3fn), torch.where(some, top / 448, 0.0)


def _plain_adamw_one(s, p, g, m_at, v_at, scales=None, rnd=None):
    (b1, b2), t = s["betas"], s["step"]
    g = g.float() * s["grad_scale"]
    n = p.numel()
    if scales is not None:
        blocks = scales.shape[0]
        wide = lambda x: torch.nn.functional.pad(x, (0, blocks * _BLOCK - n)).view(blocks, _BLOCK)  # noqa: E731
        m = (wide(m_at.float()) * scales[:, :1]).view(-1)[:n]
        r = (wide(v_at.float()) * scales[:, 1:]).view(-1)[:n]
        v = r * r
    else:
        m, v = m_at, v_at
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p.mul_(1 - s["lr"] * s["weight_decay"]).sub_(s["lr"] / (1 - b1 ** t) * m / (v.sqrt() / math.sqrt(1 - b2 ** t) + s["eps"]))
    if scales is None:
        m_at.copy_(m)
        v_at.copy_(v)
        return
    bits = wide(rnd)
    u = lambda x: ((x & 0xFFFF).float() + 0.5) / 65536  # noqa: E731
    mc, ms = _round8(wide(m), u(bits), False)
    rc, rs = _round8(wide(v.sqrt()), u(bits >> 16), True)
    m_at.copy_(mc.view(-1)[:n])
    v_at.copy_(rc.view(-1)[:n])
    scales.copy_(torch.cat([ms, rs], 1))


def _adamw_out(s):
    out = {"p": s["p"], "m": s["m"], "v": s["v"]}
    if s["bits"] == 8:
        out["scales"] = s["scales"]
    return out


# -- one pass ------------------------------------------------------------------------------------------------------------------------
def run(state):
    s = state
    if own:
        return _run_own(s)
    if s["op"] == "adamw":
        more = ([], []) if s["bits"] == 32 else (s["scale_list"], s["random"])
        [_plain_adamw_one(s, *a) for a in zip(s["params"], s["grads"], s["ms"], s["vs"], *[x for x in more if x])]
        return _adamw_out(s)
    with torch.no_grad():
        return _plain_step(s) if s["op"] == "step" else _plain_sequences(s)


def _run_own(s):
    if s["op"] == "adamw":
        from timediff_amd.optim import adamw_
        adamw_(s["params"], s["grads"], s["ms"], s["vs"], s["scale_list"], lr=s["lr"], betas=s["betas"], eps=s["eps"],
               weight_decay=s["weight_decay"], step=s["step"], grad_scale=s["grad_scale"], random=s["random"])
        return _adamw_out(s)
    from timediff_amd.decay_attention import decay_attention, decay_attention_step
    if s["op"] == "step":
        return {"o": decay_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], scale=s["scale"]), "state": s["state"]}
    more = dict(scale=s["scale"], offsets=s["offsets"], initial_state=s["state"], return_state=s["state"] is not None)
    if s["op"] == "forward":
        with torch.no_grad():
            got = decay_attention(s["q"], s["k"], s["v"], s["log_decay"], **more)
        return {"o": got[0], "state": got[1]} if s["state"] is not None else {"o": got}
    got = decay_attention(s["q"], s["k"], s["v"], s["log_decay"], **more)
    outs, grads = ([got[0], got[1]], [s["do"], s["dstate"]]) if s["state"] is not None else ([got], [s["do"]])
    names = ["q", "k", "v", "log_decay"] + (["state"] if s["state"] is not None else [])
    d = torch.autograd.grad(outs, [s[n] for n in names], grads)
    out = {"o": outs[0].detach(), **{"d" + n: x for n, x in zip(names, d)}}
    if s["state"] is not None:
        out["state"] = outs[1].detach()
    return out


def work(case):
    if case["op"] == "adamw":
        n, gb = case["values"], 4 if case["grad"] == "float32" else 2
        # parameters and moments are read and written, gradients (and the random bits and scales of 8-bit moments) read
        return {"bytes": n * (24 + gb if case["bits"] == 32 else 12 + gb + 4 + 16 / _BLOCK), "flops": 12.0 * n}
    H, Dk, Dv, B = case["H"], case["Dk"], case["Dv"], case["B"]
    e = 4 if case["dtype"] == "float32" else 2
    rows = B if case["op"] == "step" else case["T"] if case["packed"] else B * case["T"]
    inputs, out = rows * e * ((case["Hq"] + case["Hk"]) * Dk + case["Hv"] * Dv), rows * e * H * Dv
    states = 4.0 * B * H * Dk * Dv
    if case["op"] == "step":
        return {"bytes": inputs + out + 2 * states, "flops": 4.0 * rows * H * Dk * Dv}
    if not case["state"]:
        states = 0
    if case["op"] == "forward":
        return {"bytes": inputs + out + 2 * states, "flops": 4.0 * rows * H * Dk * Dv}
    # forward; then the inputs and the output's gradient read again and three gradients written
    return {"bytes": inputs + out + 2 * inputs + out + 5 * states, "flops": 14.0 * rows * H * Dk * Dv}


# -- 64 bits, from the definition ------------------------------------------------------------------------------------------------------
def _exact_sequence(q, k, v, ld, scale, S0, do, dS, block):
    """One group of sequences of equal length, (G, T, D) in 64 bits with a log decay each (G,): o, S and the gradients, from
    the full matrix of weights, `block` rows at a time."""
    G, T, _ = q.shape
    t = torch.arange(T, device=q.device)
    lam = ld[:, None]
    into, out_of = torch.exp(lam * (t + 1)), torch.exp(lam * (T - 1 - t))
    o = torch.zeros(G, T, v.shape[2], dtype=torch.float64, device=q.device)
    back = None if do is None else [torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros(G, dtype=torch.float64, device=q.device)]
    for a in range(0, T, block):
        b = min(T, a + block)
        far = (t[a:b, None] - t[None, :b]).double()
        w = torch.exp(ld[:, None, None] * far).masked_fill_(far < 0, 0.0) * scale
        A = torch.matmul(q[:, a:b], k[:, :b].transpose(1, 2))
        o[:, a:b] = torch.matmul(A * w, v[:, :b])
        if do is not None:
            dA = torch.matmul(do[:, a:b], v[:, :b].transpose(1, 2))
            back[0][:, a:b] = torch.matmul(dA * w, k[:, :b])
            back[1][:, :b] += torch.matmul((dA * w).transpose(1, 2), q[:, a:b])
            back[2][:, :b] += torch.matmul((A * w).transpose(1, 2), do[:, a:b])
            back[3] += (A * dA * w * far).sum((1, 2))
    S, dS0 = None, None
    if S0 is not None:
        qs = q * scale * into[:, :, None]
        o += torch.matmul(qs, S0)
        S = torch.exp(ld * T)[:, None, None] * S0 + torch.matmul((k * out_of[:, :, None]).transpose(1, 2), v)
    if do is not None and S0 is not None:
        dS0 = torch.matmul(qs.transpose(1, 2), do) + torch.exp(ld * T)[:, None, None] * dS
        back[0] += torch.matmul(do, S0.transpose(1, 2)) * scale * into[:, :, None]
        back[1] += torch.matmul(v, dS.transpose(1, 2)) * out_of[:, :, None]
        back[2] += torch.matmul(k, dS) * out_of[:, :, None]
        back[3] += (torch.matmul(qs * (t + 1)[None, :, None], S0) * do).sum((1, 2))
        late = T * torch.exp(ld * T)[:, None, None] * S0 + torch.matmul((k * (out_of * (T - 1 - t))[:, :, None]).transpose(1, 2), v)
        back[3] += (dS * late).sum((1, 2))
    return o, S, back, dS0


def _exact_sequences(case, s):
    rows_shape = s["q"].shape[:-2]
    H, dev = s["log_decay"].numel(), s["q"].device
    ld = s["log_decay"].detach().double()
    flat = lambda x: x.detach().double().reshape(-1, *x.shape[-2:])  # noqa: E731
    spread = lambda x: flat(x)[:, torch.arange(H, device=dev) // (H // x.shape[-2])]  # noqa: E731
    q, k, v = spread(s["q"]), spread(s["k"]), spread(s["v"])
    do = flat(s["do"]) if case["op"] == "train" else None
    spans = ([(i * case["T"], (i + 1) * case["T"]) for i in range(case["B"])] if s["offsets"] is None
             else list(zip(s["offsets"].tolist()[:-1], s["offsets"].tolist()[1:])))
    res = {"o": torch.zeros(q.shape[0], H, v.shape[2], dtype=torch.float64, device=dev)}
    if s["state"] is not None:
        res["state"] = torch.zeros(len(spans), H, q.shape[2], v.shape[2], dtype=torch.float64, device=dev)
    if do is not None:
        res.update(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v), dlog_decay=torch.zeros_like(ld))
        if s["state"] is not None:
            res["dstate"] = torch.zeros_like(res["state"])
    n = 0
    while n < len(spans):
        T = spans[n][1] - spans[n][0]
        # sequences of one length that follow each other go together, as many as a few GB of weights hold
        most, stop = max(1, int(2.5e8 // max(1, H * T * T))), n + 1
        while stop < len(spans) and stop - n < most and spans[stop][1] - spans[stop][0] == T:
            stop += 1
        g, a, b = stop - n, spans[n][0], spans[stop - 1][1]
        cut = lambda x: x[a:b].reshape(g, T, H, -1).transpose(1, 2).reshape(g * H, T, -1)  # noqa: E731, B023
        put = lambda x: x.reshape(g, H, T, -1).transpose(1, 2).reshape(g * T, H, -1)  # noqa: E731, B023
        one = lambda x: None if x is None else x.detach()[n:stop].double().flatten(0, 1)  # noqa: E731, B023
        o, S, back, dS0 = _exact_sequence(cut(q) if T else q.new_zeros(g * H, 0, q.shape[2]), cut(k) if T else k.new_zeros(g * H, 0, k.shape[2]),
                                          cut(v) if T else v.new_zeros(g * H, 0, v.shape[2]), ld.repeat(g), s["scale"], one(s["state"]),
                                          None if do is None else cut(do) if T else v.new_zeros(g * H, 0, v.shape[2]), one(s.get("dstate")),
                                          max(1, int(5e8 // max(1, g * H * T))))
        if T:
            res["o"][a:b] = put(o)
        if S is not None:
            res["state"][n:stop] = S.unflatten(0, (g, H))
        if back is not None:
            if T:
                for name, x in zip(("dq", "dk", "dv"), back):
                    res[name][a:b] = put(x)
            res["dlog_decay"] += back[3].view(g, H).sum(0)
            if dS0 is not None:
                res["dstate"][n:stop] = dS0.unflatten(0, (g, H))
        n = stop
    for name, x in (("dq", s["q"]), ("dk", s["k"]), ("dv", s["v"])):
        if name in res:
            res[name] = res[name].unflatten(1, (x.shape[-2], H // x.shape[-2])).sum(2).reshape(x.shape)
    res["o"] = res["o"].reshape(*rows_shape, H, -1)
    return res


def _exact_adamw(s):
    (b1, b2), t = s["betas"], s["step"]
    out = {"p": s["p"].double(), "m": s["m"].float().double(), "v": s["v"].float().double()}
    scales = None if s["bits"] == 32 else s["scales"].double()
    base = s["p"].data_ptr()
    for i, p in enumerate(s["params"]):
        a, n = (p.data_ptr() - base) // 4, p.numel()
        at = slice(a, a + n)
        m, v = out["m"][at].clone(), out["v"][at].clone()
        blocks = slice(a // _BLOCK, a // _BLOCK + -(-n // _BLOCK))
        if scales is not None:
            of = torch.arange(n, device=p.device) // _BLOCK
            m, v = m * scales[blocks][of, 0], (v * scales[blocks][of, 1]) ** 2
        g = s["grads"][i].double() * s["grad_scale"].double()
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g ** 2
        step = s["lr"] / (1 - b1 ** t) * m / (torch.sqrt(v / (1 - b2 ** t)) + s["eps"])
        out["p"][at] = out["p"][at] * (1 - s["lr"] * s["weight_decay"]) - step
        if scales is None:
            out["m"][at], out["v"][at] = m, v
            continue
        bits = s["random"][i].long() & 0xFFFFFFFF
        for name, x, u, j in (("m", m, bits % 65536, 0), ("v", torch.sqrt(v), bits // 65536, 1)):
            full = torch.zeros((blocks.stop - blocks.start) * _BLOCK, dtype=torch.float64, device=p.device)
            full[:n] = x.abs()
            top = full.view(-1, _BLOCK).max(1).values
            y = x.abs() / top[of] * 448
            gap = 2.0 ** (torch.floor(torch.log2(y.clamp(min=2.0 ** -6))).clamp(min=-6) - 3)
            low = torch.floor(y / gap + (u.double() + 0.5) / 65536) * gap
            if j:
                low = torch.where(x > 0, low.clamp(min=2.0 ** -9), low)
            out[name][at] = low * torch.sign(x)
            scales[blocks, j] = top / 448
    if scales is not None:
        out["scales"] = scales
    return out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "adamw":
            return _exact_adamw(s)
        if case["op"] == "step":
            H = case["H"]
            q, k, v = (s[n].double().repeat_interleave(H // s[n].shape[1], 1) for n in ("q", "k", "v"))
            S = torch.exp(s["log_decay"].double())[:, None, None] * s["state"].double() + torch.einsum("bhk,bhv->bhkv", k, v)
            return {"o": s["scale"] * torch.einsum("bhk,bhkv->bhv", q, S), "state": S}
        return _exact_sequences(case, s)
