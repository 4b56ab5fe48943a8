"""Decay attention in 64 bits on the CPU, from the definition: o_t = scale sum_{s <= t} g^(t-s) (q_t . k_s) v_s + the entering state's
part, one sequence and head at a time, differentiable by torch's autograd.  Used by the tests only."""
import torch


def sequence(q, k, v, log_decay, scale, state):
    """(T, Dk), (T, Dk), (T, Dv), a number, (Dk, Dv) -> (T, Dv), (Dk, Dv), in float64."""
    T = q.shape[0]
    t = torch.arange(T, dtype=torch.float64)
    far = t[:, None] - t[None, :]
    w = torch.where(far >= 0, torch.exp(torch.where(far > 0, log_decay * far, torch.zeros_like(far))), torch.zeros_like(far))
    into, left = torch.exp(log_decay * (t + 1)), torch.where(t < T - 1, torch.exp(torch.where(t < T - 1, log_decay * (T - 1 - t), 0.0 * t)), 1.0)
    o = scale * ((q @ k.T * w) @ v + into[:, None] * (q @ state))
    whole = torch.exp(log_decay * T) if T else torch.ones((), dtype=torch.float64)
    return o, whole * state + (k * left[:, None]).T @ v


def decay_attention(q, k, v, log_decay, scale=None, offsets=None, state=None):
    """The package's arguments, any type, on the CPU -> (o, state) in float64."""
    H, dense = log_decay.shape[0], offsets is None
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    q, k, v = (x.double().repeat_interleave(H // x.shape[-2], -2) for x in (q, k, v))
    ld = log_decay.double()
    spans = [(i, slice(None)) for i in range(q.shape[0])] if dense else [(slice(a, b), None) for a, b in zip(offsets.tolist()[:-1], offsets.tolist()[1:])]
    if state is None:
        state = torch.zeros(len(spans), H, q.shape[-1], v.shape[-1])
    pick = lambda x, s, h: x[s[0], :, h] if dense else x[s[0], h]  # noqa: E731
    got = [[sequence(pick(q, s, h), pick(k, s, h), pick(v, s, h), ld[h], scale, state[n, h].double()) for h in range(H)] for n, s in enumerate(spans)]
    o = [torch.stack([x[0] for x in row], 1) for row in got]
    out = torch.stack([torch.stack([x[1] for x in row]) for row in got]) if got else torch.zeros(0, H, q.shape[-1], v.shape[-1])
    if dense:
        return torch.stack(o), out
    rows = q.shape[0]
    first, last = offsets[0].item(), offsets[-1].item()
    return torch.cat([torch.zeros(first, H, v.shape[-1], dtype=torch.float64), *o, torch.zeros(rows - last, H, v.shape[-1], dtype=torch.float64)]), out


def gradients(q, k, v, log_decay, grad_o, grad_state=None, **kw):
    """-> {name: gradient in float64} of sum(o grad_o) + sum(state grad_state), by autograd on the definition."""
    leaves = {n: x.detach().double().requires_grad_() for n, x in (("q", q), ("k", k), ("v", v), ("log_decay", log_decay))}
    if kw.get("state") is not None:
        leaves["state"] = kw["state"].detach().double().requires_grad_()
        kw = dict(kw, state=leaves["state"])
    o, s = decay_attention(leaves["q"], leaves["k"], leaves["v"], leaves["log_decay"], **kw)
    loss = (o * grad_o.double()).sum() + (0.0 if grad_state is None else (s * grad_state.double()).sum())
    if not loss.requires_grad:
        return {n: torch.zeros_like(x) for n, x in leaves.items()}
    return {n: (torch.zeros_like(x) if g is None else g) for (n, x), g in zip(leaves.items(), torch.autograd.grad(loss, list(leaves.values()), allow_unused=True))}
