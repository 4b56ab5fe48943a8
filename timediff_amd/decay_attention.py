"""Decay attention: linear attention with one decay per head, beside the recurrent layers.

Per sequence and head, with g = exp(log_decay):  S_t = g S_{t-1} + k_t v_t^T,  o_t = scale * S_t^T q_t.
`decay_attention` runs it over whole sequences (one autograd node: td_decay_forward / td_decay_backward),
`decay_attention_step` over one row of each sequence from the state that `decay_attention(..., return_state=True)` leaves.
No counterpart in the reference.
"""
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import ops


class _DecayFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, state, offsets, scale, want_state):
        o, out = ops.decay_forward(q, k, v, log_decay, scale, offsets, state, want_state)
        ctx.save_for_backward(q, k, v, log_decay, state, offsets)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return o, out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_o, grad_state):
        q, k, v, log_decay, state, offsets = ctx.saved_tensors
        need = ctx.needs_input_grad[:5]
        if grad_o is None and grad_state is None:
            return (None,) * 8
        if grad_o is None:
            grad_o = torch.zeros((), dtype=q.dtype, device=q.device).expand(*q.shape[:-2], log_decay.shape[0], v.shape[-1])
        grads = ops.decay_backward(q, k, v, log_decay, ctx.scale, grad_o, offsets, state, grad_state, want=need)
        return (*grads, None, None, None)


def _no_tangents(*tensors):
    """Refuses forward-mode derivatives: the kernels would drop them."""
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("decay attention has no forward-mode derivatives")


def _claim(node):
    """Marks the nodes that gather the leaves' gradients (in their metadata) with the stream of decay attention's first graph.  Such a node lives as
    long as any graph of its leaf, and a backward pass waits for its stream: under capture that stream would have to be the captured one."""
    stream = torch.cuda.current_stream().cuda_stream
    for leaf, _ in node.next_functions:
        if hasattr(leaf, "variable") and leaf.metadata.setdefault("decay_attention stream", stream) != stream and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("decay_attention under graph capture: a graph of the same leaves, made on another stream, is still alive; drop it "
                               "before the capture (or pass detached leaves)")


def decay_attention(q, k, v, log_decay, *, scale=None, offsets=None, initial_state=None, return_state=False):
    """q (B, T, Hq, Dk), k (B, T, Hk, Dk), v (B, T, Hv, Dv), all float32 or all bfloat16; log_decay (H,) float32, meant to be
    <= 0; Hq, Hk and Hv divide H, and head h uses head h // (H // Hq) of q, and so on  ->  o (B, T, H, Dv) of q's type.
    scale: 1 / sqrt(Dk) by default.
    offsets: (N + 1,) int32 on the same device, non-decreasing: q, k and v are packed rows (R, heads, D), sequence i is rows
    offsets[i] .. offsets[i + 1] - 1 (it may be empty), and o is (R, H, Dv); rows of no sequence come back as zeros and take no
    gradient.  Their values are read on the device when the kernels run.
    initial_state: (B or N, H, Dk, Dv) float32.  return_state: -> (o, state after the last row, the same shape).
    Differentiable once, in backward mode, in q, k, v, log_decay and initial_state.  Any strides with a contiguous last dimension are read in place.
    Rows are computed 64 at a time: a NaN or an infinity in a row's q, k or v may also reach the rows of its 64 before it, so rows that pad
    a dense batch should hold finite values (packed rows of other sequences and of none are never read).  An infinity, of the inputs or of a
    state that overflowed, may come out as NaN.
    A captured backward pass needs leaves of which no graph made on another stream is alive, as torch's own operators do: refused where
    decay_attention made that graph (a graph of other operators alone is not seen here, and the capture fails in torch).
    """
    _no_tangents(q, k, v, log_decay, initial_state)
    ops.decay_check(q, k, v, log_decay, offsets, initial_state)
    scale = float(q.shape[-1] ** -0.5 if scale is None else scale)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, log_decay, initial_state)):
        o, state = _DecayFn.apply(q, k, v, log_decay, initial_state, offsets, scale, return_state)
        _claim(o.grad_fn)
    else:
        o, state = ops.decay_forward(q, k, v, log_decay, scale, offsets, initial_state, return_state)
    return (o, state) if return_state else o


def decay_attention_step(q, k, v, log_decay, state, *, scale=None):
    """One row of each sequence: q (B, Hq, Dk), k (B, Hk, Dk), v (B, Hv, Dv)  ->  o (B, H, Dv); `state` (B, H, Dk, Dv) float32,
    contiguous, is updated in place.  No gradient: under an enabled grad mode, inputs that require one are refused."""
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, log_decay, state)):
        raise RuntimeError("decay_attention_step has no gradient: call it under torch.no_grad(), or decay_attention with initial_state")
    _no_tangents(q, k, v, log_decay, state)
    return ops.decay_step(q, k, v, log_decay, state, float(q.shape[-1] ** -0.5 if scale is None else scale))
