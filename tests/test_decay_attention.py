"""Decay attention without a GPU: what the entry points refuse, and the 64-bit reference against the recurrence it stands for."""
import ctypes as C

import pytest
import torch

import decay_reference as ref
from timediff_amd import _lib
from timediff_amd.decay_attention import decay_attention, decay_attention_step


def _x(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def _call(**kw):
    a = dict(q=_x(2, 5, 2, 8), k=_x(2, 5, 2, 8), v=_x(2, 5, 4, 6), log_decay=_x(4))
    a.update(kw)
    return decay_attention(a.pop("q"), a.pop("k"), a.pop("v"), a.pop("log_decay"), **a)


@pytest.mark.parametrize("bad, error, text", [
    (dict(q=_x(2, 5, 8)), ValueError, "q must have 4 dimensions"),
    (dict(k=_x(2, 5, 2, 8, dtype=torch.bfloat16)), TypeError, "float32 or all bfloat16"),
    (dict(q=_x(2, 5, 2, 8, dtype=torch.float16)), TypeError, "float32 or all bfloat16"),
    (dict(v=_x(2, 4, 4, 6)), ValueError, "leading dimensions"),
    (dict(k=_x(2, 5, 2, 7)), ValueError, "q and k must agree"),
    (dict(q=_x(2, 5, 3, 8)), ValueError, "heads of q"),
    (dict(log_decay=_x(4, dtype=torch.float64)), ValueError, "log_decay must be a float32 vector"),
    (dict(log_decay=_x(0)), ValueError, "heads of q"),
    (dict(v=_x(2, 5, 4, 129)), ValueError, "must be 1 .. 128"),
    (dict(v=_x(2, 5, 4, 0)), ValueError, "must be 1 .. 128"),
    (dict(initial_state=_x(2, 4, 8, 7)), ValueError, "the state must be float32 of shape"),
    (dict(initial_state=_x(2, 4, 8, 6, dtype=torch.bfloat16)), ValueError, "the state must be float32 of shape"),
    (dict(offsets=torch.tensor([0, 5], dtype=torch.int32)), ValueError, "q must have 3 dimensions"),
    (dict(q=_x(5, 2, 8), k=_x(5, 2, 8), v=_x(5, 4, 6), offsets=torch.tensor([0, 5])), ValueError, "offsets must be an int32 vector"),
    (dict(q=_x(5, 2, 8), k=_x(5, 2, 8), v=_x(5, 4, 6), offsets=torch.tensor([0], dtype=torch.int32)), ValueError, "at least 2 entries"),
    (dict(), ValueError, "one ROCm device"),
])
def test_refusals(bad, error, text):
    with pytest.raises(error, match=text):
        _call(**bad)


def test_step_refusals():
    a = dict(q=_x(2, 2, 8), k=_x(2, 2, 8), v=_x(2, 4, 6), log_decay=_x(4), state=_x(2, 4, 8, 6))
    for bad, error, text in [(dict(q=_x(2, 1, 2, 8)), ValueError, "q must have 3 dimensions"), (dict(state=_x(2, 4, 6, 8)), ValueError, "of shape"),
                             (dict(v=_x(3, 4, 6)), ValueError, "leading dimensions"), (dict(), ValueError, "one ROCm device"),
                             (dict(q=_x(2, 2, 8).requires_grad_()), RuntimeError, "no gradient")]:
        with pytest.raises(error, match=text):
            decay_attention_step(**dict(a, **bad))


@pytest.mark.parametrize("field, value, text", [
    ("n_seq", 0, b"n_seq"), ("rows", -1, b"rows"), ("packed", 2, b"packed"), ("dtype", 2, b"dtype"), ("dk", 129, b"dk and dv"), ("dv", 0, b"dk and dv"),
    ("q_heads", 3, b"must divide heads"), ("k_heads", 0, b"must divide heads"), ("heads", 0, b"must divide heads")])
def test_library_refuses_bad_configurations(field, value, text):
    L = _lib.lib()
    cfg = _lib.DecayConfig(n_seq=2, rows=5, heads=4, q_heads=2, k_heads=2, v_heads=4, dk=8, dv=6, dtype=_lib.F32, scale=1.0)
    assert L.td_decay_workspace_bytes(C.byref(cfg), 0) > 0 and L.td_decay_workspace_bytes(C.byref(cfg), 1) > 0
    setattr(cfg, field, value)
    assert L.td_decay_workspace_bytes(C.byref(cfg), 1) == 0 and text in L.td_last_error()
    assert L.td_decay_forward(C.byref(cfg), *[None] * 10) == 1 and text in L.td_last_error()
    assert L.td_decay_backward(C.byref(cfg), *[None] * 15) == 1
    assert L.td_decay_step(C.byref(cfg), *[None] * 7) == 1


def test_library_refuses_null_pointers_and_wrong_forms():
    L = _lib.lib()
    cfg = _lib.DecayConfig(n_seq=2, rows=5, heads=4, q_heads=2, k_heads=2, v_heads=4, dk=8, dv=6, dtype=_lib.F32, scale=1.0)
    some = C.c_void_p(256)            # never dereferenced: the calls below return before any launch
    assert L.td_decay_forward(C.byref(cfg), *[None] * 10) == 1 and b"null pointer" in L.td_last_error()
    assert L.td_decay_forward(C.byref(cfg), some, some, some, some, None, some, some, some, some, None) == 1 and b"same memory" in L.td_last_error()
    assert L.td_decay_backward(C.byref(cfg), *[None] * 15) == 1 and b"null pointer" in L.td_last_error()
    assert L.td_decay_step(C.byref(cfg), some, some, some, some, some, some, None) == 1 and b"one row" in L.td_last_error()
    cfg.packed = 1
    assert L.td_decay_forward(C.byref(cfg), some, some, some, some, None, None, some, None, some, None) == 1 and b"offsets" in L.td_last_error()


def test_workspace_stays_bounded():
    """The states that the backward pass keeps do not grow with the rows: 512 places (packed 1024) of 64 chunks of 128 x 128 (2 or 4 GiB); what does grow are
    the states between segments, one for 4096 rows at least, twice."""
    L = _lib.lib()
    state = 128 * 128 * 4
    for n_seq, rows, heads, packed in ((8, 32768, 64, 0), (1, 2 ** 24, 64, 0), (16, 2 ** 22, 32, 1), (1, 4097, 512, 0)):
        cfg = _lib.DecayConfig(n_seq=n_seq, rows=rows, heads=heads, q_heads=heads, k_heads=heads, v_heads=heads, dk=128, dv=128, dtype=_lib.BF16,
                               packed=packed, scale=1.0)
        slots = (rows // 2048 + n_seq) if packed else n_seq * (rows // 2048 + 1)
        need = L.td_decay_workspace_bytes(C.byref(cfg), 1)
        assert 0 < need <= (1024 if packed else 512) * 64 * state + 2 * slots * heads * (state + 8) + 2048


def test_reference_is_the_recurrence():
    g = torch.Generator().manual_seed(3)
    q, k, v, s0 = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((9, 5), (9, 5), (9, 4), (5, 4)))
    ld = torch.tensor(-0.3, dtype=torch.float64)
    o, s = ref.sequence(q, k, v, ld, 0.7, s0)
    S = s0
    for t in range(9):
        S = torch.exp(ld) * S + k[t][:, None] * v[t][None, :]
        assert torch.allclose(o[t], 0.7 * q[t] @ S, rtol=1e-12, atol=1e-12)
    assert torch.allclose(s, S, rtol=1e-12, atol=1e-12)


def test_rows_are_counted_in_32_bits():
    L = _lib.lib()
    cfg = _lib.DecayConfig(n_seq=1, rows=2 ** 31 - 129, heads=1, q_heads=1, k_heads=1, v_heads=1, dk=1, dv=1, dtype=_lib.BF16, scale=1.0)
    for packed in (0, 1):
        cfg.packed = packed
        assert L.td_decay_workspace_bytes(C.byref(cfg), 0) > 0 and L.td_decay_workspace_bytes(C.byref(cfg), 1) > 0
    cfg.rows += 1
    assert L.td_decay_workspace_bytes(C.byref(cfg), 0) == 0 and b"rows must be" in L.td_last_error()


def test_workspace_is_for_the_gradients_wanted():
    """Fixed decays keep no chunk states (40 packed sequences of 131072 rows in all, 16 heads of 128 x 128: 4 GiB); shared heads have parts in float32
    for the gradients that are asked for."""
    L = _lib.lib()
    cfg = _lib.DecayConfig(n_seq=40, rows=131072, heads=16, q_heads=16, k_heads=16, v_heads=16, dk=128, dv=128, dtype=_lib.BF16, packed=1, scale=1.0)
    need = lambda b: L.td_decay_workspace_bytes(C.byref(cfg), b)  # noqa: E731
    S, Q, K, V, D = _lib.DECAY_GRAD_SOME, _lib.DECAY_GRAD_Q, _lib.DECAY_GRAD_K, _lib.DECAY_GRAD_V, _lib.DECAY_GRAD_LOG_DECAY
    every = need(_lib.DECAY_GRAD_ALL)
    assert every == need(S | Q | K | V | D) == need(S | D) > 4 * 2 ** 30
    state = 16 * 128 * 128 * 4
    assert need(S) == need(S | Q | K | V) <= 2 * (131072 // 4096 + 40) * state + 2048
    cfg.k_heads = cfg.v_heads = 4
    part = 131072 * 16 * 128 * 4
    assert need(S | Q) == need(S) and need(S | K) == need(S | V) == need(S) + part and need(S | K | V) == need(S) + 2 * part
    for bad in (3, 4, 64, 66, -1):
        assert need(bad) == 0 and b"backward must be" in L.td_last_error()


@pytest.mark.parametrize("dk, dv, side", [(8, 128, 64 * 128), (128, 8, 64 * 128), (8, 40, 64 * 64), (24, 24, 32 * 32), (128, 128, 128 * 128), (8, 127, 64 * 128)])
def test_workspace_is_of_the_kernels_own_state(dk, dv, side):
    """64 packed sequences: the chunk states of 1024 workgroups, 64 chunks each, of the state that the kernel for these sizes keeps."""
    L = _lib.lib()
    cfg = _lib.DecayConfig(n_seq=64, rows=262144, heads=16, q_heads=16, k_heads=16, v_heads=16, dk=dk, dv=dv, dtype=_lib.BF16, packed=1, scale=1.0)
    for name, d in (("q", dk), ("k", dk), ("v", dv), ("grad_o", dv)):
        getattr(cfg, name + "_stride")[1:] = [16 * d, d]
    with_slope, without = (L.td_decay_workspace_bytes(C.byref(cfg), b) for b in (_lib.DECAY_GRAD_ALL, _lib.DECAY_GRAD_SOME))
    sums = 2 * (262144 // 4096 + 64) * 16 * 8
    assert with_slope - without == 1024 * 64 * side * 4 + sums
    cfg.rows = cfg.n_seq = cfg.heads = cfg.q_heads = cfg.k_heads = cfg.v_heads = 1        # one workgroup
    with_slope, without = (L.td_decay_workspace_bytes(C.byref(cfg), b) for b in (_lib.DECAY_GRAD_ALL, _lib.DECAY_GRAD_SOME))
    assert with_slope - without == side * 4 + 256


@pytest.mark.parametrize("name", ["q", "k", "v", "log_decay", "initial_state"])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(name, grad):
    """A dual tensor, whether it also takes a gradient or not: its tangent would be dropped.  Without one the call goes on (to the next refusal here)."""
    import torch.autograd.forward_ad as fwd
    a = dict(q=_x(2, 5, 2, 8), k=_x(2, 5, 2, 8), v=_x(2, 5, 4, 6), log_decay=_x(4), initial_state=_x(2, 4, 8, 6))
    with fwd.dual_level():
        with pytest.raises(ValueError, match="one ROCm device"):
            _call(**a)
        dual = fwd.make_dual(a[name].requires_grad_(grad), torch.ones_like(a[name]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            _call(**dict(a, **{name: dual}))
        b = dict(q=a["q"][:, 0], k=a["k"][:, 0], v=a["v"][:, 0], log_decay=a["log_decay"], state=a["initial_state"])
        b = {n: t.detach() for n, t in b.items()}
        n = "state" if name == "initial_state" else name
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            decay_attention_step(**dict(b, **{n: fwd.make_dual(b[n], torch.ones_like(b[n]))}))
