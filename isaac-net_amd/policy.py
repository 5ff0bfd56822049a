"""Operators of a recurrent robot policy beside the engines: the delta-rule memory, the gated feed-forward and the block
norms, as hand-written HIP kernels behind the C ABI of include/inet_policy.h (libinet_policy.so).

A robot is one row of the batch: an engine's E envs x R robots flattened. Between two control steps a policy calls
delta_rule_step (every robot's memory takes one step, in place); to train, it calls delta_rule over a window of steps
from the state that the rollout held, with the envs' episode ends as `reset`. delta_rule, gated_ffn and block_norm take
part in torch's autograd (first derivatives, reverse mode). Every call goes on torch's current stream and returns without
waiting; workspaces come from torch's allocator.

Wrong shapes, types and devices raise ValueError, sizes and types that the kernels do not implement HipUnsupported.
"""
from __future__ import annotations

import ctypes as C

import torch
import torch.autograd.graph
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .engine import HipUnsupported

_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = ("silu", "gelu", "relu")          # "gelu" is the tanh form
MAX_HEAD, MAX_WIDTH = 128, 8192
_raw_stream = torch._C._cuda_getCurrentRawStream
_overwritten = torch.autograd.graph.increment_version    # what the kernels write, autograd does not see


def _unsupported_type(name, x):
    return HipUnsupported(f"{name}: {x.dtype}; float32, bfloat16 and float16 are implemented")


def _no_tangents(xs):
    for n, x in xs.items():
        if isinstance(x, torch.Tensor) and forward_ad.unpack_dual(x).tangent is not None:
            raise HipUnsupported(f"{n} has a tangent: the policy operators have no forward-mode derivatives")


def _on_gpu(**xs):
    """The index of the device that all tensors are on."""
    dev = -1
    if forward_ad._current_level >= 0:           # (inside a dual_level)
        _no_tangents(xs)
    for n, x in xs.items():
        if x is None:
            continue
        if not isinstance(x, torch.Tensor):
            raise ValueError(f"{n} has to be a tensor")
        d = x.get_device()
        if d < 0:
            raise ValueError(f"{n} is on {x.device}: the policy operators run on the GPU")
        if dev < 0:
            dev = d
        elif d != dev:
            raise ValueError(f"{n} is on {x.device}, the others on cuda:{dev}")
    return dev


def _rows(x):
    """x with its last axis contiguous."""
    return x if x.stride(-1) == 1 or x.shape[-1] <= 1 else x.contiguous()


def _like(x):
    """A contiguous tensor for x's gradient."""
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _ptr(x):
    return None if x is None else x.data_ptr()


def _span(x):
    """x's first byte and the one past its last."""
    at = x.data_ptr()
    return at, at + (1 + sum((n - 1) * s for n, s in zip(x.shape, x.stride()))) * x.element_size() if x.numel() else at


def _call(fn, dev, what, *args):
    """fn on the device's current stream."""
    if torch.cuda.current_device() == dev:
        rc = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    if rc == -2:                                 # INET_POLICY_EUNSUPPORTED
        raise HipUnsupported(f"{what}: more rows, heads or steps than a launch takes")
    if rc:
        _lib.check(rc, what)


# ------------------------------------------------------------------------------------------------ the memory
def _delta_check(q, k, v, g, beta, state, reset, lead):
    dev = _on_gpu(q=q, k=k, v=v, g=g, beta=beta, state=state, reset=reset)
    qs, vs = q.shape, v.shape
    if len(qs) != lead + 2 or qs != k.shape:
        axes = {1: "[B, heads, size]", 2: "[B, T, heads, size]"}[lead]
        raise ValueError(f"q and k have to be {axes} of one shape: got {tuple(qs)} and {tuple(k.shape)}")
    if len(vs) != lead + 2 or vs[:lead] != qs[:lead]:
        raise ValueError(f"v has to be laid out as q, over its batch and steps: got {tuple(vs)} with q {tuple(qs)}")
    Hk, K, H, V = qs[-2], qs[-1], vs[-2], vs[-1]
    if not (Hk > 0 and H > 0 and H % Hk == 0):
        raise ValueError(f"{H} value heads do not share {Hk} query and key heads evenly")
    if not (K > 0 and V > 0):
        raise ValueError("heads of size 0")
    if g.shape != vs[:-1] or beta.shape != vs[:-1]:
        raise ValueError(f"g and beta have to be {tuple(vs[:-1])}: got {tuple(g.shape)} and {tuple(beta.shape)}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"q, k and v have to be of one type: got {q.dtype}, {k.dtype}, {v.dtype}")
    if g.dtype != beta.dtype:
        raise ValueError(f"g and beta have to be of one type: got {g.dtype}, {beta.dtype}")
    for n, x in (("q", q), ("g", g)):
        if x.dtype not in _CODES:
            raise _unsupported_type(n, x)
    if K > MAX_HEAD or V > MAX_HEAD:
        raise HipUnsupported(f"heads of {K} x {V}: key and value sizes up to {MAX_HEAD} are implemented")
    if qs[0] * H * (-(-qs[1] // 32) if lead == 2 else 1) >= 1 << 24:
        raise HipUnsupported(f"{qs[0]} robots x {H} heads x {qs[1] if lead == 2 else 1} steps: fewer than {1 << 24} "
                             "robots x heads x chunks of 32 steps are implemented")
    if state is not None:
        if state.dtype != torch.float32:
            raise ValueError(f"state is held in float32: got {state.dtype}")
        if state.shape != (qs[0], H, K, V):
            raise ValueError(f"state has to be {(qs[0], H, K, V)}: got {tuple(state.shape)}")
    if reset is not None:
        if reset.dtype not in (torch.bool, torch.uint8):
            raise ValueError(f"reset has to be bool or uint8: got {reset.dtype}")
        if reset.shape != qs[:lead]:
            raise ValueError(f"reset has to be {tuple(qs[:lead])}: got {tuple(reset.shape)}")
    return dev


def _delta_args(q, k, v, g, beta, reset, scale, lead, chunk=0):
    qs, vs = q.shape, v.shape
    if lead == 2:
        st = [x.stride()[:3] for x in (q, k, v, g, beta)]
        rs = (0, 0) if reset is None else reset.stride()
    else:
        st = [(x.stride(0), 0, x.stride(1)) for x in (q, k, v, g, beta)]
        rs = (0 if reset is None else reset.stride(0), 0)
    return _lib.InetDelta(qs[0], qs[1] if lead == 2 else 1, qs[-2], vs[-2], qs[-1], vs[-1], _CODES[q.dtype],
                          _CODES[g.dtype], scale, chunk, *st, rs, q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(),
                          beta.data_ptr(), None if reset is None else reset.data_ptr())


def _delta_work(lib, a, dev, backward):
    n = lib.inet_policy_delta_work(C.byref(a), backward)
    work = torch.empty(n, dtype=torch.uint8, device=dev) if n > 0 else None
    a.work = _ptr(work)
    return work


def _delta_forward(q, k, v, g, beta, state, reset, scale, keep):
    """(o, state, the inputs as read, what the backward pass takes)."""
    q, k, v = _rows(q), _rows(k), _rows(v)
    if state is not None:
        state = state.contiguous()
    lib = _lib.load_policy()
    B, T, H, V = v.shape
    K, dev = q.shape[-1], v.device
    a = _delta_args(q, k, v, g, beta, reset, scale, 2)
    a.chunk = lib.inet_policy_delta_chunk(C.byref(a))
    o = torch.empty((B, T, H, V), dtype=v.dtype, device=dev)
    out = torch.empty((B, H, K, V), dtype=torch.float32, device=dev)
    a.state, a.o, a.state_out = _ptr(state), o.data_ptr(), out.data_ptr()
    chunk_state = err = None
    work = _delta_work(lib, a, dev, 0)
    if keep or work is not None:
        err = torch.empty((B, T, H, V), dtype=torch.float32, device=dev)
        if T > a.chunk:
            chunk_state = torch.empty((B, H, (T - 1) // a.chunk, K, V), dtype=torch.float32, device=dev)
        a.chunk_state, a.err = _ptr(chunk_state), err.data_ptr()
    _call(lib.inet_policy_delta_forward, dev.index, "delta_rule", C.byref(a))
    return o, out, (q, k, v, g, beta, state, reset, chunk_state, err)


class _DeltaRule(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, state, reset, scale):
        o, out, saved = _delta_forward(q, k, v, g, beta, state, reset, scale, True)
        ctx.save_for_backward(*saved)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return o, out

    @staticmethod
    @once_differentiable
    def backward(ctx, d_o, d_out):
        q, k, v, g, beta, state, reset, chunk_state, err = ctx.saved_tensors
        if d_o is None and d_out is None:
            return (None,) * 8
        lib = _lib.load_policy()
        B, T, H, V = v.shape
        K, dev = q.shape[-1], q.device
        a = _delta_args(q, k, v, g, beta, reset, ctx.scale, 2)
        a.chunk = lib.inet_policy_delta_chunk(C.byref(a))
        a.state, a.chunk_state, a.err = _ptr(state), _ptr(chunk_state), err.data_ptr()
        work = _delta_work(lib, a, dev, 1)  # noqa: F841  (held until the call is enqueued)
        d_o = None if d_o is None else d_o.contiguous()
        d_out = None if d_out is None else d_out.contiguous()
        dq, dk, dv, dg, db = map(_like, (q, k, v, g, beta))
        ds = torch.empty((B, H, K, V), dtype=torch.float32, device=dev) if ctx.needs_input_grad[5] else None
        chunk_grad, err_grad = (None, None) if chunk_state is None else (torch.empty_like(chunk_state),
                                                                         torch.empty_like(err))
        heads = torch.empty((2, B, T, H, K), dtype=torch.float32, device=dev) if H != q.shape[-2] else None
        d = _lib.InetDeltaGrad(_ptr(d_o), _ptr(d_out), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dg.data_ptr(),
                               db.data_ptr(), _ptr(ds), _ptr(chunk_grad), _ptr(err_grad), _ptr(heads))
        _call(lib.inet_policy_delta_backward, dev.index, "delta_rule backward", C.byref(a), C.byref(d))
        return dq, dk, dv, dg, db, ds, None, None


def delta_rule(q, k, v, g, beta, state=None, reset=None, scale=None):
    """The gated delta rule over a window of control steps:

        S_t = e^{g_t} S_{t-1} + beta_t k_t (v_t - (e^{g_t} S_{t-1})^T k_t)^T,    o_t = scale S_t^T q_t

    q, k [B, T, Hk, K]; v [B, T, H, V] with Hk dividing H (value head h reads query and key head h // (H // Hk)); g (log-
    decays) and beta (write strengths) [B, T, H], of the type of q or another; state [B, H, K, V] float32, the memory
    before the window (None: empty); reset [B, T] bool or uint8: an episode starts at the step, its memory empty; scale:
    K ** -0.5 by default. Any batch, step and head strides. The recurrence is stable for ||k||^2 beta <= 2: keys are
    usually of unit length and beta in 0 .. 1. A log-decay below -104, whose exponential is 0 in 32 bits, empties the
    memory as reset does: whatever it held or an earlier step was given, NaN included, later steps see nothing of it, nor
    an earlier step's gradient of a later episode's.

    Errors, states and their gradients are of 32-bit grade; o and the other gradients are of their type's (float32 gates
    beside 16-bit q, k and v have gradients of 32-bit grade). The backward pass needs `state` as it was: a
    delta_rule_step on it in between makes it raise.

    Returns (o [B, T, H, V] of v's type, the memory after the window [B, H, K, V] float32)."""
    _delta_check(q, k, v, g, beta, state, reset, 2)
    scale = float(q.shape[-1] ** -0.5 if scale is None else scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or g.requires_grad or
                                    beta.requires_grad or (state is not None and state.requires_grad)):
        return _DeltaRule.apply(q, k, v, g, beta, state, reset, scale)
    return _delta_forward(q, k, v, g, beta, state, reset, scale, False)[:2]


def delta_rule_step(q, k, v, g, beta, state, reset=None, scale=None, out=None):
    """One control step of the gated delta rule, the memory updated in place: q, k [B, Hk, K], v [B, H, V], g and beta
    [B, H], state [B, H, K, V] float32 contiguous, reset [B] (an emptied memory is empty whatever it held). Returns o
    [B, H, V] (in `out` if given, contiguous of v's type: v itself, or over none of the inputs). No derivatives (in grad
    mode an input that requires grad is refused): windows are trained through delta_rule."""
    dev = _delta_check(q, k, v, g, beta, state, reset, 1)
    if state is None or not state.is_contiguous():
        raise ValueError("state has to be a contiguous tensor: it is updated in place")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or g.requires_grad or
                                    beta.requires_grad or state.requires_grad or (out is not None and out.requires_grad)):
        raise HipUnsupported("delta_rule_step has no derivatives: call it under torch.no_grad(), or delta_rule")
    if out is not None and forward_ad._current_level >= 0:
        _no_tangents({"out": out})
    q, k, v = _rows(q), _rows(k), _rows(v)
    if out is None:
        out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    elif out.shape != v.shape or out.dtype != v.dtype or out.get_device() != dev or not out.is_contiguous():
        raise ValueError(f"out has to be a contiguous {tuple(v.shape)} tensor of {v.dtype} on {v.device}")
    else:
        first, end = _span(out)
        for n, x in (("q", q), ("k", k), ("v", v), ("g", g), ("beta", beta), ("state", state), ("reset", reset)):
            # (a wave has read its own values of v before it writes them: v itself may be out)
            if x is None or (n == "v" and x.data_ptr() == first and x.is_contiguous()):
                continue
            at, to = _span(x)
            if at < end and first < to:
                raise ValueError(f"out overlaps {n}: the kernel reads one head's while it writes another's")
    a = _delta_args(q, k, v, g, beta, reset, float(q.shape[-1] ** -0.5 if scale is None else scale), 1)
    a.o, a.state_out = out.data_ptr(), state.data_ptr()
    _call(_lib.load_policy().inet_policy_delta_step, dev, "delta_rule_step", C.byref(a))
    _overwritten((state, out))                   # (a window's backward pass may have been given either to keep)
    return out


# ------------------------------------------------------------------------------------------------ the feed-forward
def _aligned_rows(x):
    """x [rows, D] with its rows contiguous, not too far apart, and on 16 bytes where D holds whole groups of eight."""
    x = _rows(x)
    far = x.shape[0] > 1 and x.stride(0) > 1 << 22
    if far or (x.shape[1] % 8 == 0 and (x.data_ptr() % 16 or (x.shape[0] > 1 and x.stride(0) % 8))):
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def _row_stride(x):
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _ffn_args(x, w_gate, w_up, act, y=None):
    (N, D), F = x.shape, w_gate.shape[0]
    return _lib.InetFfn(N, D, F, _CODES[x.dtype], act, _row_stride(x), _row_stride(w_gate), _row_stride(w_up), F,
                        x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), _ptr(y))


def _ffn_work(lib, a, dev, backward):
    n = lib.inet_policy_ffn_work(a.N, a.D, a.F, backward)
    work = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    a.work = _ptr(work)
    return work


def _ffn_forward(x, w_gate, w_up, act):
    x, w_gate, w_up = _aligned_rows(x), _aligned_rows(w_gate), _aligned_rows(w_up)
    lib, dev = _lib.load_policy(), x.device
    y = torch.empty((x.shape[0], w_gate.shape[0]), dtype=x.dtype, device=dev)
    a = _ffn_args(x, w_gate, w_up, act, y)
    work = _ffn_work(lib, a, dev, 0) if a.D % 8 else None  # noqa: F841  (held until the call is enqueued)
    _call(lib.inet_policy_ffn_forward, dev.index, "gated_ffn", C.byref(a))
    return y, (x, w_gate, w_up)


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, act):
        y, saved = _ffn_forward(x, w_gate, w_up, act)
        ctx.save_for_backward(*saved)
        ctx.act = act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, d_y):
        x, w_gate, w_up = ctx.saved_tensors
        lib, dev = _lib.load_policy(), x.device
        d_y = _rows(d_y)
        a = _ffn_args(x, w_gate, w_up, ctx.act)
        dx, dg, du = (_like(t) if need else None for t, need in zip((x, w_gate, w_up), ctx.needs_input_grad))
        d = _lib.InetFfnGrad(d_y.data_ptr(), _row_stride(d_y), _ptr(dx), _ptr(dg), _ptr(du))
        work = _ffn_work(lib, a, dev, 1)  # noqa: F841
        _call(lib.inet_policy_ffn_backward, dev.index, "gated_ffn backward", C.byref(a), C.byref(d))
        return dx, dg, du, None


def gated_ffn(x, w_gate, w_up, activation="silu"):
    """The gated feed-forward: activation(x @ w_gate.T) * (x @ w_up.T) in one kernel, sums in 32 bits.

    x [..., D], w_gate and w_up [F, D] (torch.nn.Linear's layout), all bfloat16 or all float16; activation "silu",
    "gelu" (the tanh form) or "relu". Returns [..., F] of x's type. The backward pass computes the projections again; their
    gradients are rounded once to x's type before the products over them (float16's scaled into its range as needed)."""
    _on_gpu(x=x, w_gate=w_gate, w_up=w_up)
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation {activation!r}: one of {ACTIVATIONS}")
    xs, ws = x.shape, w_gate.shape
    if len(xs) < 1 or len(ws) != 2 or w_up.shape != ws or xs[-1] != ws[1]:
        raise ValueError(f"x [..., D] with w_gate and w_up [F, D]: got {tuple(xs)}, {tuple(ws)}, {tuple(w_up.shape)}")
    if not (ws[0] > 0 and ws[1] > 0):
        raise ValueError("weights of size 0")
    if not (x.dtype == w_gate.dtype == w_up.dtype):
        raise ValueError(f"x, w_gate and w_up have to be of one type: got {x.dtype}, {w_gate.dtype}, {w_up.dtype}")
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise HipUnsupported(f"gated_ffn of {x.dtype}: bfloat16 and float16 are implemented")
    rows = x if len(xs) == 2 else x.reshape(-1, xs[-1])
    if rows.shape[0] > 1 << 23:
        raise HipUnsupported(f"gated_ffn of {rows.shape[0]} rows: up to {1 << 23}")
    act = ACTIVATIONS.index(activation)
    if torch.is_grad_enabled() and (rows.requires_grad or w_gate.requires_grad or w_up.requires_grad):
        y = _GatedFfn.apply(rows, w_gate, w_up, act)
    else:
        y = _ffn_forward(rows, w_gate, w_up, act)[0]
    return y if len(xs) == 2 else y.view(*xs[:-1], ws[0])


# ------------------------------------------------------------------------------------------------ the norms
def _norm_args(x, f, gate, scale, post, pre, eps, y=None, n=None):
    N, D = x.shape
    kind = 0 if gate is None else 2 if gate.shape[1] == D and D > 1 else 1
    return _lib.InetNorm(N, D, _CODES[x.dtype], kind, eps, _row_stride(x), 0 if f is None else _row_stride(f),
                         0 if gate is None else _row_stride(gate), x.data_ptr(), _ptr(f), _ptr(gate), _ptr(scale),
                         _ptr(post), _ptr(pre), _ptr(y), _ptr(n))


def _norm_forward(x, f, gate, scale, post, pre, eps):
    x = _rows(x)
    f, gate = None if f is None else _rows(f), None if gate is None else _rows(gate)
    scale, post, pre = (None if t is None else t.contiguous() for t in (scale, post, pre))
    y = None if f is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    n = None if pre is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    a = _norm_args(x, f, gate, scale, post, pre, eps, y, n)
    _call(_lib.load_policy().inet_policy_norm_forward, x.device.index, "block_norm", C.byref(a))
    return y, n, (x, f, gate, scale, post, pre)


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, f, gate, scale, post, pre, eps):
        y, n, saved = _norm_forward(x, f, gate, scale, post, pre, eps)
        ctx.save_for_backward(*saved)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        return y, n

    @staticmethod
    @once_differentiable
    def backward(ctx, d_y, d_n):
        x, f, gate, scale, post, pre = ctx.saved_tensors
        if d_y is None and d_n is None:
            return (None,) * 7
        lib, dev = _lib.load_policy(), x.device
        a = _norm_args(x, f, gate, scale, post, pre, ctx.eps)
        d_y, d_n = None if d_y is None else d_y.contiguous(), None if d_n is None else d_n.contiguous()
        dx, df, dgate, dscale, dpost, dpre = (None if t is None else _like(t) for t in (x, f, gate, scale, post, pre))
        work = torch.empty(lib.inet_policy_norm_work(a.N, a.D), dtype=torch.uint8, device=dev)
        d = _lib.InetNormGrad(_ptr(d_y), _ptr(d_n), dx.data_ptr(), _ptr(df), _ptr(dgate), _ptr(dscale), _ptr(dpost),
                              _ptr(dpre), work.data_ptr())
        if pre is not None and d_n is None:      # (n took no part: its weight's gradient is zero)
            a.pre_weight = d.d_pre_weight = None
            dpre.zero_()
        _call(lib.inet_policy_norm_backward, dev.index, "block_norm backward", C.byref(a), C.byref(d))
        return dx, df, dgate, dscale, dpost, dpre, None


def block_norm(x, f=None, gate=None, scale=None, post_weight=None, pre_weight=None, eps=1e-6):
    """The seam between two blocks in one pass: the norm after a block, its gate and residual scale, the residual sum,
    and the norm before the next block.

        y = x + scale * gate * (f / rms(f) * post_weight),    n = y / rms(y) * pre_weight,    rms(z)^2 = mean(z^2) + eps

    x, f [..., D], the residual and the block's output, of one type (float32, bfloat16, float16); gate [..., D] or
    [..., 1] of that type, or None (1); scale, post_weight and pre_weight [D] float32, or None: no scale, f not normed,
    no norm before a next block. f None: no block before (y is x). Sums in 32 bits; n is the norm of y before y is
    rounded. Returns (y, n), n None without pre_weight."""
    dev = _on_gpu(x=x, f=f, gate=gate, scale=scale, post_weight=post_weight, pre_weight=pre_weight)
    xs = x.shape
    if len(xs) < 1 or xs[-1] < 1:
        raise ValueError(f"x has to be [..., D]: got {tuple(xs)}")
    D = xs[-1]
    if x.dtype not in _CODES:
        raise _unsupported_type("x", x)
    if D > MAX_WIDTH:
        raise HipUnsupported(f"rows of {D} values: up to {MAX_WIDTH} are implemented")
    if f is not None and (f.shape != xs or f.dtype != x.dtype):
        raise ValueError(f"f has to be as x, {tuple(xs)} of {x.dtype}: got {tuple(f.shape)} of {f.dtype}")
    if gate is not None and (gate.dtype != x.dtype or (gate.shape != xs and gate.shape != (*xs[:-1], 1))):
        raise ValueError(f"gate has to be {tuple(xs)} or {(*xs[:-1], 1)} of {x.dtype}: got {tuple(gate.shape)} of "
                         f"{gate.dtype}")
    for n, t in (("scale", scale), ("post_weight", post_weight), ("pre_weight", pre_weight)):
        if t is not None and (t.shape != (D,) or t.dtype != torch.float32):
            raise ValueError(f"{n} has to be [{D}] float32: got {tuple(t.shape)} of {t.dtype}")
    if not eps >= 0:
        raise ValueError(f"eps has to be 0 or more: got {eps}")
    if f is None:
        if gate is not None or scale is not None or post_weight is not None:
            raise ValueError("gate, scale and post_weight belong to a block's output f")
        if pre_weight is None:
            return x, None
    flat = len(xs) == 2
    rows = (x, f, gate) if flat else [None if t is None else t.reshape(-1, t.shape[-1]) for t in (x, f, gate)]
    if rows[0].shape[0] > 1 << 24:
        raise HipUnsupported(f"block_norm of {rows[0].shape[0]} rows on cuda:{dev}: up to {1 << 24}")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                       for t in (x, f, gate, scale, post_weight, pre_weight)):
        y, n = _BlockNorm.apply(*rows, scale, post_weight, pre_weight, float(eps))
    else:
        y, n, _ = _norm_forward(*rows, scale, post_weight, pre_weight, float(eps))
    if flat:
        return (x if y is None else y), n
    return (x if y is None else y.view(xs)), (None if n is None else n.view(xs))
