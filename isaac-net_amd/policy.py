"""Operators of a recurrent robot policy beside the engines: the delta-rule memory, the gated feed-forward and the block
norms, as hand-written HIP kernels behind the C ABI of include/inet_policy.h (libinet_policy.so).

A robot is one row of the batch: an engine's E envs x R robots flattened. Between two control steps a policy calls
delta_rule_step (every robot's memory takes one step, in place); to train, it calls delta_rule over a window of steps
from the state that the rollout held, with the envs' episode ends as `reset`. delta_rule, gated_ffn and block_norm take
part in torch's autograd (first derivatives). Every call goes on torch's current stream and returns without waiting;
workspaces come from torch's allocator.

Wrong shapes, types and devices raise ValueError, sizes and types that the kernels do not implement HipUnsupported.
"""
from __future__ import annotations

import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .engine import HipUnsupported

_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = ("silu", "gelu", "relu")          # "gelu" is the tanh form
MAX_HEAD, MAX_WIDTH = 128, 8192


def _need(ok, msg):
    if not ok:
        raise ValueError(msg)


def _code(name, x, of=None):
    if x.dtype not in _CODES:
        raise HipUnsupported(f"{name}: {x.dtype}; float32, bfloat16 and float16 are implemented")
    return _CODES[x.dtype]


def _on_gpu(**xs):
    dev = None
    for n, x in xs.items():
        if x is None:
            continue
        _need(isinstance(x, torch.Tensor), f"{n} has to be a tensor")
        _need(x.is_cuda, f"{n} is on {x.device}: the policy operators run on the GPU")
        _need(dev is None or x.device == dev, f"{n} is on {x.device}, the others on {dev}")
        dev = x.device
    return dev


def _rows(x):
    """x with its last axis contiguous."""
    return x if x.stride(-1) == 1 or x.shape[-1] <= 1 else x.contiguous()


def _ptr(x):
    return None if x is None else x.data_ptr()


def _call(fn, dev, what, *args):
    with torch.cuda.device(dev):
        _lib.check(fn(*args, torch.cuda.current_stream(dev).cuda_stream), what)


# ------------------------------------------------------------------------------------------------ the memory
def _delta_check(q, k, v, g, beta, state, reset, lead):
    dev = _on_gpu(q=q, k=k, v=v, g=g, beta=beta, state=state, reset=reset)
    axes = {1: "[B, heads, size]", 2: "[B, T, heads, size]"}[lead]
    _need(q.dim() == lead + 2 and q.shape == k.shape, f"q and k have to be {axes} of one shape: got {tuple(q.shape)} "
                                                      f"and {tuple(k.shape)}")
    _need(v.dim() == lead + 2 and v.shape[:lead] == q.shape[:lead],
          f"v has to be {axes} over q's batch and steps: got {tuple(v.shape)} with q {tuple(q.shape)}")
    Hk, K, H, V = q.shape[-2], q.shape[-1], v.shape[-2], v.shape[-1]
    _need(Hk > 0 and H > 0 and H % Hk == 0, f"{H} value heads do not share {Hk} query and key heads evenly")
    _need(K > 0 and V > 0, "heads of size 0")
    for n, x in (("g", g), ("beta", beta)):
        _need(tuple(x.shape) == (*v.shape[:lead], H), f"{n} has to be {(*v.shape[:lead], H)}: got {tuple(x.shape)}")
    _need(k.dtype == q.dtype and v.dtype == q.dtype, f"q, k and v have to be of one type: got {q.dtype}, {k.dtype}, "
                                                     f"{v.dtype}")
    _need(g.dtype == beta.dtype, f"g and beta have to be of one type: got {g.dtype}, {beta.dtype}")
    _code("q", q), _code("g", g)
    if K > MAX_HEAD or V > MAX_HEAD:
        raise HipUnsupported(f"heads of {K} x {V}: key and value sizes up to {MAX_HEAD} are implemented")
    if q.shape[0] * H * (-(-q.shape[1] // 32) if lead == 2 else 1) >= 1 << 24:
        raise HipUnsupported(f"{q.shape[0]} robots x {H} heads x {q.shape[1] if lead == 2 else 1} steps: fewer than {1 << 24} robots x heads "
                             "x chunks of 32 steps are implemented")
    if state is not None:
        _need(state.dtype == torch.float32, f"state is held in float32: got {state.dtype}")
        _need(tuple(state.shape) == (q.shape[0], H, K, V), f"state has to be {(q.shape[0], H, K, V)}: got "
                                                          f"{tuple(state.shape)}")
    if reset is not None:
        _need(reset.dtype in (torch.bool, torch.uint8), f"reset has to be bool or uint8: got {reset.dtype}")
        _need(tuple(reset.shape) == tuple(q.shape[:lead]), f"reset has to be {tuple(q.shape[:lead])}: got "
                                                           f"{tuple(reset.shape)}")
    return dev


def _delta_args(q, k, v, g, beta, reset, scale, lead):
    a = _lib.InetDelta()
    a.B, a.T = q.shape[0], (q.shape[1] if lead == 2 else 1)
    a.Hk, a.K, a.H, a.V = q.shape[-2], q.shape[-1], v.shape[-2], v.shape[-1]
    a.dtype, a.gate_dtype, a.scale = _CODES[q.dtype], _CODES[g.dtype], scale
    for n, x in (("q", q), ("k", k), ("v", v), ("g", g), ("beta", beta)):
        s = x.stride()
        setattr(a, n + "_s", (_lib.i64 * 3)(s[0], s[1] if lead == 2 else 0, s[lead]))
        setattr(a, n, x.data_ptr())
    if reset is not None:
        a.reset_s = (_lib.i64 * 2)(reset.stride(0), reset.stride(1) if lead == 2 else 0)
        a.reset = reset.data_ptr()
    return a


def _delta_work(lib, a, dev, backward):
    n = lib.inet_policy_delta_work(C.byref(a), backward)
    work = torch.empty(n, dtype=torch.uint8, device=dev) if n > 0 else None
    a.work = _ptr(work)
    return work


class _DeltaRule(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, state, reset, scale, keep):
        q, k, v = _rows(q), _rows(k), _rows(v)
        if state is not None:
            state = state.contiguous()
        lib = _lib.load_policy()
        B, T, H, V = v.shape
        K = q.shape[-1]
        a = _delta_args(q, k, v, g, beta, reset, scale, 2)
        a.chunk = lib.inet_policy_delta_chunk(T, K, V, a.dtype)
        o = torch.empty(B, T, H, V, dtype=v.dtype, device=v.device)
        out = torch.empty(B, H, K, V, dtype=torch.float32, device=v.device)
        a.state, a.o, a.state_out = _ptr(state), o.data_ptr(), out.data_ptr()
        chunk_state = err = None
        work = _delta_work(lib, a, v.device, 0)
        if keep or work is not None:
            err = torch.empty(B, T, H, V, dtype=torch.float32, device=v.device)
            if T > a.chunk:
                chunk_state = torch.empty(B, H, (T - 1) // a.chunk, K, V, dtype=torch.float32, device=v.device)
            a.chunk_state, a.err = _ptr(chunk_state), err.data_ptr()
        _call(lib.inet_policy_delta_forward, v.device, "delta_rule", C.byref(a))
        if keep:
            ctx.save_for_backward(q, k, v, g, beta, state, reset, chunk_state, err)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return o, out

    @staticmethod
    @once_differentiable
    def backward(ctx, d_o, d_out):
        q, k, v, g, beta, state, reset, chunk_state, err = ctx.saved_tensors
        if d_o is None and d_out is None:
            return (None,) * 9
        lib = _lib.load_policy()
        B, T, H, V = v.shape
        Hk, K = q.shape[-2:]
        a = _delta_args(q, k, v, g, beta, reset, ctx.scale, 2)
        a.chunk = lib.inet_policy_delta_chunk(T, K, V, a.dtype)
        a.state, a.chunk_state, a.err = _ptr(state), _ptr(chunk_state), err.data_ptr()
        work = _delta_work(lib, a, q.device, 1)  # noqa: F841  (held until the call is enqueued)
        new = lambda *s, dtype=q.dtype: torch.empty(*s, dtype=dtype, device=q.device)  # noqa: E731
        d_o = None if d_o is None else d_o.contiguous()
        d_out = None if d_out is None else d_out.contiguous()
        dq, dk, dv = new(B, T, Hk, K), new(B, T, Hk, K), new(B, T, H, V)
        dg, db = new(B, T, H, dtype=g.dtype), new(B, T, H, dtype=g.dtype)
        ds = new(B, H, K, V, dtype=torch.float32) if ctx.needs_input_grad[5] else None
        chunk_grad, err_grad = (None, None) if chunk_state is None else (torch.empty_like(chunk_state),
                                                                         torch.empty_like(err))
        heads = new(2, B, T, H, K, dtype=torch.float32) if H != Hk else None
        d = _lib.InetDeltaGrad(_ptr(d_o), _ptr(d_out), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dg.data_ptr(),
                               db.data_ptr(), _ptr(ds), _ptr(chunk_grad), _ptr(err_grad), _ptr(heads))
        _call(lib.inet_policy_delta_backward, q.device, "delta_rule backward", C.byref(a), C.byref(d))
        return dq, dk, dv, dg, db, ds, None, None, None


def delta_rule(q, k, v, g, beta, state=None, reset=None, scale=None):
    """The gated delta rule over a window of control steps:

        S_t = e^{g_t} S_{t-1} + beta_t k_t (v_t - (e^{g_t} S_{t-1})^T k_t)^T,    o_t = scale S_t^T q_t

    q, k [B, T, Hk, K]; v [B, T, H, V] with Hk dividing H (value head h reads query and key head h // (H // Hk)); g (log-
    decays) and beta (write strengths) [B, T, H], of the type of q or another; state [B, H, K, V] float32, the memory
    before the window (None: empty); reset [B, T] bool or uint8: an episode starts at the step, its memory empty; scale:
    K ** -0.5 by default. Any batch, step and head strides. The recurrence is stable for ||k||^2 beta <= 2: keys are
    usually of unit length and beta in 0 .. 1. A log-decay below -104, whose exponential is 0 in 32 bits, empties the
    memory as reset does.

    Returns (o [B, T, H, V] of v's type, the memory after the window [B, H, K, V] float32)."""
    _delta_check(q, k, v, g, beta, state, reset, 2)
    scale = float(q.shape[-1] ** -0.5 if scale is None else scale)
    keep = torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, v, g, beta, state))
    return _DeltaRule.apply(q, k, v, g, beta, state, reset, scale, keep)


@torch.no_grad()
def delta_rule_step(q, k, v, g, beta, state, reset=None, scale=None, out=None):
    """One control step of the gated delta rule, the memory updated in place: q, k [B, Hk, K], v [B, H, V], g and beta
    [B, H], state [B, H, K, V] float32 contiguous, reset [B] (an emptied memory is empty whatever it held). Returns o
    [B, H, V] (in `out` if given, contiguous of v's type). No derivatives: windows are trained through delta_rule."""
    dev = _delta_check(q, k, v, g, beta, state, reset, 1)
    _need(state is not None and state.is_contiguous(), "state has to be a contiguous tensor: it is updated in place")
    q, k, v = _rows(q), _rows(k), _rows(v)
    if out is None:
        out = torch.empty(v.shape, dtype=v.dtype, device=dev)
    else:
        _need(out.shape == v.shape and out.dtype == v.dtype and out.device == dev and out.is_contiguous(),
              f"out has to be a contiguous {tuple(v.shape)} tensor of {v.dtype} on {dev}")
    a = _delta_args(q, k, v, g, beta, reset, float(q.shape[-1] ** -0.5 if scale is None else scale), 1)
    a.o, a.state_out = out.data_ptr(), state.data_ptr()
    _call(_lib.load_policy().inet_policy_delta_step, dev, "delta_rule_step", C.byref(a))
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


def _ffn_args(x, w_gate, w_up, act):
    a = _lib.InetFfn()
    (a.N, a.D), a.F = x.shape, w_gate.shape[0]
    a.dtype, a.act = _CODES[x.dtype], act
    a.x_s, a.w_gate_s, a.w_up_s, a.y_s = _row_stride(x), _row_stride(w_gate), _row_stride(w_up), a.F
    a.x, a.w_gate, a.w_up = x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr()
    return a


def _ffn_work(lib, a, dev, backward):
    n = lib.inet_policy_ffn_work(a.N, a.D, a.F, backward)
    work = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    a.work = _ptr(work)
    return work


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, act):
        x, w_gate, w_up = _aligned_rows(x), _aligned_rows(w_gate), _aligned_rows(w_up)
        lib = _lib.load_policy()
        y = torch.empty(x.shape[0], w_gate.shape[0], dtype=x.dtype, device=x.device)
        a = _ffn_args(x, w_gate, w_up, act)
        a.y = y.data_ptr()
        work = _ffn_work(lib, a, x.device, 0)  # noqa: F841  (held until the call is enqueued)
        _call(lib.inet_policy_ffn_forward, x.device, "gated_ffn", C.byref(a))
        ctx.save_for_backward(x, w_gate, w_up)
        ctx.act = act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, d_y):
        x, w_gate, w_up = ctx.saved_tensors
        lib = _lib.load_policy()
        d_y = _rows(d_y)
        a = _ffn_args(x, w_gate, w_up, ctx.act)
        new = lambda i, t: torch.empty(t.shape, dtype=t.dtype, device=t.device) if ctx.needs_input_grad[i] else None  # noqa: E731,E501
        dx, dg, du = new(0, x), new(1, w_gate), new(2, w_up)
        d = _lib.InetFfnGrad(d_y.data_ptr(), _row_stride(d_y), _ptr(dx), _ptr(dg), _ptr(du))
        work = _ffn_work(lib, a, x.device, 1)  # noqa: F841
        _call(lib.inet_policy_ffn_backward, x.device, "gated_ffn backward", C.byref(a), C.byref(d))
        return dx, dg, du, None


def gated_ffn(x, w_gate, w_up, activation="silu"):
    """The gated feed-forward: activation(x @ w_gate.T) * (x @ w_up.T) in one kernel, sums in 32 bits.

    x [..., D], w_gate and w_up [F, D] (torch.nn.Linear's layout), all bfloat16 or all float16; activation "silu",
    "gelu" (the tanh form) or "relu". Returns [..., F] of x's type. The backward pass computes the projections again."""
    dev = _on_gpu(x=x, w_gate=w_gate, w_up=w_up)
    _need(activation in ACTIVATIONS, f"activation {activation!r}: one of {ACTIVATIONS}")
    _need(x.dim() >= 1 and w_gate.dim() == 2 and w_gate.shape == w_up.shape and x.shape[-1] == w_gate.shape[1],
          f"x [..., D] with w_gate and w_up [F, D]: got {tuple(x.shape)}, {tuple(w_gate.shape)}, {tuple(w_up.shape)}")
    _need(w_gate.shape[0] > 0 and w_gate.shape[1] > 0, "weights of size 0")
    _need(x.dtype == w_gate.dtype == w_up.dtype, f"x, w_gate and w_up have to be of one type: got {x.dtype}, "
                                                 f"{w_gate.dtype}, {w_up.dtype}")
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise HipUnsupported(f"gated_ffn of {x.dtype}: bfloat16 and float16 are implemented")
    rows = x.reshape(-1, x.shape[-1])
    if rows.shape[0] > 1 << 23:
        raise HipUnsupported(f"gated_ffn of {rows.shape[0]} rows: up to {1 << 23}")
    y = _GatedFfn.apply(rows, w_gate, w_up, ACTIVATIONS.index(activation))
    return y.view(*x.shape[:-1], w_gate.shape[0])


# ------------------------------------------------------------------------------------------------ the norms
def _norm_args(x, f, gate, scale, post, pre, eps):
    a = _lib.InetNorm()
    a.N, a.D = x.shape
    a.dtype, a.eps = _CODES[x.dtype], eps
    a.x, a.x_s = x.data_ptr(), _row_stride(x)
    if f is not None:
        a.f, a.f_s = f.data_ptr(), _row_stride(f)
    if gate is not None:
        a.gate_kind = 2 if gate.shape[1] == x.shape[1] and x.shape[1] > 1 else 1
        a.gate, a.gate_s = gate.data_ptr(), _row_stride(gate)
    a.scale, a.post_weight, a.pre_weight = _ptr(scale), _ptr(post), _ptr(pre)
    return a


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, f, gate, scale, post, pre, eps):
        x = _rows(x)
        f, gate = (None if t is None else _rows(t) for t in (f, gate))
        scale, post, pre = (None if t is None else t.contiguous() for t in (scale, post, pre))
        lib = _lib.load_policy()
        a = _norm_args(x, f, gate, scale, post, pre, eps)
        new = lambda: torch.empty(x.shape, dtype=x.dtype, device=x.device)  # noqa: E731
        y, n = (new() if f is not None else None), (new() if pre is not None else None)
        a.y, a.n = _ptr(y), _ptr(n)
        _call(lib.inet_policy_norm_forward, x.device, "block_norm", C.byref(a))
        ctx.save_for_backward(x, f, gate, scale, post, pre)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        return y, n

    @staticmethod
    @once_differentiable
    def backward(ctx, d_y, d_n):
        x, f, gate, scale, post, pre = ctx.saved_tensors
        if d_y is None and d_n is None:
            return (None,) * 7
        lib = _lib.load_policy()
        a = _norm_args(x, f, gate, scale, post, pre, ctx.eps)
        d_y, d_n = (None if t is None else t.contiguous() for t in (d_y, d_n))
        new = lambda t: None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device)  # noqa: E731
        dx, df, dgate, dscale, dpost, dpre = map(new, (x, f, gate, scale, post, pre))
        work = torch.empty(lib.inet_policy_norm_work(a.N, a.D), dtype=torch.uint8, device=x.device)
        d = _lib.InetNormGrad(*map(_ptr, (d_y, d_n, dx, df, dgate, dscale, dpost, dpre, work)))
        if pre is not None and d_n is None:      # (n took no part: its weight's gradient is zero)
            a.pre_weight = d.d_pre_weight = None
            dpre.zero_()
            if f is None:
                return d_y, None, None, None, None, dpre, None
        _call(lib.inet_policy_norm_backward, x.device, "block_norm backward", C.byref(a), C.byref(d))
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
    _need(x.dim() >= 1 and x.shape[-1] > 0, f"x has to be [..., D]: got {tuple(x.shape)}")
    D = x.shape[-1]
    _code("x", x)
    if D > MAX_WIDTH:
        raise HipUnsupported(f"rows of {D} values: up to {MAX_WIDTH} are implemented")
    for n, t, shapes in (("f", f, (x.shape,)), ("gate", gate, (x.shape, (*x.shape[:-1], 1)))):
        if t is not None:
            _need(tuple(t.shape) in [tuple(s) for s in shapes], f"{n} of {tuple(t.shape)} with x {tuple(x.shape)}")
            _need(t.dtype == x.dtype, f"{n} has to be of x's type {x.dtype}: got {t.dtype}")
    for n, t in (("scale", scale), ("post_weight", post_weight), ("pre_weight", pre_weight)):
        if t is not None:
            _need(tuple(t.shape) == (D,) and t.dtype == torch.float32, f"{n} has to be [{D}] float32: got "
                                                                       f"{tuple(t.shape)} {t.dtype}")
    _need(f is not None or (gate is None and scale is None and post_weight is None),
          "gate, scale and post_weight belong to a block's output f")
    if f is None and pre_weight is None:
        return x, None
    rows = [None if t is None else t.reshape(-1, t.shape[-1]) for t in (x, f, gate)]
    if rows[0].shape[0] > 1 << 24:
        raise HipUnsupported(f"block_norm of {rows[0].shape[0]} rows on {dev}: up to {1 << 24}")
    y, n = _BlockNorm.apply(*rows, scale, post_weight, pre_weight, float(eps))
    return (x if y is None else y.view(x.shape)), (None if n is None else n.view(x.shape))
