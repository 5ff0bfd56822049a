"""The policy operators on the GPU (delta_rule, delta_rule_step, gated_ffn, block_norm) against their definitions in 64
bits (oracle/policy_oracle.py) on the same inputs, their derivatives against the definitions' and against differences, and
the sizes, layouts and values at which they can go wrong.

Tolerances, as the 2-norm of the difference over the 2-norm of the value. A result rounded once to a type is off by at most
half a unit in the last place of every element: u = 2^-8 (bfloat16, 8 significand bits), 2^-11 (float16), 2^-24
(float32). Sums and states are held in 32 bits: n roundings of 2^-24 in a row are off by at most n 2^-24 of the terms'
size, n the window's steps plus the two sizes of a head (delta rule), or the row's length (norms); four times that covers
the products of such factors and the gradients' sums. Where a gradient's terms are themselves rounded to 16 bits
(gated_ffn's da and du) it may be off by u more for each of the two.

Two gradients are differences of larger terms, and may be off by those shares of the terms' size, not of their own: the
log-decays' (sums over the following steps of q . dq and k . dk; for keys that are all alike and written in full they
cancel down to the rounding of the keys' length), where the 16-bit types' products drop 2^-16 of each of their two
factors; and that of a norm's input in a row of one value, whose norm is its sign.

Differences are taken along the gradient's signs, so that the loss changes by the sum of its magnitudes; what they leave
out is the third derivative's share, the step squared over 6 times a ratio of the order of one to ten for steps of at most
2^-6 of inputs of size one: under 1 %."""
import math

import pytest
import torch

import isaac_net_amd as P
from oracle import policy_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def close(what, x, ref, terms, roundings=1, size=0.0, products=0.0):
    """size: the 2-norm of the terms, where they cancel; products: the share of it that a product may drop"""
    x, ref, u = x.detach().double().cpu(), ref.detach().double().cpu(), U[x.dtype]
    assert x.shape == ref.shape and torch.isfinite(x).all(), what
    n = ref.norm().item()
    off, tol = (x - ref).norm().item(), 1.01 * roundings * u * n + (4 * terms * 2.0 ** -24 + products) * max(n, size)
    assert off <= tol, f"{what}: off by {off:.3g}, {tol:.3g} allowed ({n:.3g} large)"


def rand(gen, *s):
    return torch.randn(*s, generator=gen)


def delta_inputs(B, T, Hk, H, K, V, dt, seed=0, end=0.1, alike=0.7, gate_dt=None):
    gen = torch.Generator().manual_seed(seed)
    unit = lambda x: x / (x.norm(dim=-1, keepdim=True) + 1e-6)  # noqa: E731
    q = unit(rand(gen, B, T, Hk, K)).to(dt)
    k = unit(rand(gen, B, T, Hk, K) + alike * rand(gen, B, 1, Hk, K)).to(dt)
    v = rand(gen, B, T, H, V).to(dt)
    g = (-torch.exp(2.0 * rand(gen, B, T, H) - 2.0)).to(gate_dt or dt)
    beta = torch.sigmoid(rand(gen, B, T, H)).to(gate_dt or dt)
    state = 0.5 * rand(gen, B, H, K, V)
    reset = torch.rand(B, T, generator=gen) < end
    d_o, d_s = rand(gen, B, T, H, V).to(dt), 0.3 * rand(gen, B, H, K, V)
    return [q, k, v, g, beta, state], reset, d_o, d_s


def delta_both(ins, reset, d_o, d_s, scale=None):
    """(GPU outputs and gradients, the definition's)"""
    got = []
    for f, dev in ((P.delta_rule, DEV), (O.delta_rule, "cpu")):
        x = [None if t is None else t.to(dev).requires_grad_(True) for t in ins]
        o, s = f(*x, reset=None if reset is None else reset.to(dev), scale=scale)
        heads, grads = [o, s], [d_o.to(dev), d_s.to(dev)]
        if dev == "cpu":
            grads = [y.double() for y in grads]
        leaves = [t for t in x if t is not None]
        got.append([o, s] + list(torch.autograd.grad(heads, leaves, grads)))
    return got


NAMES = ("o", "state", "dq", "dk", "dv", "dg", "dbeta", "dstate")


def check_delta(ins, reset, d_o, d_s, scale=None):
    a, b = delta_both(ins, reset, d_o, d_s, scale)
    T, K, V = ins[0].shape[1], ins[0].shape[3], ins[2].shape[3]
    terms = sum((ins[i].double() * b[2 + i].double()).sum(-1).norm().item() for i in (0, 1))
    for n, x, y in zip(NAMES, a, b):
        if n == "dg":
            close(n, x, y, T + K + V, size=terms, products=0.0 if ins[0].dtype == torch.float32 else 2 * 2.0 ** -16)
        else:
            close(n, x, y, T + K + V)
    return a


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,T,Hk,H,K,V", [
    (3, 1, 1, 1, 16, 16), (2, 15, 2, 2, 32, 32), (2, 32, 1, 2, 64, 64), (3, 33, 2, 2, 64, 64), (2, 64, 1, 3, 40, 56),
    (1, 65, 2, 2, 128, 128), (2, 127, 1, 1, 96, 24), (1, 200, 2, 4, 64, 128), (2, 70, 1, 2, 7, 13), (1, 40, 1, 1, 1, 1),
    (2, 50, 2, 2, 65, 33), (1, 129, 1, 1, 128, 17)])
def test_window(dt, B, T, Hk, H, K, V):
    check_delta(*delta_inputs(B, T, Hk, H, K, V, DT[dt]))


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,T,Hk,H,K,V", [
    (1, 161, 1, 2, 32, 24), (2, 530, 1, 1, 48, 64), (1, 577, 1, 2, 128, 96), (1, 1025, 1, 1, 24, 72),  # a few robots
    (40, 70, 1, 3, 32, 40), (33, 130, 3, 3, 64, 64), (20, 100, 5, 5, 100, 128)])                       # many
def test_window_of_several_chunks(dt, B, T, Hk, H, K, V):
    check_delta(*delta_inputs(B, T, Hk, H, K, V, DT[dt], seed=16, end=0.02))


@pytest.mark.parametrize("dt,gate", [("bf16", "f32"), ("f32", "bf16"), ("f16", "f32")])
def test_window_gates_of_another_type(dt, gate):
    check_delta(*delta_inputs(2, 75, 1, 2, 48, 32, DT[dt], gate_dt=DT[gate]))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("case", ["no_reset", "every_step", "no_state", "beta0", "g0", "g_minus_inf", "g_lowest", "alike",
                                  "strong_decay"])
def test_window_values(dt, case):
    ins, reset, d_o, d_s = delta_inputs(2, 70, 1, 2, 32, 48, DT[dt], seed=3)
    g, beta = ins[3], ins[4]
    if case == "no_reset":
        reset = None
    elif case == "every_step":
        reset[:] = True
    elif case == "no_state":
        ins[5] = None
    elif case == "beta0":
        beta[:, ::3] = 0.0
    elif case == "g0":
        g[:] = 0.0
    elif case == "g_minus_inf":
        g[:, 11] = -math.inf
    elif case == "g_lowest":
        g[:, 11] = torch.finfo(g.dtype).min
    elif case == "alike":                  # a robot that stands still: the same key at every step, written in full
        ins[1][:] = ins[1][:, :1].clone()
        beta[:] = 1.0
    elif case == "strong_decay":
        g[:, 5::7] = -60.0
    check_delta(ins, reset, d_o, d_s)


@pytest.mark.parametrize("dt,B,T", [("f32", 3, 70), ("f32", 3, 20), ("bf16", 3, 200), ("bf16", 3, 600), ("f16", 50, 200)])
def test_window_emptied_memory_is_empty(dt, B, T):
    """Whatever the state held, an episode that starts at the window's first step sees none of it, in either direction."""
    ins, reset, d_o, d_s = delta_inputs(B, T, 1, 2, 32, 32, DT[dt], seed=4)
    reset[0, 0] = True
    ins[5][0] = math.nan
    a, b = delta_both([*ins[:5], torch.nan_to_num(ins[5], nan=0.0)], reset, d_o, d_s)
    c, _ = delta_both(ins, reset, d_o, d_s)
    for n, x, y in zip(NAMES, c, a):
        assert torch.equal(x, y), n


@pytest.mark.parametrize("T", [20, 90, 200])
@pytest.mark.parametrize("used", ["o", "state"])
def test_window_one_output_used(T, used):
    ins, reset, d_o, d_s = delta_inputs(2, T, 1, 2, 32, 48, torch.float32, seed=14, end=0.02)
    (d_s if used == "o" else d_o).zero_()
    want = delta_both(ins, reset, d_o, d_s)[1]
    x = [t.to(DEV).requires_grad_(True) for t in ins]
    o, s = P.delta_rule(*x, reset=reset.to(DEV))
    got = torch.autograd.grad([o if used == "o" else s], x, [(d_o if used == "o" else d_s).to(DEV)], allow_unused=True)
    for n, a, b in zip(NAMES[2:], got, want[2:]):
        terms = sum((ins[i].double() * want[2 + i].double()).sum(-1).norm().item() for i in (0, 1))
        close(n, torch.zeros_like(b) if a is None else a, b, T + 80, size=terms if n == "dg" else 0.0)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_window_layouts(dt):
    """Views of one projection, step-major storage, a last axis that is not contiguous, rows off the 16-byte grid."""
    B, T, H, K, V = 2, 45, 2, 32, 32
    ins, reset, d_o, d_s = delta_inputs(B, T, H, H, K, V, DT[dt], seed=5)
    want = [x.to(DEV) for x in delta_both(ins, reset, d_o, d_s)[0]]

    def run(q, k, v, g, beta, reset):
        x = [t.detach().requires_grad_(True) for t in (q, k, v, g, beta, ins[5].to(DEV))]
        o, s = P.delta_rule(*x, reset=reset)
        got = [o, s, *torch.autograd.grad([o, s], x, [d_o.to(DEV).transpose(1, 2).contiguous().transpose(1, 2),
                                                      d_s.to(DEV)])]
        for n, a, b in zip(NAMES, got, want):
            assert torch.equal(a, b), n
    q, k, v, g, beta = (x.to(DEV) for x in ins[:5])
    r = reset.to(DEV)
    fused = torch.cat([q, k, v], -1)
    run(fused[..., :K], fused[..., K:2 * K], fused[..., 2 * K:], g, beta, r)
    run(*(x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v, g, beta)), r.t().contiguous().t())
    run(*(x.transpose(2, 3).contiguous().transpose(2, 3) for x in (q, k, v)), g, beta, r.to(torch.uint8))

    def odd(x):
        y = torch.empty(*x.shape[:-1], x.shape[-1] + 3, dtype=x.dtype, device=DEV)[..., 1:x.shape[-1] + 1]
        return y.copy_(x)
    run(odd(q), odd(k), odd(v), odd(g), odd(beta), r)


def test_window_gradient_against_differences():
    ins, reset, d_o, d_s = delta_inputs(2, 40, 1, 2, 16, 16, torch.float32, seed=6)
    got = delta_both(ins, reset, d_o, d_s)[0][2:]
    x = [t.to(DEV) for t in ins]
    loss = lambda y: sum((a.double() * b.to(DEV).double()).sum().item()  # noqa: E731
                         for a, b in zip(P.delta_rule(*y, reset=reset.to(DEV)), (d_o, d_s)))
    h = 2.0 ** -8
    for i, n in enumerate(NAMES[2:]):
        step = got[i].sign()
        diff = (loss([t + h * step if j == i else t for j, t in enumerate(x)]) -
                loss([t - h * step if j == i else t for j, t in enumerate(x)])) / (2 * h)
        want = got[i].double().abs().sum().item()
        assert abs(diff - want) <= 0.01 * want, n


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,Hk,H,K,V", [(1, 1, 1, 1, 1), (5, 2, 2, 32, 32), (3, 1, 3, 64, 64), (7, 2, 4, 128, 128),
                                        (4, 1, 1, 17, 5), (3, 1, 2, 128, 66), (2, 1, 1, 40, 24), (2, 1, 1, 100, 16)])
def test_step(dt, B, Hk, H, K, V):
    ins, reset, _, _ = delta_inputs(B, 3, Hk, H, K, V, DT[dt], seed=7, end=0.3)
    want_o, want_s = O.delta_rule(*ins, reset=reset)
    state = ins[5].to(DEV).clone()
    for t in range(3):
        q, k, v, g, beta = (x[:, t].to(DEV) for x in ins[:5])       # views over the steps
        o = P.delta_rule_step(q, k, v, g, beta, state, reset=reset[:, t].to(DEV))
        close(f"o at {t}", o, want_o[:, t], 3 + K)
    close("state", state, want_s, 3 + K)


def test_step_agrees_with_window():
    ins, reset, _, _ = delta_inputs(6, 20, 2, 2, 64, 64, torch.float32, seed=8)
    x = [t.to(DEV) for t in ins]
    o, s = P.delta_rule(*x, reset=reset.to(DEV))
    state = x[5].clone()
    out = torch.empty(6, 2, 64, device=DEV)
    for t in range(20):
        y = P.delta_rule_step(*(a[:, t] for a in x[:5]), state, reset=reset[:, t].to(DEV), out=out)
        assert y is out
        close("o", y, o[:, t], 20 + 64)
    close("state", state, s, 20 + 64)


def test_step_emptied_memory_is_empty():
    ins, _, _, _ = delta_inputs(3, 1, 1, 1, 32, 32, torch.float32, seed=9)
    x = [t[:, 0].to(DEV) for t in ins[:5]]
    state = torch.full((3, 1, 32, 32), math.nan, device=DEV)
    o = P.delta_rule_step(*x, state, reset=torch.ones(3, dtype=torch.bool, device=DEV))
    z = torch.zeros(3, 1, 32, 32, device=DEV)
    assert torch.equal(o, P.delta_rule_step(*x, z)) and torch.equal(state, z)


def test_step_offsets_past_32_bits():
    """A state of more than 2^31 elements: its last robots are computed as they are alone."""
    B, H, K, V = 263000, 2, 64, 64
    assert B * H * K * V > 2 ** 31
    state = torch.zeros(B, H, K, V, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(1)
    q, k, v = (torch.randn(B, H, 64, device=DEV, generator=gen).mul_(0.1).bfloat16() for _ in range(3))
    g, beta = (torch.rand(B, H, device=DEV, generator=gen).bfloat16() for _ in range(2))
    state[-5:] = torch.randn(5, H, K, V, device=DEV, generator=gen)
    few = state[-5:].clone()
    o = P.delta_rule_step(q, k, v, -g, beta, state)
    assert torch.equal(o[-5:], P.delta_rule_step(q[-5:], k[-5:], v[-5:], -g[-5:], beta[-5:], few))
    assert torch.equal(state[-5:], few)


@pytest.mark.parametrize("B,T", [(0, 5), (3, 0)])
def test_window_of_nothing(B, T):
    ins, reset, d_o, d_s = delta_inputs(max(B, 1), max(T, 1), 1, 2, 16, 16, torch.float32)
    x = [t[:B, :T].to(DEV).requires_grad_(True) for t in ins[:5]] + [ins[5][:B].to(DEV).requires_grad_(True)]
    o, s = P.delta_rule(*x, reset=reset[:B, :T].to(DEV))
    assert o.shape == (B, T, 2, 16) and torch.equal(s, x[5])
    grads = torch.autograd.grad([o, s], x, [d_o[:B, :T].to(DEV), d_s[:B].to(DEV)])
    assert torch.equal(grads[5], d_s[:B].to(DEV)) and all(y.shape == z.shape for y, z in zip(grads, x))


# ------------------------------------------------------------------------------------------------ the feed-forward
def ffn_both(N, D, F, dt, act, seed=0):
    gen = torch.Generator().manual_seed(seed)
    ins = [rand(gen, N, D).to(dt), (rand(gen, F, D) / math.sqrt(D)).to(dt), (rand(gen, F, D) / math.sqrt(D)).to(dt)]
    d_y = rand(gen, N, F).to(dt)
    got = []
    for f, dev in ((P.gated_ffn, DEV), (O.gated_ffn, "cpu")):
        x = [t.to(dev).requires_grad_(True) for t in ins]
        y = f(*x, activation=act)
        got.append([y, *torch.autograd.grad([y], x, [d_y.to(y)])])
    return got


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("N,D,F,act", [
    (1, 8, 8, "silu"), (5, 64, 128, "gelu"), (127, 120, 136, "relu"), (128, 128, 128, "silu"), (129, 136, 264, "gelu"),
    (300, 100, 77, "silu"), (1030, 512, 344, "silu"), (33, 1, 1, "gelu"), (64, 65, 130, "relu"), (2100, 64, 72, "silu")])
def test_ffn(dt, N, D, F, act):
    a, b = ffn_both(N, D, F, DT[dt], act)
    close("y", a[0], b[0], D)
    for n, x, y, terms in zip(("dx", "dw_gate", "dw_up"), a[1:], b[1:], (F + D, N + D, N + D)):
        close(n, x, y, terms, roundings=3)


def test_ffn_layouts():
    gen = torch.Generator().manual_seed(2)
    x, wg, wu = rand(gen, 3, 50, 64).bfloat16().to(DEV), rand(gen, 96, 64).bfloat16().to(DEV), \
        rand(gen, 96, 64).bfloat16().to(DEV)
    want = P.gated_ffn(x, wg, wu)
    assert want.shape == (3, 50, 96)
    both = torch.cat([wg, wu], 1)                                    # halves of one matrix: rows 128 apart
    assert torch.equal(P.gated_ffn(x, both[:, :64], both[:, 64:]), want)
    assert torch.equal(P.gated_ffn(x.transpose(0, 2).contiguous().transpose(0, 2), wg.t().contiguous().t(), wu), want)
    odd = torch.empty(96, 67, dtype=torch.bfloat16, device=DEV)[:, 1:65].copy_(wg)
    assert torch.equal(P.gated_ffn(x, odd, wu), want)
    assert P.gated_ffn(x[:, :0], wg, wu).shape == (3, 0, 96)


def test_ffn_no_rows_gradient():
    w = torch.randn(16, 8, device=DEV).bfloat16().requires_grad_(True)
    y = P.gated_ffn(torch.empty(0, 8, dtype=torch.bfloat16, device=DEV), w, w.detach())
    assert torch.equal(torch.autograd.grad(y.sum(), w)[0], torch.zeros_like(w))


def test_ffn_gradient_against_differences():
    """Along the float16 values that the moved inputs round to, the loss in 64 bits."""
    gen = torch.Generator().manual_seed(3)
    x, w = rand(gen, 200, 32).half().to(DEV), [(rand(gen, 48, 32) / 6).half().to(DEV) for _ in range(2)]
    d = rand(gen, 200, 48).half().to(DEV)
    leaves = [t.requires_grad_(True) for t in (x, *w)]
    grads = torch.autograd.grad([P.gated_ffn(*leaves)], leaves, [d])
    loss = lambda y: (P.gated_ffn(*y).double() * d.double()).sum().item()  # noqa: E731
    with torch.no_grad():
        for i in range(3):
            step = grads[i].sign() * 2.0 ** -6
            hi, lo = (leaves[i] + step).half(), (leaves[i] - step).half()
            diff = loss([hi if j == i else t for j, t in enumerate(leaves)]) - \
                loss([lo if j == i else t for j, t in enumerate(leaves)])
            want = (grads[i].double() * (hi.double() - lo.double())).sum().item()
            assert abs(diff - want) <= 0.01 * want, i


# ------------------------------------------------------------------------------------------------ the norms
def norm_both(N, D, dt, gate="full", f=True, scale=True, post=True, pre=True, seed=0, dy=True, dn=True):
    gen = torch.Generator().manual_seed(seed)
    ins = {"x": 2 * rand(gen, N, D).to(dt), "f": 3 * rand(gen, N, D).to(dt) if f else None,
           "gate": {"full": lambda: torch.sigmoid(rand(gen, N, D)).to(dt),
                    "row": lambda: torch.sigmoid(rand(gen, N, 1)).to(dt), None: lambda: None}[gate](),
           "scale": 0.3 + 0.1 * rand(gen, D) if scale else None, "post_weight": 1 + 0.1 * rand(gen, D) if post else None,
           "pre_weight": 1 + 0.1 * rand(gen, D) if pre else None}
    d = [rand(gen, N, D).to(dt), rand(gen, N, D).to(dt)]
    got = []
    for fn, dev in ((P.block_norm, DEV), (O.block_norm, "cpu")):
        x = {n: None if t is None else t.to(dev).requires_grad_(True) for n, t in ins.items()}
        outs = fn(**x)
        pairs = [(o, e.to(o)) for o, e, used in zip(outs, d, (dy, dn)) if o is not None and used]
        leaves = {n: t for n, t in x.items() if t is not None}
        grads = torch.autograd.grad([o for o, _ in pairs], list(leaves.values()), [e for _, e in pairs],
                                    allow_unused=True)
        got.append({**dict(zip("yn", outs)), **{"d_" + n: t for n, t in zip(leaves, grads)}})
    return got[0], got[1], ins, d


def check_norm(N, D, *args, **kw):
    a, b, ins, d = norm_both(N, D, *args, **kw)
    for n in b:
        if b[n] is None or a[n] is None:
            assert a[n] is None or not a[n].any(), n      # (a zero gradient may come as one)
            continue
        size = 0.0
        if D == 1 and n in ("d_x", "d_f"):
            size = ((d[0].double().abs() + d[1].double().abs()) * 2 / (ins["f"] if n == "d_f" else b["y"]).double().abs()
                    ).norm().item()
        close(n, a[n], b[n], D + (N if n.startswith("d_") and a[n].shape == (D,) else 0), size=size)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N,D", [(1, 1), (3, 8), (17, 127), (33, 128), (5, 200), (9, 256), (70, 500), (6, 512), (5, 999),
                                 (4, 1024), (7, 1111), (600, 1032), (9, 1536), (6, 1704), (3, 2048), (3, 4000), (2, 8192), (2100, 64)])
def test_norm(dt, N, D):
    check_norm(N, D, DT[dt])


@pytest.mark.parametrize("kw", [dict(gate="row"), dict(gate=None), dict(scale=False), dict(post=False), dict(pre=False),
                                dict(pre=False, post=False, scale=False, gate=None), dict(dn=False), dict(dy=False),
                                dict(f=False, gate=None, scale=False, post=False)])
@pytest.mark.parametrize("dt,D", [("f32", 96), ("bf16", 333)])
def test_norm_parts(dt, D, kw):
    check_norm(40, D, DT[dt], **kw)


def test_norm_layouts_and_empty_rows():
    gen = torch.Generator().manual_seed(1)
    x, f = rand(gen, 4, 30, 64).to(DEV), rand(gen, 4, 30, 64).to(DEV)
    gate, w = torch.sigmoid(rand(gen, 4, 30, 1)).to(DEV), torch.ones(64, device=DEV)
    f[1, 3] = 0.0                                                   # a block that gave nothing
    y, n = P.block_norm(x, f, gate=gate, post_weight=w, pre_weight=w)
    assert torch.equal(y[1, 3], x[1, 3]) and torch.isfinite(n).all()
    xf = torch.cat([x, f], -1)
    y2, n2 = P.block_norm(xf[..., :64], xf[..., 64:], gate=gate, post_weight=w, pre_weight=w)
    assert torch.equal(y, y2) and torch.equal(n, n2)
    y3, _ = P.block_norm(x.transpose(0, 1), f.transpose(0, 1), gate=gate.transpose(0, 1), post_weight=w, pre_weight=w)
    assert torch.equal(y3, y.transpose(0, 1))
    assert P.block_norm(x[:0], f[:0], pre_weight=w)[1].shape == (0, 30, 64)
    w0 = w.clone().requires_grad_(True)
    assert not torch.autograd.grad(P.block_norm(x[:0], pre_weight=w0)[1].sum(), w0)[0].any()


def test_norm_gradient_against_differences():
    gen = torch.Generator().manual_seed(5)
    ins = [rand(gen, 20, 48).to(DEV), rand(gen, 20, 48).to(DEV), rand(gen, 20, 48).to(DEV), rand(gen, 48).to(DEV),
           rand(gen, 48).to(DEV), rand(gen, 48).to(DEV)]
    d = [rand(gen, 20, 48).to(DEV) for _ in range(2)]
    leaves = [t.requires_grad_(True) for t in ins]
    grads = torch.autograd.grad(P.block_norm(*leaves), leaves, d)
    loss = lambda z: sum((a.double() * b.double()).sum().item() for a, b in zip(P.block_norm(*z), d))  # noqa: E731
    with torch.no_grad():
        for i in range(6):
            step, h = grads[i].sign(), 2.0 ** -9
            diff = (loss([t + h * step if j == i else t for j, t in enumerate(ins)]) -
                    loss([t - h * step if j == i else t for j, t in enumerate(ins)])) / (2 * h)
            want = grads[i].double().abs().sum().item()
            assert abs(diff - want) <= 0.01 * want, i


def test_too_many_rows_are_refused():
    x = torch.zeros(1, 8, dtype=torch.bfloat16, device=DEV).expand((1 << 24) + 1, 8)
    with pytest.raises(P.HipUnsupported, match="block_norm"):
        P.block_norm(x, pre_weight=torch.ones(8, device=DEV))
    with pytest.raises(P.HipUnsupported, match="gated_ffn"):
        P.gated_ffn(x, x[:8], x[:8])
    q = torch.zeros(1, 1, 1, 1, device=DEV).expand(1 << 24, 1, 1, 1)
    with pytest.raises(P.HipUnsupported, match="robots x heads x chunks"):
        P.delta_rule(q, q, q, q[..., 0], q[..., 0])


# ------------------------------------------------------------------------------------------------ as a user runs them
def test_twice_the_same_and_another_stream():
    """Results do not vary from run to run, nor on a stream of the caller's."""
    ins, reset, d_o, d_s = delta_inputs(4, 70, 1, 3, 64, 64, torch.bfloat16, seed=11)
    a, _ = delta_both(ins, reset, d_o, d_s)
    f = ffn_both(700, 64, 72, torch.bfloat16, "silu")[0]
    n = norm_both(3000, 96, torch.float32)[0]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        b, _ = delta_both(ins, reset, d_o, d_s)
        f2 = ffn_both(700, 64, 72, torch.bfloat16, "silu")[0]
        n2 = norm_both(3000, 96, torch.float32)[0]
    s.synchronize()
    for x, y in [*zip(a, b), *zip(f, f2), *((n[m], n2[m]) for m in n)]:
        assert torch.equal(x, y)


def test_rollout_in_a_graph():
    """A rollout's step recorded once and replayed, the engine's own graphs aside: every replay equals the eager call."""
    gen = torch.Generator().manual_seed(12)
    B, H, D = 64, 2, 32
    x = rand(gen, B, H * D).bfloat16().to(DEV)
    w = [(rand(gen, 96, H * D) / 8).bfloat16().to(DEV) for _ in range(2)]
    q, k, v = (rand(gen, B, H, D).mul(0.2).bfloat16().to(DEV) for _ in range(3))
    g, beta = -torch.rand(B, H, generator=gen).to(DEV), torch.rand(B, H, generator=gen).to(DEV)
    one = torch.ones(H * D, device=DEV)
    state, eager = torch.zeros(B, H, D, D, device=DEV), torch.zeros(B, H, D, D, device=DEV)
    reset = torch.zeros(B, dtype=torch.bool, device=DEV)

    def step(st):
        o = P.delta_rule_step(q, k, v, g, beta, st, reset=reset)
        y, n = P.block_norm(x, o.view(B, H * D), post_weight=one, pre_weight=one)
        return y, P.gated_ffn(n, *w)
    with torch.no_grad():
        step(torch.zeros_like(state))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(state)
        state.zero_()
        for i in range(5):
            reset.copy_(torch.arange(B, device=DEV) % 5 == i)
            x.add_(0.125)
            graph.replay()
            want = step(eager)
            torch.cuda.synchronize()
            assert torch.equal(state, eager) and all(torch.equal(a, b) for a, b in zip(out, want)), i
