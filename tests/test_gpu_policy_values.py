"""The policy operators where values are not finite, or where a step between finite ones would not be: a robot whose memory
or inputs went wrong, a norm without an epsilon, gradients larger than their 16-bit type."""
import math

import pytest
import torch

import isaac_net_amd as P
from oracle import policy_oracle as O
from test_gpu_policy import DEV, DT, NAMES, close, delta_both, delta_inputs, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N,D", [(17, 127), (17, 128), (33, 200), (9, 500), (3, 999), (1100, 1032), (9001, 64), (5, 3000)])
def test_norm_without_an_epsilon(dt, N, D):
    """eps = 0: rows past the last, which a workgroup computes along, take no part in the weights' gradients."""
    gen = torch.Generator().manual_seed(30)
    x, f, gate = (rand(gen, N, D).to(DT[dt]) for _ in range(3))
    w = [1 + 0.1 * rand(gen, D) for _ in range(3)]
    d = [rand(gen, N, D).to(DT[dt]) for _ in range(2)]
    got = []
    for fn, dev in ((P.block_norm, DEV), (O.block_norm, "cpu")):
        leaves = [t.to(dev).requires_grad_(True) for t in (x, f, gate, *w)]
        outs = fn(*leaves, eps=0.0)
        got.append([*outs, *torch.autograd.grad(outs, leaves, [e.to(o) for o, e in zip(outs, d)])])
    for n, a, b in zip(("y", "n", "d_x", "d_f", "d_gate", "d_scale", "d_post_weight", "d_pre_weight"), *got):
        close(n, a, b, D + (N if a.dim() == 1 else 0))


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_ffn_passes_nan_on(dt, act):
    """A robot's NaN, or one in a gate projection alone, comes out as one and nowhere else."""
    gen = torch.Generator().manual_seed(31)
    x, wg, wu = rand(gen, 40, 64).to(DT[dt]), rand(gen, 48, 64).to(DT[dt]), rand(gen, 48, 64).to(DT[dt])
    x[3, 5] = math.nan
    wg[7, 9] = math.nan
    with torch.no_grad():
        y = P.gated_ffn(x.to(DEV), wg.to(DEV), wu.to(DEV), activation=act).cpu()
    want = torch.zeros(40, 48, dtype=torch.bool)
    want[3, :] = want[:, 7] = True
    assert torch.equal(torch.isnan(y), want)


def test_gelu_far_out():
    """Gate projections of 2^65 and more, whose square is past 32 bits: the activation is the identity there, or zero."""
    x = torch.tensor([[2.0 ** 40, 1.0]], dtype=torch.bfloat16)
    wg = torch.tensor([[2.0 ** 30, 0.0], [-2.0 ** 30, 0.0], [0.0, 0.5]], dtype=torch.bfloat16)
    wu = torch.tensor([[0.0, 2.0 ** -30]] * 3, dtype=torch.bfloat16)
    got = []
    for f, dev in ((P.gated_ffn, DEV), (O.gated_ffn, "cpu")):
        leaves = [t.to(dev).requires_grad_(True) for t in (x, wg, wu)]
        y = f(*leaves, activation="gelu")
        got.append([y, *torch.autograd.grad([y], leaves, [torch.ones_like(y)])])
    for n, a, b, roundings in zip(("y", "dx", "dw_gate", "dw_up"), *got, (1, 3, 3, 3)):
        close(n, a, b, 5, roundings=roundings)


def close_where_finite(what, x, ref, terms, **kw):
    """As close() where the definition is finite; where it is not, x is not either."""
    ok = torch.isfinite(ref.detach())
    x = x.detach().cpu()
    wrong = (torch.isfinite(x) != ok).sum().item()
    assert not wrong, f"{what}: {wrong} of {ok.numel()} values finite where the definition is not, or the reverse"
    close(what, torch.where(ok, x, torch.zeros_like(x)), torch.where(ok, ref, torch.zeros_like(ref)), terms, **kw)


# the ways through a window: one chunk; several in one pass; few robots by chunks of 32 and, in bfloat16 alone, of 64; rows of
# whole groups of eight on 16 bytes or not; one or several blocks of 64 columns
WAYS = [("f32", 3, 24, 32, 32), ("bf16", 3, 24, 64, 64), ("f16", 3, 31, 40, 72), ("f32", 2, 70, 64, 40),
        ("bf16", 50, 200, 32, 32), ("f16", 2, 70, 100, 17), ("f32", 2, 200, 48, 64), ("bf16", 2, 300, 128, 128),
        ("bf16", 1, 600, 64, 64), ("bf16", 1, 530, 33, 65)]


def outputs_where_finite(ins, reset):
    got = P.delta_rule(*(t.to(DEV) for t in ins), reset=reset.to(DEV))
    want = O.delta_rule(*ins, reset=reset)
    for n, x, y in zip(NAMES, got, want):
        close_where_finite(n, x, y, ins[0].shape[1] + ins[0].shape[3] + ins[2].shape[3])


WRONG = ["state", "state_inf", "q", "k", "v", "v_inf", "g", "beta", "v_column"]


def gone_wrong(dt, B, T, K, V, what):
    """A window of whose robots the first has a memory or inputs that are not finite, its episode ending inside a chunk."""
    ins, reset, d_o, d_s = delta_inputs(B, T, 1, 2, K, V, DT[dt], seed=34, end=0.02)
    end = T - 7 if "state" not in what else 5
    at = end - 6
    reset[0] = False
    reset[0, end] = True
    q, k, v, g, beta, state = ins
    if what == "state":
        state[0, 1] = math.nan
    elif what == "state_inf":
        state[0, 0, 0, 0] = math.inf
    elif what in ("q", "k", "v"):
        {"q": q, "k": k, "v": v}[what][0, at, 0, 3] = math.nan
    elif what == "v_inf":
        v[0, at, 1] = math.inf
    elif what == "g":
        g[0, at, 1] = math.nan
    elif what == "beta":
        beta[0, end - 1, 1] = math.nan                 # the episode's last step: in no later one's equation
    elif what == "v_column":
        v[0, at, :, V - 1] = math.nan
    return ins, reset, d_o, d_s


def history_that_ends(dt, B, T, K, V):
    """The last steps hold no values."""
    ins, reset, d_o, d_s = delta_inputs(B, T, 1, 2, K, V, DT[dt], seed=35, end=0.02)
    for x in ins[:5]:
        x[0, T - 5:] = math.nan
    reset[0, T - 5:] = False
    return ins, reset, d_o, d_s


@pytest.mark.parametrize("what", WRONG)
@pytest.mark.parametrize("dt,B,T,K,V", WAYS)
def test_an_episode_sees_nothing_of_the_one_before(dt, B, T, K, V, what):
    """From the reset on, and in the memory after the window, all is as the recurrence has it, and so are the steps before
    the first wrong one."""
    outputs_where_finite(*gone_wrong(dt, B, T, K, V, what)[:2])


@pytest.mark.parametrize("dt,B,T,K,V", WAYS)
def test_steps_see_nothing_of_later_ones(dt, B, T, K, V):
    outputs_where_finite(*history_that_ends(dt, B, T, K, V)[:2])


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("T", [24, 70, 200, 600])
def test_a_memory_gone_wrong_is_empty_after_its_reset(dt, T):
    """Against the same window from a sound memory: equal outputs from the reset on, up to the order of sums."""
    ins, reset, _, _ = delta_inputs(3, T, 1, 2, 32, 32, DT[dt], seed=37, end=0.02)
    reset[0, :6], reset[0, 5] = False, True
    x = [t.to(DEV) for t in ins]
    o, s = P.delta_rule(*x, reset=reset.to(DEV))
    x[5][0] = math.nan
    o2, s2 = P.delta_rule(*x, reset=reset.to(DEV))
    assert torch.isnan(o2[0, :5]).all() and torch.isfinite(o2[0, 5:]).all() and torch.isfinite(s2).all()
    assert torch.equal(o[1:], o2[1:]) and torch.equal(s[1:], s2[1:])
    close("o", o2[0, 5:], o[0, 5:], T + 64, roundings=2)
    close("state", s2[0], s[0], T + 64)


def check_where_finite(ins, reset, d_o, d_s):
    a, b = delta_both(ins, reset, d_o, d_s)
    T, K, V = ins[0].shape[1], ins[0].shape[3], ins[2].shape[3]
    terms = sum(torch.nan_to_num((ins[i].double() * b[2 + i].double()).sum(-1), 0.0, 0.0, 0.0).norm().item() for i in (0, 1))
    for n, x, y in zip(NAMES, a, b):
        if n == "dg":
            close_where_finite(n, x, y, T + K + V, size=terms,
                               products=0.0 if ins[0].dtype == torch.float32 else 2 * 2.0 ** -16)
        else:
            close_where_finite(n, x, y, T + K + V)


@pytest.mark.parametrize("what", WRONG)
@pytest.mark.parametrize("dt,B,T,K,V", WAYS)
def test_gradients_of_an_episode_see_nothing_of_another(dt, B, T, K, V, what):
    check_where_finite(*gone_wrong(dt, B, T, K, V, what))


@pytest.mark.parametrize("dt,B,T,K,V", WAYS)
def test_gradients_where_a_history_ends(dt, B, T, K, V):
    check_where_finite(*history_that_ends(dt, B, T, K, V))


@pytest.mark.parametrize("what", ["d_o", "d_state"])
@pytest.mark.parametrize("dt,B,T,K,V", WAYS)
def test_a_gradient_stays_in_its_episode(dt, B, T, K, V, what):
    ins, reset, d_o, d_s = delta_inputs(B, T, 1, 2, K, V, DT[dt], seed=36, end=0.02)
    reset[0] = False
    reset[0, T - 9] = True
    if what == "d_o":
        d_o[0, T - 5, 0] = math.nan
    else:
        d_s[0, 0] = math.inf
    check_where_finite(ins, reset, d_o, d_s)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("B,T,K,V", [(3, 24, 64, 64), (2, 33, 32, 40), (40, 70, 128, 128), (2, 200, 100, 64), (2, 600, 64, 128),
                                       (1, 530, 128, 128)])
def test_gates_of_32_bits_have_gradients_of_32_bits(dt, B, T, K, V):
    """dg and dbeta are of the gates' type: beside 16-bit q, k and v they are as exact as those of the same values in
    float32: at most four times their distance, which is the order of sums, of other lengths in chunks of other sizes."""
    ins, reset, d_o, d_s = delta_inputs(B, T, 1, 2, K, V, DT[dt], seed=33, end=0.02, gate_dt=torch.float32)
    narrow, want = delta_both(ins, reset, d_o, d_s)
    wide, _ = delta_both([t.float() for t in ins], reset, d_o.float(), d_s)
    for i in (5, 6):
        off = [(x[i].double().cpu() - want[i]).norm().item() for x in (narrow, wide)]
        assert narrow[i].dtype == torch.float32 and off[0] <= 4 * off[1], (NAMES[i], off, want[i].norm().item())


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("N,D,F", [(20, 32, 48), (33, 7, 50), (300, 72, 136), (2100, 520, 1032)])
@pytest.mark.parametrize("of", ["x", "weights"])
def test_ffn_float16_gradients_through_larger_ones(N, D, F, act, of):
    """The gradients of the projections, up to eight times past 65504, between finite ones: small weights for dx, small
    inputs for those of the weights. (gelu's and silu's gate times its own size: h is a for a > 0.)"""
    gen = torch.Generator().manual_seed(32)
    w_size, x_size = (2.0 ** -9, 2.0 ** 13) if of == "x" else (2.0 ** 7, 2.0 ** -8)
    big = 64.0 * 4096.0 / (w_size * x_size * math.sqrt(D))             # |dy| |h| of 2^18 at |a| of its usual size
    x = (x_size * rand(gen, N, D)).half()
    w = [(w_size * rand(gen, F, D)).half() for _ in range(2)]
    # few robots and columns with such gradients, so that their sums, rounded to float16, are finite
    d = torch.zeros(N, F)
    d[::max(1, N // 8), ::max(1, F // 8)] = big
    d = d.clamp(max=60000.0).half()
    got = []
    for f, dev in ((P.gated_ffn, DEV), (O.gated_ffn, "cpu")):
        leaves = [t.to(dev) for t in (x, *w)]
        want = leaves[:1] if of == "x" else leaves[1:]
        for t in want:
            t.requires_grad_(True)
        y = f(*leaves, activation=act)
        got.append(torch.autograd.grad([y], want, [d.to(y)]))
    for a, b in zip(*got):
        assert b.abs().max() < 65504
        close(of, a, b, F + D if of == "x" else N + D, roundings=3)


@pytest.mark.parametrize("act", ["silu", "relu"])
@pytest.mark.parametrize("N,D,F", [(20, 32, 48), (300, 72, 136), (2100, 520, 1032)])
def test_ffn_float16_gradients_through_smaller_ones(N, D, F, act):
    """The gradients of the projections around 2^-21, where float16 has three bits: those of the weights, of inputs around
    2^6, have all of theirs."""
    gen = torch.Generator().manual_seed(39)
    x = (2.0 ** 6 * rand(gen, N, D)).half()
    w = [(2.0 ** -6 / math.sqrt(D) * rand(gen, F, D)).half() for _ in range(2)]
    d = (2.0 ** -20 * torch.sign(rand(gen, N, F))).half()
    got = []
    for f, dev in ((P.gated_ffn, DEV), (O.gated_ffn, "cpu")):
        leaves = [x.to(dev), *(t.to(dev).requires_grad_(True) for t in w)]
        y = f(*leaves, activation=act)
        got.append(torch.autograd.grad([y], leaves[1:], [d.to(y)]))
    for n, a, b in zip(("dw_gate", "dw_up"), *got):
        close(n, a, b, N + D, roundings=3)
