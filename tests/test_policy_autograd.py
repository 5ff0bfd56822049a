"""The policy operators beside torch's autograd: what a call overwrites is known to it, and derivatives that an operator
does not have are refused, not dropped."""
import contextlib

import pytest
import torch
from torch.autograd import forward_ad

import isaac_net_amd as P
from isaac_net_amd import policy
from test_gpu_policy import delta_inputs
from test_policy import _OnGpu

DEV = "cuda:0"


@pytest.mark.gpu
@pytest.mark.parametrize("T", [20, 200])
def test_memory_overwritten_before_the_backward_pass_is_noticed(T):
    """delta_rule keeps the state that it was given for its backward pass; a step on the same tensor takes that away."""
    ins, reset, _, _ = delta_inputs(2, T, 1, 2, 32, 32, torch.bfloat16, seed=20)
    x = [t.to(DEV) for t in ins]
    for t in x[:5]:
        t.requires_grad_(True)
    o, _ = P.delta_rule(*x, reset=reset.to(DEV))
    with torch.no_grad():
        P.delta_rule_step(*(t[:, 0] for t in x[:5]), x[5])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.float().sum().backward()


@pytest.mark.gpu
def test_values_overwritten_before_the_backward_pass_are_noticed():
    """The same for a tensor that a step's `out` overwrites."""
    ins, _, _, _ = delta_inputs(2, 1, 1, 2, 32, 32, torch.float32, seed=21)
    x = [t.to(DEV) for t in ins]
    x[0].requires_grad_(True)
    o, _ = P.delta_rule(*x)
    with torch.no_grad():
        P.delta_rule_step(*(t[:, 0].clone() for t in x[:5]), x[5].clone(), out=x[2][:, 0])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()


def test_a_step_that_would_drop_derivatives_is_refused():
    """delta_rule_step has none: in grad mode it takes no tensor that asks for them, and leaves the state as it was."""
    x = [torch.zeros(2, 1, 8), torch.zeros(2, 1, 8), torch.zeros(2, 2, 4), torch.zeros(2, 2), torch.zeros(2, 2)]
    state, out = torch.zeros(2, 2, 8, 4), torch.zeros(2, 2, 4)
    with _OnGpu():
        for t in (*x, state, out):
            t.requires_grad_(True)
            with pytest.raises(P.HipUnsupported, match="derivatives"):
                P.delta_rule_step(*x, state, out=out)
            t.requires_grad_(False)


@pytest.mark.gpu
def test_a_step_without_grad_mode_takes_any_tensor():
    ins, _, _, _ = delta_inputs(2, 1, 1, 2, 32, 32, torch.float32, seed=22)
    x = [t.to(DEV) for t in ins]
    y = [t[:, 0].clone() for t in x[:5]]
    state = x[5].clone()
    want = P.delta_rule_step(*y, state)
    with torch.no_grad():
        got = P.delta_rule_step(*(t.requires_grad_(True) for t in y), x[5])
    assert torch.equal(got, want) and torch.equal(x[5], state) and not got.requires_grad


def test_forward_mode_derivatives_are_refused():
    """A tangent goes through no operator: with one on any input they refuse, in grad mode or not."""
    q, k, v, g, beta = (torch.zeros(2, 3, 1, 8), torch.zeros(2, 3, 1, 8), torch.zeros(2, 3, 2, 4), torch.zeros(2, 3, 2),
                        torch.zeros(2, 3, 2))
    x, w = torch.zeros(3, 8).half(), torch.zeros(5, 8).half()
    y, one = torch.zeros(3, 8), torch.ones(8)
    calls = [(P.delta_rule, dict(q=q, k=k, v=v, g=g, beta=beta, state=torch.zeros(2, 2, 8, 4))),
             (P.delta_rule_step, dict(q=q[:, 0], k=k[:, 0], v=v[:, 0], g=g[:, 0], beta=beta[:, 0],
                                      state=torch.zeros(2, 2, 8, 4), out=torch.zeros(2, 2, 4))),
             (P.gated_ffn, dict(x=x, w_gate=w, w_up=w.clone())),
             (P.block_norm, dict(x=y, f=y.clone(), gate=y.clone(), scale=one, post_weight=one.clone(),
                                 pre_weight=one.clone()))]
    for f, kw in calls:
        for n, t in kw.items():
            for grad in (True, False):
                with _OnGpu() if n == "out" else contextlib.nullcontext(), forward_ad.dual_level(), torch.set_grad_enabled(grad):
                    dual = forward_ad.make_dual(t, torch.ones_like(t))
                    with pytest.raises(P.HipUnsupported, match=f"{n}.*forward-mode"):
                        f(**{**kw, n: dual})


def test_an_output_over_an_input_is_refused():
    """A step's heads are written while others are read: `out` may lie over none of the tensors that the call reads
    (but be v)."""
    buf = torch.zeros(2 * 2 * 8 * 4 + 64)
    x = [torch.zeros(2, 2, 4) for _ in range(3)] + [torch.zeros(2, 2) for _ in range(2)]
    state = buf[:2 * 2 * 4 * 4].view(2, 2, 4, 4)
    with _OnGpu():
        policy._on_gpu = lambda **x: -1               # (what a CPU tensor says of itself)
        for i in range(5):
            y = [t.clone() for t in x]
            y[i] = buf[100:].as_strided(x[i].shape, x[i].stride())
            with pytest.raises(ValueError, match="overlaps"):
                P.delta_rule_step(*y, torch.zeros(2, 2, 4, 4), out=buf[101:117].view(2, 2, 4))
        with pytest.raises(ValueError, match="overlaps"):
            P.delta_rule_step(*x, state, out=buf[60:76].view(2, 2, 4))
        reset = torch.zeros(64, dtype=torch.uint8)
        with pytest.raises(ValueError, match="overlaps"):
            P.delta_rule_step(*x, state, reset=reset[10:12], out=reset.view(torch.float32).view(2, 2, 4))


@pytest.mark.gpu
@pytest.mark.parametrize("H,V", [(2, 32), (3, 128), (1, 5)])
def test_a_step_may_write_its_heads_over_v(H, V):
    ins, _, _, _ = delta_inputs(70, 1, 1, H, 32, V, torch.bfloat16, seed=23)
    x = [t.to(DEV) for t in ins]
    y, states = [t[:, 0].clone() for t in x[:5]], [x[5].clone(), x[5].clone()]
    want = P.delta_rule_step(*y, states[0])
    assert P.delta_rule_step(*y, states[1], out=y[2]) is y[2]
    assert torch.equal(y[2], want) and torch.equal(*states)
