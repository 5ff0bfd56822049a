"""What the policy operators refuse before any launch, at their C entry points and in Python: values out of range."""
import ctypes
import math

import pytest
import torch

import isaac_net_amd as P
from isaac_net_amd import _lib
from test_policy import _OnGpu, lib  # noqa: F401


@pytest.mark.parametrize("eps", [-1e-6, math.nan, -math.inf])
def test_norm_epsilons_below_zero_are_refused(lib, eps):  # noqa: F811
    with _OnGpu(), pytest.raises(ValueError, match="eps"):
        P.block_norm(torch.zeros(3, 8), pre_weight=torch.ones(8), eps=eps)
    n = _lib.InetNorm()
    n.D, n.eps = 8, eps                                   # (no rows: nothing would be launched)
    assert lib.inet_policy_norm_forward(ctypes.byref(n), None) == -1
    n.eps = 0.0
    assert lib.inet_policy_norm_forward(ctypes.byref(n), None) == 0


def test_launches_past_the_grid_are_refused(lib):  # noqa: F811
    """2^32 lanes and more, at sizes that the arguments' own bounds let through. (The pointers are never read.)"""
    d = _lib.InetDelta()
    d.B, d.T, d.Hk, d.H, d.K, d.V = (1 << 24) - 1, 1, 1, 1, 1, 127          # eight blocks of 16 columns a head
    d.q = d.k = d.v = d.g = d.beta = d.o = d.state_out = 16
    assert lib.inet_policy_delta_step(ctypes.byref(d), None) == -2
    n = _lib.InetNorm()
    n.N, n.D, n.x = 1 << 24, 4000, 16                                         # a workgroup a row
    n.pre_weight = n.n = 16
    assert lib.inet_policy_norm_forward(ctypes.byref(n), None) == -2
    f, g = _lib.InetFfn(), _lib.InetFfnGrad()
    f.N, f.D, f.F, f.dtype = 1, 1 << 20, 1 << 20, 1
    f.x = f.w_gate = f.w_up = f.work = g.d_y = g.d_w_gate = 16
    f.x_s = f.w_gate_s = f.w_up_s = 1 << 20
    assert lib.inet_policy_ffn_backward(ctypes.byref(f), ctypes.byref(g), None) == -2


@pytest.mark.gpu
def test_ffn_of_more_than_2_to_the_32_padded_values():
    """An odd width, whose rows are copied first: the last rows of 2^23 as they are alone."""
    gen = torch.Generator().manual_seed(1)
    x, w = (torch.randn(1, 511, generator=gen).bfloat16().cuda() for _ in range(2))
    w = w.expand(8, 511)
    rows = x.expand(1 << 23, 511)
    y = P.gated_ffn(rows, w, w)
    want = P.gated_ffn(x, w, w)
    assert torch.equal(y[-1:], want) and torch.equal(y[:1], want) and bool((y == want).all())


@pytest.mark.gpu
def test_shared_heads_gradients_of_more_than_2_to_the_32_values():
    """2^25 steps of one query and key head of 128 under two value heads (70 GB of their own gradients): the last robot's
    are as those of a few robots."""
    if torch.cuda.mem_get_info()[0] < 120 << 30:
        pytest.skip("needs 120 GiB of free memory")
    gen = torch.Generator().manual_seed(2)
    rand = lambda *s: torch.randn(*s, generator=gen).bfloat16().cuda()  # noqa: E731
    q, k = (t / t.float().norm(dim=-1, keepdim=True).bfloat16() for t in (rand(1, 32, 1, 128), rand(1, 32, 1, 128)))
    v, g, beta, d_o = rand(1, 32, 2, 1), -rand(1, 32, 2).abs(), rand(1, 32, 2).sigmoid(), rand(1, 32, 2, 1)
    got = []
    for B in (1 << 20, 3):
        x = [t.detach().requires_grad_(True) for t in (q, k)]
        x = [t.expand(B, *t.shape[1:]) for t in x]
        o, _ = P.delta_rule(*x, v.expand(B, -1, -1, -1), g.expand(B, -1, -1), beta.expand(B, -1, -1))
        grads = torch.autograd.grad([o], x, [d_o.expand(B, -1, -1, -1)])
        got.append([t[-1].clone() for t in (o, *grads)])
        del o, grads, x
    torch.cuda.empty_cache()
    for a, b in zip(*got):
        assert torch.equal(a, b)
