"""The policy operators where values are not finite, or where a step between finite ones would not be: a robot whose memory
or inputs went wrong, a norm without an epsilon, gradients larger than their 16-bit type."""
import math

import pytest
import torch

import isaac_net_amd as P
from oracle import policy_oracle as O
from test_gpu_policy import DEV, DT, close, rand

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
