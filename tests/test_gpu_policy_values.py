"""The policy operators where values are not finite, or where a step between finite ones would not be: a robot whose memory
or inputs went wrong, a norm without an epsilon, gradients larger than their 16-bit type."""
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
