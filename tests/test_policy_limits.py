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
