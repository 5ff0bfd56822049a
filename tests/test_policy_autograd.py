"""The policy operators beside torch's autograd: what a call overwrites is known to it, and derivatives that an operator
does not have are refused, not dropped."""
import pytest
import torch

import isaac_net_amd as P
from test_gpu_policy import delta_inputs

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
