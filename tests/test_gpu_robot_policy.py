"""The example of a policy on an engine (examples/robot_policy.py): the rollout's single steps and the training window
compute the same, the gradient reaches every weight, and an update moves the likelihood the way it should."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("robot_policy", os.path.join(ROOT, "examples", "robot_policy.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def start(example, E=6, R=8, steps=12):
    from isaac_net_amd import scenarios
    torch.manual_seed(5)
    work = scenarios.Workload(E, R, steps, seed=5, device="cuda:0")
    engine = example.P.make_engine("L2", E, R, "cuda:0", work.cfg, seed=5)
    policy = example.RobotPolicy(example.Rollout.ACTIONS).to("cuda:0")
    return example.Rollout(engine, policy, work.poses, episode=5), policy


def test_window_recomputes_the_rollout(example):
    rollout, policy = start(example)
    rollout.window(7)                                    # so that the window starts from memories that hold something
    obs, act, rew, reset, first = rollout.window(12)
    assert reset.any() and not reset.all() and torch.isfinite(rew).all() and torch.isfinite(obs).all()
    logits = policy(obs, first, reset)
    states = [s.clone() for s in first]
    steps = torch.stack([policy.step(obs[:, t], states, reset[:, t]) for t in range(12)], 1)
    # both round the same tensors to bfloat16 (half a last place, 2^-9, of each): a dozen a layer, two layers, which the
    # different order of the 32-bit sums can put either way; 24 of them add up to 24 x 2^-9 at the very most
    assert (logits - steps).norm() <= 24 * 2.0 ** -9 * steps.norm()
    for a, b in zip(states, rollout.states):             # (the same calls on the same inputs)
        assert torch.equal(a, b)


def test_update_raises_the_likelihood_of_what_paid(example):
    rollout, policy = start(example)
    window = rollout.window(12)
    obs, act, rew, reset, first = window
    gain = example.returns(rew, reset)
    gain = (gain - gain.mean()) / (gain.std() + 1e-6)

    def score():
        logp = torch.log_softmax(policy(obs, first, reset), -1)
        return (gain * logp.gather(-1, act[..., None])[..., 0]).mean().item()
    before = score()
    optimizer = torch.optim.SGD(policy.parameters(), lr=0.05)
    for _ in range(4):
        example.update(policy, optimizer, window)
    for n, p in policy.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any(), n
    assert score() > before


def test_returns_stop_at_episode_ends(example):
    rew = torch.tensor([[1.0, 2.0, 4.0]])
    reset = torch.tensor([[False, False, True]])
    assert torch.allclose(example.returns(rew, reset, 0.5), torch.tensor([[2.0, 2.0, 4.0]]))
