"""A control step captured in the middle of a run (PhysicsRollout.capture_graph) and the memory that a caller keeps for a policy."""

import pytest
import torch
from test_gpu_policy import _rollout, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fused_reset", [True, False])
def test_capturing_in_the_middle_of_a_run_forgets_no_reset(fused_reset):
  """capture_graph() runs a control step of its own: the environments that the step before it reset, and those that it resets, are cut from the caller's memory."""
  kw = dict(fused_reset=fused_reset, control_kernel=fused_reset, episode_length_s=0.2)
  a, b = _rollout(**kw), _rollout(**kw)
  for r in (a, b):  # environments end their episodes of 10 steps at different times
    r.episode_length.copy_(torch.arange(64, device="cuda") % 7)
  p = make(1, obs_dim=a.observation_rows().shape[1], action_dim=a.m.nu)
  mine, other = p.initial_state(64), p.initial_state(64)
  captures = both = 0
  for _ in range(25):
    before = a.step(a.policy_action(p, mine)) != 0
    assert torch.equal(before, b.step(b.policy_action(p, other)) != 0)
    assert torch.equal(mine, other)
    if captures < 5 and before.any():
      captures += 1
      before = before.clone()
      a.capture_graph()
      warm = b.step(torch.zeros((64, b.m.nu), device="cuda")) != 0
      other[:, before] = 0.0
      both += bool((before & ~warm).any() and (warm & ~before).any())
  assert captures == 5 and both and mine.any()
