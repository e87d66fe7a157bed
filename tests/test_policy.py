"""mjlab_amd/policy.py without a GPU: what a policy is made of, and what it refuses."""

import math

import pytest
import torch

from mjlab_amd.policy import Policy, PolicyCfg


@pytest.mark.parametrize("kw", [
  dict(obs_dim=0), dict(action_dim=0), dict(hidden_dims=(8, 0)), dict(activation="mish"), dict(gated_activation="x"), dict(dtype=torch.float64), dict(memory_blocks=-1),
  dict(memory_blocks=1, heads=0), dict(memory_blocks=1, head_dim=129), dict(memory_blocks=1, hidden_dims=()), dict(memory_steps=(0.0, 4.0)), dict(memory_steps=(8.0, 4.0)),
])  # fmt: skip
def test_configuration_refusals(kw):
  with pytest.raises(ValueError):
    PolicyCfg(**{"obs_dim": 9, "action_dim": 3, **kw})


def test_parameters_and_state():
  p = Policy(PolicyCfg(99, 29, memory_blocks=2, heads=4, head_dim=16, memory_steps=(4.0, 256.0)), "cpu")
  assert [tuple(w.shape) for w in p.weights] == [(512, 99), (256, 512), (128, 256)] and p.head_weight.shape == (29, 128)
  assert p.initial_state(5).shape == (2, 5, 4, 16, 16) and not p.initial_state(5).any()
  assert torch.allclose(-1.0 / p.log_decay, torch.tensor([4.0, 16.0, 64.0, 256.0]))
  assert len({id(x) for x in p.parameters()}) == 3 + 3 + 2 + 2 * 5
  assert Policy(PolicyCfg(9, 3), "cpu").initial_state(5) is None
  q = Policy(p.cfg, "cpu")
  q.load_state_dict(p.state_dict())
  assert all(torch.equal(a, b) for a, b in zip(p.parameters(), q.parameters(), strict=True))


def test_from_mlp():
  act = torch.nn.ELU()
  mlp = torch.nn.Sequential(torch.nn.Linear(9, 16), act, torch.nn.Linear(16, 8), act, torch.nn.Linear(8, 3))
  params = {f"actor.{k}": v for k, v in mlp.state_dict().items()} | {"critic.0.weight": torch.zeros(2, 2), "std": torch.ones(3)}
  p = Policy.from_mlp(params, device="cpu")
  assert p.cfg.hidden_dims == (16, 8) and p.cfg.obs_dim == 9 and p.cfg.action_dim == 3
  assert torch.equal(p.weights[1], mlp[2].weight) and torch.equal(p.head_bias, mlp[4].bias)
  with pytest.raises(ValueError, match="no parameter"):
    Policy.from_mlp(params, prefix="student.", device="cpu")
  with pytest.raises(ValueError, match="follow"):
    Policy.from_mlp({**params, "actor.2.weight": torch.zeros(8, 15)}, device="cpu")
  with pytest.raises(ValueError, match="expected"):
    Policy.from_mlp({**params, "actor.0.bias": torch.zeros(15)}, device="cpu")


def test_shapes_are_checked_before_anything_runs():
  p = Policy(PolicyCfg(9, 3, memory_blocks=1), "cpu")
  with pytest.raises(ValueError, match="observations"):
    p.act(torch.zeros(4, 8))
  with pytest.raises(ValueError, match="needs its state"):
    p.act(torch.zeros(4, 9))
  with pytest.raises(ValueError, match="state"):
    p.act(torch.zeros(4, 9), state=p.initial_state(5))
  with pytest.raises(ValueError, match="observations"):
    p(torch.zeros(4, 9))
  with pytest.raises(TypeError, match="no CPU fallback"):
    p.act(torch.zeros(4, 9), state=p.initial_state(4))
  assert math.isfinite(float(p.log_decay.sum()))
