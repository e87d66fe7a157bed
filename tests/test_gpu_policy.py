"""The policy network as it is used: its operators together against the same network in 64 bits, control steps against the update's recomputation, and
inside PhysicsRollout's captured control step."""

import numpy as np
import pytest
import torch

from mjlab_amd import robots
from mjlab_amd.policy import Policy, PolicyCfg

pytestmark = pytest.mark.gpu


def network(p, obs, state, reset):
  """forward() in 64 bits; parameters and their gradients live in a list of doubles, in the order of p.parameters()."""
  params = [x.detach().double().requires_grad_(True) for x in p.parameters()]
  by_name = dict(zip([n for n, _ in p.named_parameters()], params, strict=True))
  act = torch.nn.functional.elu
  x = obs.double()
  for i in range(len(p.weights)):
    x = act(x @ by_name[f"weights.{i}"].t() + by_name[f"biases.{i}"])
  c = p.cfg
  lam = p.log_decay.double().exp()[None, :, None, None]
  n, t = obs.shape[:2]
  for i in range(c.memory_blocks):
    qkv = (x @ by_name[f"blocks.{i}.qkv"].t()).reshape(n, t, 3, c.heads, c.head_dim)
    s = state[i].double()
    rows = []
    for j in range(t):
      q, k, v = qkv[:, j].unbind(1)
      s = torch.where(reset[:, j, None, None, None] != 0, torch.zeros_like(s), s * lam) + k[..., :, None] * v[..., None, :]
      rows.append((q[..., :, None] * s).sum(-2) * c.head_dim**-0.5)
    x = x + torch.stack(rows, 1).reshape(n, t, -1) @ by_name[f"blocks.{i}.out"].t()
    up, gate = x @ by_name[f"blocks.{i}.up"].t(), x @ by_name[f"blocks.{i}.gate"].t()
    x = x + (torch.nn.functional.silu(gate) * up) @ by_name[f"blocks.{i}.down"].t()
  return x @ by_name["head_weight"].t() + by_name["head_bias"], params


def make(memory_blocks=2, seed=0, dtype=torch.float32, obs_dim=37, action_dim=11):
  torch.manual_seed(seed)
  p = Policy(PolicyCfg(obs_dim, action_dim, (96, 64), memory_blocks=memory_blocks, heads=2, head_dim=16, memory_steps=(3.0, 40.0), dtype=dtype), "cuda")
  with torch.no_grad():
    for b in p.biases:
      b.uniform_(-0.1, 0.1)
  return p


# float32: a chain of about a dozen products of up to 128 terms, 30 steps of memory: 2^-24 times (12 x 128 + 30 x 4), times a condition of about 10 of the
# chain (its blocks add to x what they read from it).  bfloat16: about 40 roundings of 2^-8 on the way, which mostly average out: their root times a condition of 4.
TOL = {torch.float32: 2.0**-24 * 1656 * 10, torch.bfloat16: 2.0**-8 * 40**0.5 * 4}


@pytest.mark.parametrize("dtype", list(TOL))
@pytest.mark.parametrize("time_major", [False, True])
def test_update_and_its_gradients(dtype, time_major):
  p = make(dtype=dtype)
  gen = torch.Generator(device="cuda").manual_seed(1)
  n, t = 50, 30
  buf = torch.randn((t, n, 37) if time_major else (n, t, 37), generator=gen, device="cuda").to(dtype).float()
  obs = buf.transpose(0, 1) if time_major else buf
  reset = (torch.rand((n, t), generator=gen, device="cuda") < 0.1).int()
  state = torch.randn(p.initial_state(n).shape, generator=gen, device="cuda")
  up = torch.randn((n, t, 11), generator=gen, device="cuda")
  actions, final = p(obs, state=state, reset=reset)
  grads = torch.autograd.grad((actions * up).sum(), list(p.parameters()))
  want, params = network(p, obs, state, reset)
  wgrads = torch.autograd.grad((want * up.double()).sum(), params)
  assert final.shape == state.shape
  for name, g, w in zip(["actions", *[n_ for n_, _ in p.named_parameters()]], [actions, *grads], [want, *wgrads], strict=True):
    assert g.isfinite().all() and (g.double() - w).norm() <= TOL[dtype] * w.norm(), (name, float((g.double() - w).norm() / w.norm()))


def test_control_steps_equal_the_update():
  p = make()
  gen = torch.Generator(device="cuda").manual_seed(2)
  n, t = 33, 20
  obs = torch.randn((n, t, 37), generator=gen, device="cuda")
  reset = (torch.rand((n, t), generator=gen, device="cuda") < 0.15).int()
  state = p.initial_state(n)
  rows = []
  for j in range(t):
    out = torch.empty((n, 11), device="cuda")
    assert p.act(obs[:, j], state=state, reset=reset[:, j], out=out) is out
    rows.append(out)
  actions, final = p(obs, reset=reset)
  steps = torch.stack(rows, 1)
  assert (steps - actions).norm() <= TOL[torch.float32] * actions.norm() and (state - final).norm() <= TOL[torch.float32] * final.norm()
  # a reset at the first step forgets whatever came before
  again, _ = p(obs, reset=torch.ones_like(reset), state=torch.randn_like(state))
  alone, _ = p(obs.reshape(n * t, 1, 37))
  assert (again.reshape(n * t, 1, 11) - alone).norm() <= TOL[torch.float32] * alone.norm()


def test_no_environments_and_no_steps():
  p = make()
  for n, t in ((0, 3), (2, 0)):
    actions, final = p(torch.zeros((n, t, 37), device="cuda"))
    assert actions.shape == (n, t, 11) and final.shape == p.initial_state(n).shape and not final.any()
    sum(x.sum() for x in (actions, final)).backward()
  assert all(not x.grad.any() for x in p.parameters())
  assert p.act(torch.zeros((0, 37), device="cuda"), state=p.initial_state(0)).shape == (0, 11)


def test_from_mlp_equals_the_sequential():
  torch.manual_seed(3)
  act = torch.nn.ELU()
  mlp = torch.nn.Sequential(torch.nn.Linear(99, 512), act, torch.nn.Linear(512, 256), act, torch.nn.Linear(256, 128), act, torch.nn.Linear(128, 29)).cuda()
  p = Policy.from_mlp({f"actor.{k}": v for k, v in mlp.state_dict().items()})
  obs = torch.randn((500, 99), device="cuda")
  want = mlp.double()(obs.double())
  got = p.act(obs)
  assert (got.double() - want).norm() <= 2.0**-24 * (99 + 512 + 256 + 128 + 16) * want.norm() and got.dtype == torch.float32


def _rollout(**kw):
  from mjlab_amd.rollout import PhysicsRollout, g1_action_scale
  from mjlab_amd.sim import Simulation, SimulationCfg

  model = robots.load_model("g1_velocity_flat")
  sim = Simulation(64, SimulationCfg(njmax=300), model, "cuda:0")
  return PhysicsRollout(sim, action_scale=g1_action_scale(model), seed=5, **kw)


@pytest.mark.parametrize("memory_blocks", [0, 1])
@pytest.mark.parametrize("fused_reset", [True, False])
@pytest.mark.parametrize("inside", [True, False])
def test_rollout_with_a_policy_captured_equals_eager(memory_blocks, fused_reset, inside):
  """observation rows -> policy -> physics: the captured control step, with the policy inside or before it, replays what separate calls compute; resets cut
  the memory in both."""
  kw = dict(fused_reset=fused_reset, control_kernel=fused_reset, episode_length_s=0.2)
  a, b = _rollout(**kw), _rollout(**kw)
  p = make(memory_blocks, obs_dim=a.observation_rows().shape[1], action_dim=a.m.nu)
  mine, other = p.initial_state(64), p.initial_state(64)
  with pytest.raises(ValueError, match="action"):
    a.step()
  if inside:
    a.capture_graph(p)  # (runs one control step to warm up)
    b.step(b.policy_action(p, other))
  else:
    a.capture_graph()
    b.step(torch.zeros((64, b.m.nu), device="cuda"))
  resets = 0
  for _ in range(25):
    ra = a.step(None if inside else a.policy_action(p, mine, out=a.action_buffer))
    rb = b.step(b.policy_action(p, other))
    assert torch.equal(ra != 0, rb != 0)
    resets += int((ra != 0).sum())
    assert torch.equal(a.sim.data.qpos, b.sim.data.qpos)
    if memory_blocks:
      memory = a.policy_memory if inside else mine
      assert torch.equal(memory, other) and memory.any()
  assert resets > 64  # episodes of 10 steps: every environment was cut at least twice
  if memory_blocks:  # reset_all() cuts every memory
    b.reset_all()
    assert torch.equal(b.policy_action(p, other), p.act(b.observation_rows(), p.initial_state(64)))
  if not inside:
    return
  with pytest.raises(ValueError, match="action"):
    a.step(torch.zeros((64, a.m.nu), device="cuda"))
  a.reset_all()
  assert not memory_blocks or not a.policy_memory.any()
  # parameters are read at every replay
  with torch.no_grad():
    p.head_weight.zero_()
    p.head_bias.fill_(0.25)
  a.step()
  assert (a.action_buffer == 0.25).all()
  a.capture_graph()  # without the policy again: step() takes an action
  a.step(a.random_action(out=a.action_buffer))
  assert np.isfinite(a.sim.data.qpos.cpu().numpy()).all()
