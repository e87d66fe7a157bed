"""The policy network between an environment's observation rows and its action rows, on the operators of mjlab_amd/policy_ops.py.

The reference trains an actor of dense layers (src/mjlab/tasks/velocity/config/g1/rl_cfg.py:17-28: 512-256-128, ELU) through an external
learner; ``Policy.from_mlp`` takes such an actor's parameters.  ``PolicyCfg.memory_blocks`` adds a memory over the control steps: blocks of linear
attention with a decay per head, whose state (one matrix per environment and head) is cut where an environment was reset, each followed by a gated layer:

  x <- x + W_o decay_attention(W_q x, W_k x, W_v x);   x <- x + W_down (act(W_gate x) * W_up x)

``act`` is one control step (what PhysicsRollout.policy_action calls, inside the captured control step if there is one); ``forward`` recomputes stored
steps for an update, with gradients."""

from __future__ import annotations

import dataclasses
import re

import torch

from . import policy_ops


@dataclasses.dataclass
class PolicyCfg:
  obs_dim: int
  action_dim: int
  hidden_dims: tuple[int, ...] = (512, 256, 128)
  activation: str = "elu"
  memory_blocks: int = 0
  heads: int = 4
  head_dim: int = 32
  gated_dim: int | None = None  # width inside a block's gated layer; None: twice the last hidden width
  gated_activation: str = "silu"
  memory_steps: tuple[float, float] = (4.0, 256.0)  # control steps after which the fastest / slowest head has forgotten all but 1 / e
  dtype: torch.dtype = torch.float32

  def __post_init__(self) -> None:
    if self.obs_dim < 1 or self.action_dim < 1 or any(d < 1 for d in self.hidden_dims):
      raise ValueError("PolicyCfg: the dimensions must be positive")
    for name in (self.activation, self.gated_activation):
      if name not in policy_ops.ACTIVATIONS:
        raise ValueError(f"PolicyCfg: unknown activation {name!r} (one of {', '.join(policy_ops.ACTIVATIONS)})")
    if self.dtype not in policy_ops.DTYPES:
      raise ValueError(f"PolicyCfg: dtype must be one of {list(policy_ops.DTYPES)}")
    if self.memory_blocks < 0:
      raise ValueError("PolicyCfg: memory_blocks must not be negative")
    if self.memory_blocks and (not self.hidden_dims or self.heads < 1 or not 1 <= self.head_dim <= policy_ops.MAX_HEAD_DIM):
      raise ValueError(f"PolicyCfg: memory blocks need a hidden layer before them, a head and a head size in [1, {policy_ops.MAX_HEAD_DIM}]")
    if not 0 < self.memory_steps[0] <= self.memory_steps[1]:
      raise ValueError("PolicyCfg: memory_steps must be positive and in order")


class Policy(torch.nn.Module):
  def __init__(self, cfg: PolicyCfg, device: torch.device | str = "cuda") -> None:
    super().__init__()
    self.cfg = cfg

    def linear(out: int, inp: int) -> torch.nn.Parameter:  # uniform in +- in^-1/2, as torch.nn.Linear
      return torch.nn.Parameter(((torch.rand((out, inp), device=device) * 2 - 1) * inp**-0.5).to(cfg.dtype))

    def zeros(out: int) -> torch.nn.Parameter:
      return torch.nn.Parameter(torch.zeros((out,), dtype=cfg.dtype, device=device))

    dims = (cfg.obs_dim, *cfg.hidden_dims)
    self.weights = torch.nn.ParameterList([linear(o, i) for i, o in zip(dims[:-1], dims[1:], strict=True)])
    self.biases = torch.nn.ParameterList([zeros(o) for o in dims[1:]])
    self.head_weight, self.head_bias = linear(cfg.action_dim, dims[-1]), zeros(cfg.action_dim)
    width, inner = dims[-1], cfg.heads * cfg.head_dim
    gated = cfg.gated_dim or 2 * width
    self.blocks = torch.nn.ModuleList()
    for _ in range(cfg.memory_blocks):
      b = torch.nn.Module()
      b.qkv, b.out, b.gate, b.up, b.down = linear(3 * inner, width), linear(width, inner), linear(gated, width), linear(gated, width), linear(width, gated)
      self.blocks.append(b)
    fast, slow = cfg.memory_steps
    steps = fast * (slow / fast) ** (torch.arange(cfg.heads, dtype=torch.float64) / max(1, cfg.heads - 1))
    self.register_buffer("log_decay", (-1.0 / steps).to(torch.float32).to(device))

  @classmethod
  def from_mlp(cls, parameters: dict[str, torch.Tensor], activation: str = "elu", prefix: str = "actor.", device: torch.device | str = "cuda",
               dtype: torch.dtype = torch.float32) -> "Policy":
    """A policy without memory from the parameters of a torch.nn.Sequential of linear layers (``{prefix}{n}.weight`` / ``.bias``, n ascending): the form in
    which the reference's learner stores its actor."""
    pat = re.compile(re.escape(prefix) + r"(\d+)\.weight$")
    order = sorted(int(m.group(1)) for m in map(pat.match, parameters) if m)
    if not order:
      raise ValueError(f"from_mlp: no parameter is called {prefix}<n>.weight")
    ws = [parameters[f"{prefix}{n}.weight"] for n in order]
    bs = [parameters.get(f"{prefix}{n}.bias") for n in order]
    if any(w.dim() != 2 for w in ws) or any(a.shape[0] != b.shape[1] for a, b in zip(ws[:-1], ws[1:], strict=True)):
      raise ValueError(f"from_mlp: the layers do not follow on one another: {[tuple(w.shape) for w in ws]}")
    self = cls(PolicyCfg(ws[0].shape[1], ws[-1].shape[0], tuple(w.shape[0] for w in ws[:-1]), activation, dtype=dtype), device)
    with torch.no_grad():
      for mine, theirs in zip((*self.weights, self.head_weight, *self.biases, self.head_bias), (*ws, *bs), strict=True):
        if theirs is not None:
          if mine.shape != theirs.shape:
            raise ValueError(f"from_mlp: expected {tuple(mine.shape)}, got {tuple(theirs.shape)}")
          mine.copy_(theirs)
    return self

  def initial_state(self, num_envs: int) -> torch.Tensor | None:
    """The empty memory of `num_envs` environments: (blocks, environments, heads, head_dim, head_dim) float32; None without memory blocks."""
    c = self.cfg
    return torch.zeros((c.memory_blocks, num_envs, c.heads, c.head_dim, c.head_dim), device=self.log_decay.device) if c.memory_blocks else None

  def _check(self, obs: torch.Tensor, dims: int, state: torch.Tensor | None) -> None:
    if obs.dim() != dims or obs.shape[-1] != self.cfg.obs_dim:
      raise ValueError(f"Policy: expected observations of {dims} dimensions, the last one {self.cfg.obs_dim}, got {tuple(obs.shape)}")
    if state is not None:
      c = self.cfg
      want = (c.memory_blocks, obs.shape[0], c.heads, c.head_dim, c.head_dim)
      if not c.memory_blocks or tuple(state.shape) != want:
        raise ValueError(f"Policy: expected a state {want}, got {tuple(state.shape)}")

  def _encode(self, x: torch.Tensor) -> torch.Tensor:
    x = x.to(self.cfg.dtype)
    for w, b in zip(self.weights, self.biases, strict=True):
      x = policy_ops.dense(x, w, b, activation=self.cfg.activation)
    return x

  def _heads(self, block: torch.nn.Module, x: torch.Tensor) -> tuple[torch.Tensor, ...]:
    qkv = policy_ops.dense(x, block.qkv)
    return qkv.view(*x.shape[:-1], 3, self.cfg.heads, self.cfg.head_dim).unbind(-3)

  def _close(self, block: torch.nn.Module, x: torch.Tensor, o: torch.Tensor) -> torch.Tensor:
    x = policy_ops.dense(o.reshape(*x.shape[:-1], block.out.shape[1]), block.out, residual=x)
    return policy_ops.dense(policy_ops.gated(x, block.gate, block.up, activation=self.cfg.gated_activation), block.down, residual=x)

  @torch.no_grad()
  def act(self, obs: torch.Tensor, state: torch.Tensor | None = None, reset: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """One control step: obs (environments, obs_dim) -> actions (environments, action_dim) float32.  ``state`` (initial_state()) is updated in place; ``reset``
    (environments,): non-zero where the environment was reset since the last call.  ``out``: a contiguous float32 tensor for the actions."""
    self._check(obs, 2, state)
    if self.cfg.memory_blocks and state is None:
      raise ValueError("Policy.act: a policy with memory needs its state")
    x = self._encode(obs)
    for i, block in enumerate(self.blocks):
      q, k, v = self._heads(block, x)
      o, _ = policy_ops.decay_attention_step(q, k, v, self.log_decay, state[i], reset=reset)
      x = self._close(block, x, o)
    if out is None or self.cfg.dtype == torch.float32:
      return policy_ops.dense(x, self.head_weight, self.head_bias, out=out).to(torch.float32)
    return out.copy_(policy_ops.dense(x, self.head_weight, self.head_bias))

  def forward(self, obs: torch.Tensor, state: torch.Tensor | None = None, reset: torch.Tensor | None = None,
              lengths: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Stored steps: obs (environments, steps, obs_dim) -> actions (environments, steps, action_dim) float32 and the memory after the last step.  ``reset``
    (environments, steps): non-zero where a step was the first of an episode; ``state``: the memory before the first step.  A time-major buffer goes in as
    ``buffer.transpose(0, 1)`` and is worked on as it lies."""
    self._check(obs, 3, state)
    turned = obs.shape[0] > 1 and obs.shape[1] > 1 and obs.stride(1) > obs.stride(0)
    x = self._encode(obs.transpose(0, 1) if turned else obs)
    finals = []
    for i, block in enumerate(self.blocks):
      q, k, v = (t.transpose(0, 1) if turned else t for t in self._heads(block, x))
      o, final = policy_ops.decay_attention(q, k, v, self.log_decay, state=None if state is None else state[i], reset=reset, lengths=lengths)
      finals.append(final)
      x = self._close(block, x, o.transpose(0, 1) if turned else o)
    actions = policy_ops.dense(x, self.head_weight, self.head_bias).to(torch.float32)
    return actions.transpose(0, 1) if turned else actions, torch.stack(finals) if finals else None
