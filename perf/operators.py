"""The operators of a policy network, as cases: dense layers, gated layers, and linear attention with a decay per head.

``own`` false: elementary torch operations in 32 bits, rounded once at the end.  ``own`` true: the calls that a user makes of
``mjlab_amd.policy_ops``.  Sizes: 4096 environments per device, observation rows of 99 / 286 floats, 29 actions, hidden layers of
512-256-128, updates over 24 stored steps in 4 minibatches (24576 rows); the larger ones are generic.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ACTIVATIONS = ("none", "relu", "elu", "tanh", "sigmoid", "silu", "gelu")
MAX_FLOPS = 3.7e11  # the largest listed case (gated_large_bf16)
MAX_PAIRS = 2 * 8 * 8192 * 8192  # batch x heads x length^2 of the longest listed sequence


def listed() -> list:
  return [
    # the first layer of an actor at every control step of 4096 environments
    dict(name="dense_step_f32", op="dense", dtype="f32", rows=4096, inp=99, out=512, act="elu", bias=True, residual=False, train=False),
    # the action head of a handful of environments (an evaluation run): pure latency
    dict(name="dense_head_f32_small", op="dense", dtype="f32", rows=16, inp=128, out=29, act="none", bias=True, residual=False, train=False),
    # a hidden layer inside one minibatch of an update
    dict(name="dense_update_f32", op="dense", dtype="f32", rows=24576, inp=512, out=256, act="elu", bias=True, residual=False, train=True),
    # a wide residual layer in 16 bits, same minibatch
    dict(name="dense_update_bf16_residual", op="dense", dtype="bf16", rows=24576, inp=1024, out=1024, act="gelu", bias=True, residual=True, train=True),
    # nothing is a multiple of anything: a critic row of 286 floats, an odd batch, an odd width
    dict(name="dense_ragged_f16", op="dense", dtype="f16", rows=5003, inp=286, out=517, act="silu", bias=True, residual=True, train=True),
    # the gated layer of a memory block at every control step
    dict(name="gated_step_f32", op="gated", dtype="f32", rows=4096, inp=256, out=512, act="silu", bias=False, train=False),
    # the same in an update, with the odd width that two thirds of a power of two give
    dict(name="gated_update_bf16", op="gated", dtype="bf16", rows=24576, inp=512, out=1365, act="silu", bias=True, train=True),
    # a large layer: the matrix cores are the bound
    dict(name="gated_large_bf16", op="gated", dtype="bf16", rows=16384, inp=2048, out=2816, act="gelu", bias=False, train=False),
    # the memory of 4096 environments over one control step, some of them just reset
    dict(name="memory_step_f32", op="step", dtype="f32", batch=4096, heads=4, dk=64, dv=64, reset=0.01),
    # stored rollouts: 1024 environments, 24 steps, cut where episodes ended, a state carried in
    dict(name="memory_update_f32", op="chunk", dtype="f32", batch=1024, length=24, heads=4, dk=64, dv=64, reset=0.02, carry=True, ragged=False,
         time_major=True, train=True),
    # few long sequences: the time axis has to be split
    dict(name="memory_long_bf16", op="chunk", dtype="bf16", batch=2, length=8192, heads=8, dk=128, dv=128, reset=0.0, carry=False, ragged=False,
         time_major=False, train=True),
    # sequences of different lengths, head sizes off the grid, a state carried in and out
    dict(name="memory_prompt_f16_ragged", op="chunk", dtype="f16", batch=5, length=1999, heads=6, dk=48, dv=80, reset=0.001, carry=True, ragged=True,
         time_major=False, train=False),
  ]


def _log_int(rng, lo: int, hi: int) -> int:
  return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng) -> dict:
  dtype = rng.choice(tuple(DTYPES))
  op = rng.choice(("dense", "gated", "step", "chunk"))
  if op in ("dense", "gated"):
    while True:
      case = dict(op=op, dtype=dtype, rows=_log_int(rng, 1, 65536), inp=_log_int(rng, 1, 2048), out=_log_int(rng, 1, 4096), act=rng.choice(ACTIVATIONS),
                  bias=rng.random() < 0.7, train=rng.random() < 0.6)
      if op == "dense":
        case["residual"] = rng.random() < 0.5
      if work(case)["flops"] <= MAX_FLOPS:
        return case
  sizes = (8, 16, 24, 32, 33, 48, 64, 80, 96, 128)
  case = dict(op=op, dtype=dtype, heads=rng.choice((1, 2, 3, 4, 6, 8, 16)), dk=rng.choice(sizes), dv=rng.choice(sizes), reset=rng.choice((0.0, 0.002, 0.05)))
  if op == "step":
    case["batch"] = _log_int(rng, 1, 8192)
    return case
  while True:
    case.update(batch=_log_int(rng, 1, 2048), length=_log_int(rng, 1, 8192), carry=rng.random() < 0.5, ragged=rng.random() < 0.5,
                time_major=rng.random() < 0.5, train=rng.random() < 0.6)
    if case["batch"] * case["heads"] * case["length"] ** 2 <= MAX_PAIRS and case["batch"] * case["heads"] * case["length"] <= 2 * 8 * 8192:
      return case


def prepare(case: dict, seed: int) -> dict:
  gen = torch.Generator(device="cuda")
  gen.manual_seed(seed)
  dt = DTYPES[case["dtype"]]

  def normal(*shape, scale=1.0, dtype=dt):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)

  if case["op"] in ("dense", "gated"):
    m, k, n = case["rows"], case["inp"], case["out"]
    st = dict(case=case, x=normal(m, k))
    for name in ("w",) if case["op"] == "dense" else ("w", "w_up"):
      st[name] = normal(n, k, scale=k**-0.5)
      st[name.replace("w", "b")] = normal(n, scale=0.3) if case["bias"] else None
    if case["op"] == "dense":
      st["r"] = normal(m, n) if case["residual"] else None
    st["dy"] = normal(m, n) if case["train"] else None
    leaves = ("x", "w", "b", "r") if case["op"] == "dense" else ("x", "w", "w_up", "b", "b_up")
  else:
    bsz, h, dk, dv = case["batch"], case["heads"], case["dk"], case["dv"]
    st = dict(case=case, scale=dk**-0.5, log_decay=torch.log1p(-torch.exp2(-2.0 - 4.0 * torch.arange(h, device="cuda") / h)))
    if case["op"] == "step":
      st.update(q=normal(bsz, h, dk), k=normal(bsz, h, dk), v=normal(bsz, h, dv), state=normal(bsz, h, dk, dv, dtype=torch.float32),
                reset=torch.rand((bsz,), generator=gen, device="cuda") < case["reset"], out_state=torch.empty((bsz, h, dk, dv), device="cuda"))
    else:
      t = case["length"]

      def rows(d):  # (batch, time, heads, d), stored time-major where a rollout buffer is
        return normal(t, bsz, h, d).transpose(0, 1) if case["time_major"] else normal(bsz, t, h, d)

      st.update(q=rows(dk), k=rows(dk), v=rows(dv), reset=None, lengths=None, state=None, do=None, dstate=None)
      if case["reset"] > 0:
        st["reset"] = torch.rand((bsz, t), generator=gen, device="cuda") < case["reset"]
      if case["ragged"]:
        st["lengths"] = torch.randint(0, t + 1, (bsz,), generator=gen, device="cuda", dtype=torch.int32)
      if case["carry"]:
        st["state"] = normal(bsz, h, dk, dv, dtype=torch.float32)
      if case["train"]:
        st["do"] = rows(dv)
        if case["carry"]:
          st["dstate"] = normal(bsz, h, dk, dv, dtype=torch.float32)
    leaves = ("q", "k", "v", "state")
  if case.get("train"):
    st["leaves"] = [st[name].requires_grad_(True) for name in leaves if st[name] is not None]
  return st


# ---------------------------------------------------------------------------------------------------------------- one pass


def run(st: dict):
  case = st["case"]
  if case["op"] == "step":
    return _step(st)
  with torch.set_grad_enabled(case["train"]):
    outs, ups = _chunk(st) if case["op"] == "chunk" else _layer(st)
    if not case["train"]:
      return outs
    grads = torch.autograd.grad(outs, st["leaves"], ups)
    return [o.detach() for o in outs] + list(grads)


def _layer(st: dict):
  case = st["case"]
  if own:
    from mjlab_amd import policy_ops

    if case["op"] == "dense":
      y = policy_ops.dense(st["x"], st["w"], st["b"], activation=case["act"], residual=st["r"])
    else:
      y = policy_ops.gated(st["x"], st["w"], st["w_up"], st["b"], st["b_up"], activation=case["act"])
    return [y], [st["dy"]]
  x = st["x"].float()

  def product(w, b):
    z = x @ w.float().t()
    return z if b is None else z + b.float()

  y = _act(product(st["w"], st["b"]), case["act"])
  if case["op"] == "gated":
    y = y * product(st["w_up"], st["b_up"])
  elif st["r"] is not None:
    y = y + st["r"].float()
  return [y.to(st["x"].dtype)], [st["dy"]]


def _act(z: torch.Tensor, name: str) -> torch.Tensor:
  if name == "none":
    return z
  if name == "relu":
    return torch.where(z < 0, torch.zeros_like(z), z)
  if name == "elu":
    return torch.where(z > 0, z, torch.expm1(torch.where(z > 0, torch.zeros_like(z), z)))
  if name == "tanh":
    return torch.tanh(z)
  if name == "sigmoid":
    return torch.sigmoid(z)
  if name == "silu":
    return z * torch.sigmoid(z)
  return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))


def _step(st: dict):
  if own:
    from mjlab_amd import policy_ops

    return list(policy_ops.decay_attention_step(st["q"], st["k"], st["v"], st["log_decay"], st["state"], scale=st["scale"], reset=st["reset"],
                                                out_state=st["out_state"]))
  keep = torch.where(st["reset"][:, None, None, None], torch.zeros_like(st["state"]), st["state"])
  state = keep * torch.exp(st["log_decay"])[None, :, None, None] + st["k"].float()[..., :, None] * st["v"].float()[..., None, :]
  o = (st["q"].float()[..., :, None] * state).sum(dim=2) * st["scale"]
  return [o.to(st["q"].dtype), state]


def _chunk(st: dict):
  if own:
    from mjlab_amd import policy_ops

    o, state = policy_ops.decay_attention(st["q"], st["k"], st["v"], st["log_decay"], scale=st["scale"], state=st["state"], reset=st["reset"],
                                          lengths=st["lengths"])
  else:
    o, state = _chunk_plain(st)
  if st["case"]["carry"]:
    return [o, state], [st["do"], st["dstate"]]
  return [o], [st["do"]]


def _chunk_plain(st: dict):
  """Every pair (i, j) of one episode with j <= i, weighted by decay^(i - j): (length x length) matrices per sequence and head."""
  q, k, v = (st[n].float().transpose(1, 2) for n in ("q", "k", "v"))  # (batch, heads, time, d)
  bsz, _, t, _ = q.shape
  g = st["log_decay"]
  pos = torch.arange(t, device=q.device)
  length = torch.full((bsz,), t, device=q.device) if st["lengths"] is None else st["lengths"].long()
  live = pos[None, :] < length[:, None]
  episode = torch.zeros((bsz, t), dtype=torch.long, device=q.device) if st["reset"] is None else torch.cumsum((st["reset"] & live).long(), dim=1)
  gap = pos[:, None] - pos[None, :]
  pair = (gap >= 0)[None] & (episode[:, :, None] == episode[:, None, :]) & live[:, :, None] & live[:, None, :]
  weight = torch.exp(g[:, None, None] * gap.clamp(min=0)[None])
  a = (q @ k.transpose(2, 3)) * torch.where(pair[:, None], weight[None], torch.zeros_like(weight[None]))
  o = a @ v
  last = episode.gather(1, (length - 1).clamp(min=0)[:, None])[:, 0] if t else torch.zeros_like(length)
  tail = torch.where((live & (episode == last[:, None]))[:, None], torch.exp(g[None, :, None] * (length[:, None] - 1 - pos[None]).clamp(min=0)[:, None]), 0.0)
  state = (k * tail[..., None]).transpose(2, 3) @ v
  if st["state"] is not None:
    s0 = st["state"]
    head = torch.where((live & (episode == 0))[:, None], torch.exp(g[None, :, None] * (pos + 1)[None, None]), 0.0)
    o = o + head[..., None] * (q @ s0)
    state = state + torch.where((last == 0)[:, None], torch.exp(g[None] * length[:, None]), 0.0)[..., None, None] * s0
  return (o * st["scale"]).transpose(1, 2).to(st["q"].dtype), state


# ---------------------------------------------------------------------------------------------------------------- the work


def work(case: dict) -> dict:
  size = 4 if case["dtype"] == "f32" else 2
  if case["op"] in ("dense", "gated"):
    m, k, n = case["rows"], case["inp"], case["out"]
    pair = 1 if case["op"] == "dense" else 2
    weights = pair * (n * k + (n if case["bias"] else 0))
    moved = m * k + weights + m * n * (2 if case.get("residual") else 1)
    flops = 2.0 * pair * m * n * k
    if case["train"]:  # the upstream gradient in; the gradients of x, the weights, the biases and the residual out
      moved += m * n + m * k + weights + (m * n if case.get("residual") else 0)
      flops *= 3
    return {"bytes": moved * size, "flops": flops}
  bsz, h, dk, dv = case["batch"], case["heads"], case["dk"], case["dv"]
  if case["op"] == "step":
    return {"bytes": bsz * h * (8 * dk * dv + size * (2 * dk + 2 * dv)) + bsz, "flops": 5.0 * bsz * h * dk * dv}
  t = case["length"]
  mean = t / 2 if case["ragged"] else t
  moved = bsz * h * t * (2 * dk + 2 * dv) * size + (bsz * t if case["reset"] > 0 else 0) + (8 * bsz * h * dk * dv if case["carry"] else 0)
  flops = bsz * h * min(4.0 * mean * dk * dv, mean * (mean + 1) * (dk + dv))
  if case["train"]:
    moved += bsz * h * t * (2 * dk + 2 * dv) * size + (8 * bsz * h * dk * dv if case["carry"] else 0)
    flops *= 3
  return {"bytes": moved, "flops": flops}


# ------------------------------------------------------------------------------------------- the definitions, in 64 bits


def exact(case: dict, seed: int):
  st = prepare(case, seed)
  with torch.no_grad():
    if case["op"] in ("dense", "gated"):
      return _layer_exact(st)
    return _recurrence_exact(st)


def _act_exact(z: torch.Tensor, name: str):
  """(value, derivative) in the type of ``z``."""
  one = torch.ones_like(z)
  if name == "none":
    return z, one
  if name == "relu":
    return z.clamp(min=0), (z > 0).to(z.dtype)
  if name == "elu":
    low = z.clamp(max=0)
    return z.clamp(min=0) + low.expm1(), torch.where(z > 0, one, low.exp())
  if name == "tanh":
    return z.tanh(), z.cosh().reciprocal().square()
  s = (1 + (-z).exp()).reciprocal()
  ds = s * (1 + z.exp()).reciprocal()
  if name == "sigmoid":
    return s, ds
  if name == "silu":
    return z * s, s + z * ds
  phi = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
  return z * phi, phi + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)


def _layer_exact(st: dict):
  case = st["case"]
  d = {n: None if st.get(n) is None else st[n].detach().double() for n in ("x", "w", "w_up", "b", "b_up", "r", "dy")}
  z = d["x"].mm(d["w"].t().contiguous()) + (0 if d["b"] is None else d["b"])
  f, df = _act_exact(z, case["act"])
  if case["op"] == "dense":
    y = f if d["r"] is None else f + d["r"]
    if not case["train"]:
      return [y]
    dz = d["dy"] * df
    out = [y, dz.mm(d["w"]), dz.t().contiguous().mm(d["x"])]
    if d["b"] is not None:
      out.append(dz.sum(0))
    if d["r"] is not None:
      out.append(d["dy"])
    return out
  u = d["x"].mm(d["w_up"].t().contiguous()) + (0 if d["b_up"] is None else d["b_up"])
  if not case["train"]:
    return [f * u]
  dg, du = d["dy"] * u * df, d["dy"] * f
  out = [f * u, dg.mm(d["w"]) + du.mm(d["w_up"]), dg.t().contiguous().mm(d["x"]), du.t().contiguous().mm(d["x"])]
  if d["b"] is not None:
    out += [dg.sum(0), du.sum(0)]
  return out


def _recurrence_exact(st: dict):
  """One token after the other: S <- decay S (0 at a reset) + k v^T, o = scale q S, and the adjoint of that, last token first."""
  case = st["case"]
  one = case["op"] == "step"
  q, k, v = (st[n].detach().double() for n in ("q", "k", "v"))
  if one:
    q, k, v = (x[:, None] for x in (q, k, v))
  bsz, t, h, dk = q.shape
  dv = v.shape[3]
  lam = st["log_decay"].double().exp()[None, :, None, None]
  s = torch.zeros((bsz, h, dk, dv), dtype=torch.float64, device=q.device) if st["state"] is None else st["state"].detach().double()
  reset = torch.zeros((bsz, t), dtype=torch.bool, device=q.device) if st["reset"] is None else st["reset"].reshape(bsz, t)
  lengths = torch.full((bsz,), t, device=q.device) if st.get("lengths") is None else st["lengths"].long()
  live = torch.arange(t, device=q.device)[None] < lengths[:, None]
  kept = torch.where(reset, 0.0, 1.0).double()[:, :, None, None, None]
  on = live.double()[:, :, None, None]
  ragged = st.get("lengths") is not None
  train = bool(case.get("train"))
  do = st["do"].detach().double() * on if train else None
  o = torch.zeros((bsz, t, h, dv), dtype=torch.float64, device=q.device)
  dq = torch.zeros_like(q)
  for i in range(t):
    new = s * lam * kept[:, i] + k[:, i, :, :, None] * v[:, i, :, None, :]
    s = torch.where(live[:, i, None, None, None], new, s) if ragged else new
    o[:, i] = torch.matmul(q[:, i, :, None, :], s)[:, :, 0]
    if train:
      dq[:, i] = torch.matmul(s, do[:, i, :, :, None])[..., 0]
  o = o * on * st["scale"]
  if one:
    return [o[:, 0], s]
  outs = [o] + ([s] if case["carry"] else [])
  if not train:
    return outs
  q = q * on * st["scale"]
  adj = torch.zeros_like(s) if st["dstate"] is None else st["dstate"].double()
  dk_, dv_ = torch.zeros_like(k), torch.zeros_like(v)
  for i in reversed(range(t)):
    adj = adj + q[:, i, :, :, None] * do[:, i, :, None, :]
    dk_[:, i] = torch.matmul(adj, v[:, i, :, :, None])[..., 0]
    dv_[:, i] = torch.matmul(k[:, i, :, None, :], adj)[:, :, 0]
    back = adj * lam * kept[:, i]
    adj = torch.where(live[:, i, None, None, None], back, adj) if ragged else back
  outs += [dq * on * st["scale"], dk_ * on, dv_ * on]
  if case["carry"]:
    outs.append(adj)
  return outs
