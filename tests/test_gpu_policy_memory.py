"""Linear attention with a decay per head (mjlab_amd/policy_ops.py) against its recurrence in 64 bits, element by element.

Bounds: every output is a sum of products; M is the same sum over the magnitudes (the recurrence run on absolute values).  In 32 bits a term passes
at most d + length + 4 chunks + |log_decay| length + 32 roundings (its dot product, the running sums, the chunks' decays, the powers exp(n log_decay) with
n log_decay rounded).  bfloat16 operands of the matrix cores are rounded besides: a weighted key and the state, or a weighted pair -- two roundings at
most.  float16: a pair and the state are two bfloat16, which is two roundings of 2^-17.  What the state in the end is made of (weighted keys as three bfloat16) is
not rounded.  Then the output's own."""

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
U32 = 2.0**-24
TINY = {torch.float32: 2.0**-126, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-126}


def recurrence(q, k, v, lam, scale, state, reset, lengths, do=None, dstate=None):
  """(o, final[, dq, dk, dv, dstate0]) in 64 bits; (batch, length, heads, d)."""
  b, t, h, dk = q.shape
  q, k, v = q.double(), k.double(), v.double()
  s = torch.zeros((b, h, dk, v.shape[3]), dtype=torch.float64, device=q.device) if state is None else state.double().clone()
  live = torch.ones((b, t), dtype=torch.bool, device=q.device) if lengths is None else torch.arange(t, device=q.device)[None] < lengths.long()[:, None]
  cut = torch.zeros((b, t), dtype=torch.bool, device=q.device) if reset is None else reset != 0
  lam = lam.double()[None, :, None, None]
  zero = torch.zeros((), dtype=torch.float64, device=q.device)
  o = torch.zeros((b, t, h, v.shape[3]), dtype=torch.float64, device=q.device)
  dq, dk_, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
  if do is not None:
    do = torch.where(live[:, :, None, None], do.double(), zero)
  for i in range(t):
    on = live[:, i, None, None, None]
    s = torch.where(on, torch.where(cut[:, i, None, None, None], zero, s * lam) + k[:, i, :, :, None] * v[:, i, :, None, :], s)
    o[:, i] = torch.where(on[..., 0], scale * (q[:, i, :, :, None] * s).sum(2), zero)
    if do is not None:
      dq[:, i] = torch.where(on[..., 0], scale * (s * do[:, i, :, None, :]).sum(3), zero)
  if do is None:
    return o, s
  g = torch.zeros_like(s) if dstate is None else dstate.double().clone()
  for i in reversed(range(t)):
    on = live[:, i, None, None, None]
    g = torch.where(on, g + scale * q[:, i, :, :, None] * do[:, i, :, None, :], g)
    dk_[:, i] = torch.where(on[..., 0], (g * v[:, i, :, None, :]).sum(3), zero)
    dv[:, i] = torch.where(on[..., 0], (g * k[:, i, :, :, None]).sum(2), zero)
    g = torch.where(on, torch.where(cut[:, i, None, None, None], zero, g * lam), g)
  return o, s, dq, dk_, dv, g


def inputs(b, t, h, dk, dv, dtype, seed=0, resets=0.0, ragged=False, carry=False, time_major=False, reset_dtype=torch.bool):
  gen = torch.Generator(device="cuda").manual_seed(seed)

  def rows(d):
    x = torch.randn((t, b, h, d) if time_major else (b, t, h, d), generator=gen, device="cuda").to(dtype)
    return x.transpose(0, 1) if time_major else x

  x = dict(q=rows(dk), k=rows(dk), v=rows(dv), do=rows(dv), log_decay=-torch.rand((h,), generator=gen, device="cuda") * 0.3)
  x["reset"] = (torch.rand((b, t), generator=gen, device="cuda") < resets).to(reset_dtype) if resets else None
  x["lengths"] = torch.randint(0, t + 1, (b,), generator=gen, device="cuda", dtype=torch.int32) if ragged else None
  x["state"] = torch.randn((b, h, dk, dv), generator=gen, device="cuda") if carry else None
  x["dstate"] = torch.randn((b, h, dk, dv), generator=gen, device="cuda") if carry else None
  return x


def check(x, dtype, scale=None):
  from mjlab_amd import policy_ops

  q, k, v, do = x["q"], x["k"], x["v"], x["do"]
  b, t, h, dk = q.shape
  sc = dk**-0.5 if scale is None else scale
  leaves = [t_.requires_grad_(True) for t_ in (q, k, v, x["state"]) if t_ is not None]
  call = lambda: policy_ops.decay_attention(q, k, v, x["log_decay"], scale=scale, state=x["state"], reset=x["reset"], lengths=x["lengths"])  # noqa: E731
  o, final = call()
  carry = x["state"] is not None
  grads = torch.autograd.grad([o, final] if carry else [o], leaves, [do, x["dstate"]] if carry else [do])
  with torch.no_grad():
    again = call()
    assert torch.equal(again[0], o) and torch.equal(again[1], final)
    lam = x["log_decay"].double().exp()
    args = (lam, sc, x["state"], x["reset"], x["lengths"], do, x["dstate"])
    want = recurrence(q, k, v, *args)
    mag = recurrence(q.abs(), k.abs(), v.abs(), lam, abs(sc), *(None if a is None else a.abs() for a in (x["state"],)), x["reset"], x["lengths"], do.abs(),
                     None if x["dstate"] is None else x["dstate"].abs())
    got = [o, final, *grads]
    names = ["o", "final", "dq", "dk", "dv", "dstate"]
    steps = max(dk, v.shape[3]) + t + 4 * (t // 32 + 1) + float(x["log_decay"].abs().max()) * t + 32
    u = U[dtype]
    for name, g, w, m in zip(names, got, want, mag, strict=False):
      assert g.shape == w.shape, name
      state = name in ("final", "dstate")
      rel = steps * U32 + (0 if state or dtype == torch.float32 else 2 * u * 1.01 if dtype == torch.bfloat16 else 2.0**-16)
      own = U32 if state else u
      bound = rel * m + own * (w.abs() + rel * m) + (0 if state else TINY[dtype])
      err = (g.double() - w).abs()
      worst = (err / bound.clamp(min=1e-300)).max().item() if err.numel() else 0.0
      assert g.isfinite().all() and worst <= 1.0, f"{name}: {worst:.3g} times its bound, error {err.max().item():.3g}"


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("t", [1, 2, 24, 31, 32, 33, 63, 64, 65, 130])
def test_lengths(t, dtype):
  check(inputs(3, t, 2, 16, 16, dtype, seed=t, resets=0.1, carry=True), dtype)
  check(inputs(3, t, 2, 16, 16, dtype, seed=t + 1, ragged=True), dtype)


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("dk,dv", [(1, 1), (5, 3), (33, 20), (64, 64), (48, 80), (128, 32), (17, 128), (127, 127), (128, 128)])
def test_head_sizes(dk, dv, dtype):
  check(inputs(2, 70, 3, dk, dv, dtype, seed=dk, resets=0.05, carry=True, ragged=True), dtype)


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("resets,ragged,carry,time_major", [(0, False, False, False), (0, True, True, True), (0.02, False, True, False), (0.3, True, False, True), (1.0, False, True, False)])
def test_split_sequences(dtype, resets, ragged, carry, time_major):
  """Few long sequences: segments, their scan, resets and ends inside and between them."""
  check(inputs(2, 1100, 2, 24, 40, dtype, seed=7, resets=resets, ragged=ragged, carry=carry, time_major=time_major), dtype, scale=0.37)


@pytest.mark.parametrize("dtype", list(U))
def test_many_sequences(dtype):
  check(inputs(300, 24, 4, 32, 32, dtype, seed=9, resets=0.05, carry=True, time_major=True, reset_dtype=torch.int32), dtype)
  check(inputs(131, 40, 2, 64, 64, dtype, seed=10, resets=0.05, ragged=True, reset_dtype=torch.uint8), dtype)


def test_lengths_of_zero_and_beyond():
  from mjlab_amd import policy_ops

  x = inputs(4, 50, 2, 8, 8, torch.float32, carry=True)
  x["lengths"] = torch.tensor([0, 50, 77, -3], dtype=torch.int32, device="cuda")
  with torch.no_grad():
    o, final = policy_ops.decay_attention(x["q"], x["k"], x["v"], x["log_decay"], state=x["state"], lengths=x["lengths"])
    full, ffinal = policy_ops.decay_attention(x["q"], x["k"], x["v"], x["log_decay"], state=x["state"])
  assert not o[[0, 3]].any() and torch.equal(final[[0, 3]], x["state"][[0, 3]])
  assert torch.equal(o[[1, 2]], full[[1, 2]]) and torch.equal(final[[1, 2]], ffinal[[1, 2]])
  x = inputs(3, 0, 2, 8, 8, torch.float32, carry=True)
  o, final = policy_ops.decay_attention(x["q"], x["k"], x["v"], x["log_decay"], state=x["state"])
  assert o.shape == (3, 0, 2, 8) and torch.equal(final, x["state"])
  s = x["state"].clone().requires_grad_(True)
  _, final = policy_ops.decay_attention(x["q"], x["k"], x["v"], x["log_decay"], state=s)
  (gs,) = torch.autograd.grad(final, s, x["dstate"])
  assert torch.equal(gs, x["dstate"])


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("which", ["q", "k", "v"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_bad_step_stays_in_its_episode(which, bad, dtype):
  from mjlab_amd import policy_ops

  b, t = 2, 600
  x = inputs(b, t, 1, 20, 20, dtype, seed=11)
  x["reset"] = torch.zeros((b, t), dtype=torch.bool, device="cuda")
  x["reset"][:, [40, 300]] = True
  clean, cfinal = policy_ops.decay_attention(x["q"], x["k"], x["v"], x["log_decay"], reset=x["reset"])
  for at in (45, 250, 299):
    y = {n: x[n].clone() for n in ("q", "k", "v")}
    y[which][1, at, 0, 3] = bad
    for n in y:
      y[n].requires_grad_(True)
    o, final = policy_ops.decay_attention(y["q"], y["k"], y["v"], x["log_decay"], reset=x["reset"])
    hit = torch.zeros((b, t), dtype=torch.bool, device="cuda")
    hit[1, at : (at + 1 if which == "q" else 300)] = True
    # (the chunk with the bad step sums in another order: 600 terms of magnitude < 100 each side, then one rounding)
    assert ((o[~hit].double() - clean[~hit].double()).abs() <= 2 * U[dtype] * clean[~hit].double().abs() + 2 * 600 * 100 * U32).all() and torch.equal(final, cfinal)
    assert not o[hit].isfinite().all(dim=-1).any()
    grads = torch.autograd.grad(o, list(y.values()), x["do"])
    episode = torch.zeros((b, t), dtype=torch.bool, device="cuda")
    episode[1, 40:300] = True
    for g in grads:
      assert g[~episode].isfinite().all()


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("dk,dv", [(16, 16), (48, 80), (128, 128), (19, 70)])
@pytest.mark.parametrize("which", ["k", "state"])
def test_an_infinite_key_or_state_stays_infinite(which, dk, dv, dtype):
  """... in the rows of the state that it reaches, and in the outputs that read them: not a NaN, and nowhere else."""
  from mjlab_amd import policy_ops

  x = inputs(2, 150, 2, dk, dv, dtype, seed=14, carry=True, resets=0.01)
  if which == "k":
    x["k"][0, 40, 1, 7] = float("inf")
  else:
    x["state"][1, 0, 3] = float("inf")
  o, final = policy_ops.decay_attention(x["q"], x["k"], x["v"], x["log_decay"], state=x["state"], reset=x["reset"])
  wo, ws = recurrence(x["q"], x["k"], x["v"], x["log_decay"].double().exp(), dk**-0.5, x["state"], x["reset"], None)
  assert not wo.isfinite().all()
  for g, w in ((o, wo), (final, ws)):
    assert torch.equal(g.isinf(), w.isinf()) and torch.equal(g.isnan(), w.isnan())
    assert torch.equal(g[g.isinf()].sign().double(), w[w.isinf()].sign())


def test_a_reset_drops_a_bad_state():
  from mjlab_amd import policy_ops

  x = inputs(2, 10, 2, 8, 8, torch.float32, carry=True)
  x["state"][0] = float("nan")
  x["reset"] = torch.zeros((2, 10), dtype=torch.bool, device="cuda")
  x["reset"][0, 0] = True
  o, final = policy_ops.decay_attention(x["q"], x["k"], x["v"], x["log_decay"], state=x["state"], reset=x["reset"])
  assert o.isfinite().all() and final.isfinite().all()
  o1, s1 = policy_ops.decay_attention_step(x["q"][:, 0], x["k"][:, 0], x["v"][:, 0], x["log_decay"], x["state"], reset=x["reset"][:, 0])
  assert o1.isfinite().all() and s1.isfinite().all()


def test_no_decay_and_full_decay():
  x = inputs(2, 100, 3, 8, 8, torch.float32, carry=True)
  x["log_decay"] = torch.tensor([0.0, float("-inf"), -200.0], device="cuda")
  from mjlab_amd import policy_ops

  o, final = policy_ops.decay_attention(x["q"], x["k"], x["v"], x["log_decay"], state=x["state"])
  want, wfinal = recurrence(x["q"], x["k"], x["v"], x["log_decay"].exp(), 8**-0.5, x["state"], None, None)
  mag, mfinal = recurrence(x["q"].abs(), x["k"].abs(), x["v"].abs(), x["log_decay"].exp(), 8**-0.5, x["state"].abs(), None, None)
  assert ((o.double() - want).abs() <= 200 * U32 * mag).all() and ((final.double() - wfinal).abs() <= 200 * U32 * mfinal).all()


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("b,h,dk,dv", [(1, 1, 1, 1), (5, 3, 33, 20), (70, 4, 64, 64), (3, 2, 48, 80), (2, 8, 128, 128), (9, 2, 7, 127)])
def test_step(b, h, dk, dv, dtype):
  from mjlab_amd import policy_ops

  x = inputs(b, 3, h, dk, dv, dtype, seed=b, resets=0.4, carry=True)
  state = x["state"].clone()
  for i in range(3):
    q, k, v = (x[n][:, i] for n in "qkv")
    before = state.clone()
    other = torch.empty_like(state)
    o2, s2 = policy_ops.decay_attention_step(q, k, v, x["log_decay"], before, reset=x["reset"][:, i], out_state=other)
    assert s2 is other and not before.equal(other)
    o, s = policy_ops.decay_attention_step(q, k, v, x["log_decay"], state, reset=x["reset"][:, i].to(torch.int32))
    assert s is state and torch.equal(o, o2) and torch.equal(state, other)
    args = (x["log_decay"].double().exp(), dk**-0.5)
    want, ws = recurrence(x["q"][:, i : i + 1], x["k"][:, i : i + 1], x["v"][:, i : i + 1], *args, before, x["reset"][:, i : i + 1], None)
    mag, ms = recurrence(x["q"][:, i : i + 1].abs(), x["k"][:, i : i + 1].abs(), x["v"][:, i : i + 1].abs(), *args, before.abs(), x["reset"][:, i : i + 1], None)
    rel = (dk + 16) * U32
    assert ((state.double() - ws).abs() <= 8 * U32 * ms).all()
    assert ((o.double() - want[:, 0]).abs() <= rel * mag[:, 0] + U[dtype] * (want[:, 0].abs() + rel * mag[:, 0]) + TINY[dtype]).all()


def test_steps_equal_the_stored_form():
  """What a rollout computes step by step is what the update recomputes from the stored steps, to rounding."""
  from mjlab_amd import policy_ops

  x = inputs(65, 40, 2, 32, 32, torch.float32, seed=3, resets=0.1, carry=True, time_major=True)
  o, final = policy_ops.decay_attention(x["q"], x["k"], x["v"], x["log_decay"], state=x["state"], reset=x["reset"])
  state = x["state"].clone()
  rows = []
  for i in range(40):
    out = torch.empty((65, 2, 32), device="cuda")
    rows.append(policy_ops.decay_attention_step(x["q"][:, i], x["k"][:, i], x["v"][:, i], x["log_decay"], state, reset=x["reset"][:, i], out=out)[0])
  lam = x["log_decay"].double().exp()
  mag, ms = recurrence(x["q"].abs(), x["k"].abs(), x["v"].abs(), lam, 32**-0.5, x["state"].abs(), x["reset"], None)
  assert ((torch.stack(rows, 1).double() - o.double()).abs() <= 400 * U32 * mag).all()
  assert ((state.double() - final.double()).abs() <= 400 * U32 * ms).all()


def test_graph_replays_equal_eager():
  from mjlab_amd import policy_ops

  x = inputs(2, 1100, 2, 40, 40, torch.bfloat16, seed=5, resets=0.01, carry=True)
  static = [x[n].clone().requires_grad_(True) for n in ("q", "k", "v", "state")]

  def update(leaves):
    o, final = policy_ops.decay_attention(*leaves[:3], x["log_decay"], state=leaves[3], reset=x["reset"])
    return [o, final, *torch.autograd.grad([o, final], leaves, [x["do"], x["dstate"]])]

  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    update(static)
  torch.cuda.current_stream().wait_stream(side)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    captured = update(static)
  for k in range(4):
    with torch.no_grad():
      static[0].copy_(x["q"] * (k + 1))
      static[3].mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    eager = update([t.detach().clone().requires_grad_(True) for t in static])
    for a, c in zip(captured, eager, strict=True):
      assert torch.equal(a, c)


@pytest.mark.parametrize("t", [20, 300])
def test_gradients_against_differences(t):
  """The outputs are linear in each of q, k, v and the state, so (f(x + d) - f(x - d)) / 2 = grad . d but for rounding: three values, each off by as many
  roundings as above of the same sums over magnitudes."""
  from mjlab_amd import policy_ops

  x = inputs(2, t, 3, 24, 40, torch.float32, seed=16, resets=0.02, ragged=True, carry=True)
  names = ("q", "k", "v", "state")
  rest = (x["reset"], x["lengths"])
  lam = x["log_decay"].double().exp()

  def f(leaves):
    o, final = policy_ops.decay_attention(*leaves[:3], x["log_decay"], state=leaves[3], reset=rest[0], lengths=rest[1])
    return (o.double() * x["do"].double()).sum() + (final.double() * x["dstate"].double()).sum()

  leaves = [x[n].requires_grad_(True) for n in names]
  grads = torch.autograd.grad(f(leaves), leaves)
  gen = torch.Generator(device="cuda").manual_seed(17)
  with torch.no_grad():
    for i, g in enumerate(grads):
      d = torch.randn(leaves[i].shape, generator=gen, device="cuda")
      moved = [[a + sign * d if j == i else a for j, a in enumerate(leaves)] for sign in (1, -1)]
      big = [(a.abs() + d.abs() if j == i else a.abs()) for j, a in enumerate(leaves)]
      mo, ms = recurrence(*big[:3], lam, 24**-0.5, big[3], *rest)
      mag = (mo * x["do"].double().abs()).sum() + (ms * x["dstate"].double().abs()).sum()
      steps = 40 + t + 4 * (t // 32 + 1) + float(x["log_decay"].abs().max()) * t + 32
      assert abs((f(moved[0]) - f(moved[1])) / 2 - (g.double() * d.double()).sum()) <= 3 * steps * U32 * mag, names[i]


def test_only_the_wanted_gradients():
  from mjlab_amd import policy_ops

  x = inputs(2, 50, 2, 8, 12, torch.float32, seed=6, carry=True)
  all_ = [t.requires_grad_(True) for t in (x["q"], x["k"], x["v"], x["state"])]
  o, final = policy_ops.decay_attention(*all_[:3], x["log_decay"], state=all_[3])
  full = torch.autograd.grad(o, all_, x["do"])
  for i in range(4):
    part = [t if j == i else t.detach() for j, t in enumerate(all_)]
    o, _ = policy_ops.decay_attention(*part[:3], x["log_decay"], state=part[3])
    (g,) = torch.autograd.grad(o, all_[i], x["do"])
    assert torch.equal(g, full[i])
  o, final = policy_ops.decay_attention(*all_[:3], x["log_decay"], state=all_[3])
  only = torch.autograd.grad(final, all_, x["dstate"], allow_unused=True)  # o unused: its gradient is zero
  assert not only[0].any()
  shared = torch.autograd.grad(policy_ops.decay_attention(all_[0], all_[0], all_[2], x["log_decay"])[0], all_[0], x["do"])[0]  # one tensor twice
  a, b = (all_[0].detach().clone().requires_grad_(True) for _ in range(2))
  ga, gb = torch.autograd.grad(policy_ops.decay_attention(a, b, all_[2], x["log_decay"])[0], (a, b), x["do"])
  assert torch.equal(shared, ga + gb)


def test_backward_twice():
  from mjlab_amd import policy_ops

  x = inputs(2, 1100, 2, 24, 40, torch.float32, seed=12, resets=0.01, carry=True)
  leaves = [t.requires_grad_(True) for t in (x["q"], x["k"], x["v"], x["state"])]
  outs = policy_ops.decay_attention(*leaves[:3], x["log_decay"], state=leaves[3], reset=x["reset"])
  first = torch.autograd.grad(outs, leaves, [x["do"], x["dstate"]], retain_graph=True)
  second = torch.autograd.grad(outs, leaves, [x["do"], x["dstate"]])
  assert all(torch.equal(a, b) for a, b in zip(first, second, strict=True))


def test_a_state_kept_for_a_backward_pass_and_then_stepped_is_noticed():
  from mjlab_amd import policy_ops

  x = inputs(3, 5, 2, 16, 16, torch.float32, seed=13, carry=True)
  q = x["q"].requires_grad_(True)
  state = x["state"].clone()
  o, _ = policy_ops.decay_attention(q, x["k"], x["v"], x["log_decay"], state=state)
  with torch.no_grad():
    policy_ops.decay_attention_step(q[:, 0], x["k"][:, 0], x["v"][:, 0], x["log_decay"], state)
  with pytest.raises(RuntimeError, match="modified by an inplace operation"):
    o.sum().backward()


def test_refusals_on_the_device():
  from mjlab_amd import policy_ops

  x = inputs(2, 6, 2, 8, 8, torch.float32, carry=True)
  q, k, v, g, s = x["q"], x["k"], x["v"], x["log_decay"], x["state"]
  one = (q[:, 0], k[:, 0], v[:, 0], g)
  big = torch.zeros((1, 2, 1, 129), device="cuda")
  bad = [
    (ValueError, lambda: policy_ops.decay_attention(q[0], k[0], v[0], g)),
    (ValueError, lambda: policy_ops.decay_attention(q, k[:, :5], v, g)),
    (TypeError, lambda: policy_ops.decay_attention(q, k.half(), v, g)),
    (ValueError, lambda: policy_ops.decay_attention(q, k, v, g[:1])),
    (ValueError, lambda: policy_ops.decay_attention(q, k, v, g.double())),
    (ValueError, lambda: policy_ops.decay_attention(q, k, v, g.clone().requires_grad_(True))),
    (ValueError, lambda: policy_ops.decay_attention(q, k, v, g, state=s[:1])),
    (ValueError, lambda: policy_ops.decay_attention(q, k, v, g, state=s.transpose(2, 3))),
    (ValueError, lambda: policy_ops.decay_attention(q, k, v, g, reset=torch.zeros((2, 5), dtype=torch.bool, device="cuda"))),
    (ValueError, lambda: policy_ops.decay_attention(q, k, v, g, reset=torch.zeros((2, 6), device="cuda"))),
    (ValueError, lambda: policy_ops.decay_attention(q, k, v, g, lengths=torch.zeros((2,), dtype=torch.int64, device="cuda"))),
    (ValueError, lambda: policy_ops.decay_attention(q.transpose(2, 3), k.transpose(2, 3), v.transpose(2, 3), g)),
    (ValueError, lambda: policy_ops.decay_attention(big, big, big, g[:1])),
    (ValueError, lambda: policy_ops.decay_attention_step(*one, s[:, :1])),
    (ValueError, lambda: policy_ops.decay_attention_step(q, k, v, g, s)),
    (ValueError, lambda: policy_ops.decay_attention_step(*one, s, out_state=s.half())),
    (ValueError, lambda: policy_ops.decay_attention_step(one[0].clone().requires_grad_(True), *one[1:], s)),
  ]
  for kind, call in bad:
    with pytest.raises(kind):
      call()
