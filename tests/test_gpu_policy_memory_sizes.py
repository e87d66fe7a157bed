"""Linear attention with a decay: every head size's kernel over at most 32 steps (one workgroup per sequence and head) and over split sequences, and bad numbers there.
Bounds as in test_gpu_policy_memory.py."""

import pytest
import torch
from test_gpu_policy_memory import U, check, inputs, recurrence

pytestmark = pytest.mark.gpu

HEADS = [(1, 1), (5, 3), (33, 20), (20, 33), (64, 64), (48, 80), (40, 104), (128, 32), (32, 128), (17, 128), (64, 128), (128, 64), (127, 127), (128, 128)]


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("dk,dv", HEADS)
@pytest.mark.parametrize("t", [1, 24, 32])
def test_short(t, dk, dv, dtype):
  check(inputs(5, t, 3, dk, dv, dtype, seed=dk + t, resets=0.05, carry=True, ragged=True, time_major=True), dtype)
  check(inputs(3, t, 2, dk, dv, dtype, seed=dv + t), dtype)


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("dk,dv", [(64, 64), (127, 127), (128, 128), (128, 32), (32, 128), (48, 80), (104, 40)])
def test_split(dk, dv, dtype):
  check(inputs(2, 1100, 2, dk, dv, dtype, seed=dk, resets=0.01, carry=True, ragged=True), dtype)
  check(inputs(1, 777, 1, dk, dv, dtype, seed=dv), dtype)


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("dk,dv", [(20, 20), (64, 64), (48, 80), (128, 128), (127, 17)])
@pytest.mark.parametrize("which", ["q", "k", "v", "do", "state", "dstate"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("t", [30, 200])
def test_a_bad_number_reaches_what_the_recurrence_takes_it_to(t, which, dk, dv, bad, dtype):
  """... and nothing else: outputs and gradients are finite where the recurrence's are, in every episode, and near them there.  (Whether an infinity or a NaN stands where they are
  not depends on the order of the sums: q (k v^T) is infinite where (q k) v are infinities of both signs.)"""
  from mjlab_amd import policy_ops

  x = inputs(3, t, 2, dk, dv, dtype, seed=19, carry=True)
  x["reset"] = torch.zeros((3, t), dtype=torch.bool, device="cuda")
  x["reset"][:, [9, 21]] = True
  x["lengths"] = torch.tensor([t, 26, t - 1], dtype=torch.int32, device="cuda")
  if which in ("state", "dstate"):
    x[which][1, 1, dk // 2, dv // 3] = bad
  else:
    x[which][1, 14, 1, min(dk, dv) // 2] = bad
  leaves = [x[n].requires_grad_(True) for n in ("q", "k", "v", "state")]
  o, final = policy_ops.decay_attention(*leaves[:3], x["log_decay"], state=leaves[3], reset=x["reset"], lengths=x["lengths"])
  got = [o, final, *torch.autograd.grad([o, final], leaves, [x["do"], x["dstate"]])]
  with torch.no_grad():
    want = recurrence(*leaves[:3], x["log_decay"].double().exp(), dk**-0.5, leaves[3], x["reset"], x["lengths"], x["do"], x["dstate"])
    for name, g, w in zip(("o", "final", "dq", "dk", "dv", "dstate"), got, want, strict=True):
      w = w.to(g.dtype)
      assert torch.equal(g.isfinite(), w.isfinite()), (name, int((g.isfinite() != w.isfinite()).sum()))
      ok = w.isfinite()
      assert (g[ok] - w[ok]).float().norm() <= 0.02 * w[ok].float().norm() + 1e-30, name
