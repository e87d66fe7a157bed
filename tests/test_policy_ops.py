"""The policy operators' library without a GPU: symbols, struct mirrors, and every refusal of the C ABI (nothing is launched)."""

import ctypes
import re
from pathlib import Path

import pytest
import torch

from mjlab_amd import native, policy_ops

ROOT = Path(__file__).resolve().parents[1]


def test_exports_every_declared_symbol():
  lib = native.policy_lib()
  declared = set(re.findall(r"\b(mjlab_[a-z_]+)\s*\(", (ROOT / "include" / "mjlab_policy.h").read_text()))
  assert declared == set(native.POLICY_SYMBOLS)
  for sym in declared:
    assert hasattr(lib, sym), sym
  assert lib.mjlab_policy_abi_version() == native.POLICY_ABI_VERSION


def test_no_cpu_fallback():
  with pytest.raises(TypeError, match="no CPU fallback"):
    policy_ops.dense(torch.zeros((2, 3)), torch.zeros((4, 3)))
  with pytest.raises(TypeError, match="no CPU fallback"):
    policy_ops.gated(torch.zeros((2, 3)), torch.zeros((4, 3)), torch.zeros((4, 3)))


def _layer(**kw):
  f = policy_ops.Layer()
  vals = dict(dtype=0, act=1, rows=4, inp=8, out=3, x=64, w=64, ldx=8, ldw=8, y=64, ldy=3)  # (addresses that no refused call reads)
  vals.update(kw)
  for k, v in vals.items():
    setattr(f, k, v)
  return f


@pytest.mark.parametrize("kw,text", [
  (dict(dtype=3), "dtype"), (dict(act=7), "activation"), (dict(act=-1), "activation"), (dict(rows=0), "sizes"), (dict(inp=0), "sizes"), (dict(out=-1), "sizes"),
  (dict(inp=1 << 30), "sizes"), (dict(out=1 << 27), "sizes"), (dict(rows=1 << 30, out=1 << 20), "2^44"), (dict(x=None), "null x or w"), (dict(w=None), "null x or w"), (dict(y=None), "null y"), (dict(ldx=-8), "negative"),
  (dict(ldy=2), "overlap"), (dict(w_up=64, ldw_up=8, r=64), "residual"), (dict(b_up=64), "b_up"), (dict(z_up=64), "z_up"),
  (dict(rows=4, inp=2048, out=2048, ldy=2048), "workspace"),
])  # fmt: skip
def test_layer_forward_refuses(kw, text):
  lib = native.policy_lib()
  assert lib.mjlab_layer_forward(ctypes.byref(_layer(**kw)), None) < 0
  assert text in lib.mjlab_policy_last_error().decode()
  assert lib.mjlab_layer_forward(None, None) < 0


@pytest.mark.parametrize("kw,text", [
  (dict(dy=None), "null dy"), (dict(f=dict(z=None)), "(z)"), (dict(f=dict(w_up=64, ldw_up=8)), "z_up"),
  (dict(f=dict(w_up=64, ldw_up=8, z_up=64), dw=64), "together"), (dict(workspace_bytes=16), "workspace"), (dict(workspace=None), "workspace"),
  (dict(f=dict(rows=-1)), "sizes"), (dict(f=dict(act=5, z_is_y=1)), "z_is_y"), (dict(f=dict(z_bytes=2)), "z_bytes"),
  (dict(f=dict(w_up=64, ldw_up=8, z=None)), "(z)"), (dict(f=dict(dtype=2, w_up=64, ldw_up=2000, inp=2000, ldw=2000, z=None)), "(z)"),
])  # fmt: skip
def test_layer_backward_refuses(kw, text):
  lib = native.policy_lib()
  g = policy_ops.LayerGrad()
  kw = dict(kw)
  g.f = _layer(**{"z": 64, "z_bytes": 4, **kw.pop("f", {})})
  vals = dict(dy=64, ld_dy=3, dx=64, workspace=64, workspace_bytes=1 << 30)
  vals.update(kw)
  for k, v in vals.items():
    setattr(g, k, v)
  assert lib.mjlab_layer_backward(ctypes.byref(g), None) < 0
  assert text in lib.mjlab_policy_last_error().decode()


def test_which_gated_layers_form_their_sums_again():
  lib = native.policy_lib()
  gated = dict(w_up=64, ldw_up=512, inp=512, ldw=512)
  assert lib.mjlab_layer_recomputes(ctypes.byref(_layer(dtype=2, **gated))) == 1
  assert lib.mjlab_layer_recomputes(ctypes.byref(_layer(dtype=0, **gated))) == 0
  assert lib.mjlab_layer_recomputes(ctypes.byref(_layer(dtype=2, **{**gated, "inp": 4096}))) == 0
  assert lib.mjlab_layer_recomputes(ctypes.byref(_layer(dtype=2))) == 0


def test_few_rows_of_a_wide_layer_split_their_sums():
  lib = native.policy_lib()
  for dtype in (0, 1, 2):
    assert lib.mjlab_layer_forward_workspace(ctypes.byref(_layer(dtype=dtype, rows=4096, inp=512, out=512))) == 0
    assert lib.mjlab_layer_forward_workspace(ctypes.byref(_layer(dtype=dtype, rows=16, inp=99, out=29))) == 0
    assert lib.mjlab_layer_forward_workspace(ctypes.byref(_layer(dtype=dtype, rows=16, inp=2048, out=2048))) >= 2 * 16 * 2048 * 4
  assert lib.mjlab_layer_forward_workspace(ctypes.byref(_layer(rows=0))) == -1


def test_workspace_covers_what_the_backward_pass_stores():
  lib = native.policy_lib()
  for dtype, size in ((0, 4), (1, 2), (2, 2)):
    for gated in (False, True):
      g = policy_ops.LayerGrad()
      g.f = _layer(dtype=dtype, rows=5000, inp=70, out=33, **(dict(w_up=64, ldw_up=70) if gated else {}))
      g.dw, g.db = 64, 64
      pairs = 2 if gated else 1
      need = lib.mjlab_layer_backward_workspace(ctypes.byref(g))
      assert need >= 5000 * 33 * pairs * size + pairs * 33 * 4 * 40 + pairs * 33 * 70 * 4
  g.f.rows = 0
  assert lib.mjlab_layer_backward_workspace(ctypes.byref(g)) == -1


def _decay(**kw):
  d = policy_ops.Decay()
  vals = dict(dtype=0, batch=2, length=5, heads=2, dk=8, dv=8, scale=1.0, log_decay=64, state=64, state_out=128)
  rows = {n: policy_ops.Rows(64, 80, 16, 8) for n in ("q", "k", "v", "o")}
  for n, p in kw.items():
    if n in rows:
      rows[n].p = p
    else:
      vals[n] = p
  for n, val in {**vals, **rows}.items():
    setattr(d, n, val)
  return d


@pytest.mark.parametrize("kw,text", [
  (dict(dtype=5), "dtype"), (dict(batch=0), "positive"), (dict(length=0), "positive"), (dict(heads=0), "positive"), (dict(batch=1 << 23, heads=2), "positive"),
  (dict(dk=129), "dk and dv"), (dict(dv=0), "dk and dv"), (dict(q=None), "null q"), (dict(v=None), "null q"), (dict(log_decay=None), "log_decay"),
  (dict(reset=64, reset_bytes=2), "reset_bytes"), (dict(o=None), "null o"), (dict(state=128), "state_out"), (dict(length=5000), "workspace"),
])  # fmt: skip
def test_decay_forward_refuses(kw, text):
  lib = native.policy_lib()
  assert lib.mjlab_decay_forward(ctypes.byref(_decay(**kw)), None) < 0
  assert text in lib.mjlab_policy_last_error().decode()
  assert lib.mjlab_decay_forward(None, None) < 0


@pytest.mark.parametrize("kw,text", [(dict(), "length"), (dict(length=1, state=None), "null o"), (dict(length=1, state_out=None), "null o"), (dict(length=1, lengths=64), "lengths")])
def test_decay_step_refuses(kw, text):
  lib = native.policy_lib()
  assert lib.mjlab_decay_step(ctypes.byref(_decay(**kw)), None) < 0
  assert text in lib.mjlab_policy_last_error().decode()


def test_decay_backward_refuses():
  lib = native.policy_lib()
  g = policy_ops.DecayGrad()
  g.f = _decay()
  assert lib.mjlab_decay_backward(ctypes.byref(g), None) < 0 and "d_out" in lib.mjlab_policy_last_error().decode()
  g.d_out, g.d_state = policy_ops.Rows(64, 80, 16, 8), 64
  assert lib.mjlab_decay_backward(ctypes.byref(g), None) < 0 and "d_state" in lib.mjlab_policy_last_error().decode()
  g.d_state = None
  g.segments = g.f.workspace = 64
  assert lib.mjlab_decay_backward(ctypes.byref(g), None) < 0 and "segments" in lib.mjlab_policy_last_error().decode()
  g.f.length = 100000
  assert lib.mjlab_decay_backward(ctypes.byref(g), None) < 0 and "workspace" in lib.mjlab_policy_last_error().decode()


def test_decay_workspace_grows_only_where_sequences_are_split():
  lib = native.policy_lib()
  assert lib.mjlab_decay_workspace(ctypes.byref(_decay(length=24, batch=4096))) == 0
  assert lib.mjlab_decay_workspace(ctypes.byref(_decay(length=8192, batch=4096))) == 0
  assert lib.mjlab_decay_workspace(ctypes.byref(_decay(length=8192))) >= 4 * 8 * 8 * 4


def test_no_kernel_spills_ahead_of_its_exec_restore():
  """As for the physics library: no spill store of the policy kernels may sit in front of an EXEC restore -- and no product kernel spills at all."""
  from mjlab_amd import code_check

  if not (code_check.LLVM / "llvm-objdump").exists():
    pytest.skip("ROCm LLVM tools not installed")
  native.policy_lib()
  assert not code_check.fatal_hits(native.POLICY_LIB_PATH)
