"""Operators of the policy network between an environment's observation rows and its action rows (include/mjlab_policy.h).

  dense(x, weight, bias, activation, residual)   y = act(x W^T + b) + r
  gated(x, weight, weight_up, ...)               y = act(x W^T + b) * (x W_up^T + b_up)

``x`` has any leading dimensions and its last one is the layer's input; float32, float16 or bfloat16, the same type everywhere, sums in 32
bits, each output rounded once.  Both are differentiable in every tensor argument (once).  Every call enqueues on torch's current stream of
the tensors' device and may be captured into a hipGraph; nothing synchronises.  The last dimension of an argument must be contiguous, rows may
be any distance apart.  No fallback: without the HIP library, or for a tensor that is not on the GPU, these raise.

A backward pass that is captured into a graph must not share leaves with an eager autograd graph that is still alive (torch synchronises
with the eager stream inside the capture): capture from leaves of its own, as for any other torch operation."""

from __future__ import annotations

import ctypes

import torch

from . import native

_vp, _ll = ctypes.c_void_p, ctypes.c_longlong

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # MJLAB_DTYPE_*
ACTIVATIONS = {"none": 0, "relu": 1, "elu": 2, "tanh": 3, "sigmoid": 4, "silu": 5, "gelu": 6}  # MJLAB_ACT_*; gelu: the exact one (erf)


class Layer(ctypes.Structure):  # mjlab_layer_t
  _fields_ = [("dtype", ctypes.c_int), ("act", ctypes.c_int), ("rows", _ll), ("inp", _ll), ("out", _ll),
              ("x", _vp), ("w", _vp), ("w_up", _vp), ("b", _vp), ("b_up", _vp), ("r", _vp),
              ("ldx", _ll), ("ldw", _ll), ("ldw_up", _ll), ("ldr", _ll), ("ldy", _ll), ("y", _vp), ("z", _vp), ("z_up", _vp)]  # fmt: skip


class LayerGrad(ctypes.Structure):  # mjlab_layer_grad_t
  _fields_ = [("f", Layer), ("dy", _vp), ("ld_dy", _ll), ("dx", _vp), ("dw", _vp), ("dw_up", _vp), ("db", _vp), ("db_up", _vp),
              ("workspace", _vp), ("workspace_bytes", _ll)]  # fmt: skip


def _stream(dev: torch.device) -> int:
  return torch.cuda.current_stream(dev).cuda_stream


def _check(t: torch.Tensor, what: str, like: torch.Tensor, shape: tuple) -> torch.Tensor:
  if t.dtype != like.dtype or t.device != like.device:
    raise TypeError(f"{what}: expected {like.dtype} on {like.device}, got {t.dtype} on {t.device}")
  if tuple(t.shape) != shape:
    raise ValueError(f"{what}: expected shape {shape}, got {tuple(t.shape)}")
  if t.dim() and shape[-1] > 1 and t.stride(-1) != 1:
    raise ValueError(f"{what}: the last dimension must be contiguous (shape {tuple(t.shape)}, strides {t.stride()})")
  return t


def _rows(t: torch.Tensor, what: str) -> torch.Tensor:
  """(rows, last) over any leading dimensions, without a copy where the strides allow it."""
  if t.shape[-1] > 1 and t.stride(-1) != 1:
    raise ValueError(f"{what}: the last dimension must be contiguous (shape {tuple(t.shape)}, strides {t.stride()})")
  return t if t.dim() == 2 else t.reshape(-1, t.shape[-1])


def _ld(t: torch.Tensor) -> int:
  return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _layer_struct(x, w, w_up, b, b_up, act: int) -> Layer:
  f = Layer()
  f.dtype, f.act, f.rows, f.inp, f.out = DTYPES[x.dtype], act, x.shape[0], x.shape[1], w.shape[0]
  f.x, f.ldx, f.w, f.ldw = x.data_ptr(), _ld(x), w.data_ptr(), _ld(w)
  if w_up is not None:
    f.w_up, f.ldw_up = w_up.data_ptr(), _ld(w_up)
  f.b = None if b is None else b.data_ptr()
  f.b_up = None if b_up is None else b_up.data_ptr()
  return f


def _forward(x, w, w_up, b, b_up, r, act: int, keep: bool, y=None):
  """-> y, z, z_up (z: the sums before the activation where the backward pass will want them)."""
  m, n = x.shape[0], w.shape[0]
  if y is None:
    y = x.new_empty((m, n))
  z = x.new_empty((m, n)) if keep and (act or w_up is not None) else None
  z_up = x.new_empty((m, n)) if keep and w_up is not None else None
  if m:
    f = _layer_struct(x, w, w_up, b, b_up, act)
    f.y, f.ldy = y.data_ptr(), _ld(y)
    f.z = None if z is None else z.data_ptr()
    f.z_up = None if z_up is None else z_up.data_ptr()
    if r is not None:
      f.r, f.ldr = r.data_ptr(), _ld(r)
    with torch.cuda.device(x.device):
      native.policy_check(native.policy_lib().mjlab_layer_forward(ctypes.byref(f), _stream(x.device)), "mjlab_layer_forward")
  return y, z, z_up


class _Layer(torch.autograd.Function):
  @staticmethod
  def forward(ctx, x, w, w_up, b, b_up, r, act):
    y, z, z_up = _forward(x, w, w_up, b, b_up, r, act, keep=True)
    ctx.save_for_backward(x, w, w_up, z, z_up)
    ctx.act, ctx.has_bias = act, (b is not None, b_up is not None)
    return y

  @staticmethod
  @torch.autograd.function.once_differentiable
  def backward(ctx, dy):
    x, w, w_up, z, z_up = ctx.saved_tensors
    need_x, need_w, need_wu, need_b, need_bu, need_r, _ = ctx.needs_input_grad
    (m, k), n, gated = x.shape, w.shape[0], w_up is not None
    dr = dy if need_r else None
    if n > 1 and dy.stride(-1) != 1:
      dy = dy.contiguous()
    dx = x.new_empty((m, k)) if need_x else None
    dw = x.new_empty((n, k)) if need_w or need_wu else None
    dwu = x.new_empty((n, k)) if gated and dw is not None else None
    db = x.new_empty((n,)) if need_b or need_bu else None
    dbu = x.new_empty((n,)) if gated and db is not None else None
    if m == 0:
      for t in (dw, dwu, db, dbu):
        if t is not None:
          t.zero_()
    elif dx is not None or dw is not None or db is not None:
      g = LayerGrad()
      g.f = _layer_struct(x, w, w_up, None, None, ctx.act)
      g.f.z = None if z is None else z.data_ptr()
      g.f.z_up = None if z_up is None else z_up.data_ptr()
      g.dy, g.ld_dy = dy.data_ptr(), _ld(dy)
      for name, t in (("dx", dx), ("dw", dw), ("dw_up", dwu), ("db", db), ("db_up", dbu)):
        setattr(g, name, None if t is None else t.data_ptr())
      lib = native.policy_lib()
      need = lib.mjlab_layer_backward_workspace(ctypes.byref(g))
      native.policy_check(min(0, need), "mjlab_layer_backward_workspace")
      ws = torch.empty((max(need, 1),), dtype=torch.uint8, device=x.device)
      g.workspace, g.workspace_bytes = ws.data_ptr(), need
      with torch.cuda.device(x.device):
        native.policy_check(lib.mjlab_layer_backward(ctypes.byref(g), _stream(x.device)), "mjlab_layer_backward")
    return dx, dw if need_w else None, dwu if need_wu else None, db if need_b else None, dbu if need_bu else None, dr, None


def _arguments(what: str, x: torch.Tensor, w: torch.Tensor, activation: str) -> tuple:
  if x.dtype not in DTYPES or not x.is_cuda:
    raise TypeError(f"{what}: x must be a float32, float16 or bfloat16 device tensor, got {x.dtype} on {x.device} (there is no CPU fallback)")
  if activation not in ACTIVATIONS:
    raise ValueError(f"{what}: unknown activation {activation!r} (one of {', '.join(ACTIVATIONS)})")
  if x.dim() < 1 or w.dim() != 2 or x.shape[-1] < 1 or w.shape[0] < 1:
    raise ValueError(f"{what}: x (..., in) and weight (out, in) with in, out >= 1, got {tuple(x.shape)} and {tuple(w.shape)}")
  _check(w, f"{what}: weight", x, (w.shape[0], x.shape[-1]))
  return ACTIVATIONS[activation], w.shape[0]


def _run(x, w, w_up, b, b_up, r, act, lead: tuple, out):
  x2 = _rows(x, "x")
  if r is not None:
    r = _rows(r, "residual")
  grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x2, w, w_up, b, b_up, r))
  if out is not None:
    if grad:
      raise ValueError("out= takes no part in a graph of gradients: call it under torch.no_grad()")
    out2 = out.view(-1, out.shape[-1])
    _forward(x2, w, w_up, b, b_up, r, act, keep=False, y=out2)
    return out
  y = _Layer.apply(x2, w, w_up, b, b_up, r, act) if grad else _forward(x2, w, w_up, b, b_up, r, act, keep=False)[0]
  return y if x.dim() == 2 else y.view(*lead, w.shape[0])


def dense(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, activation: str = "none", residual: torch.Tensor | None = None,
          out: torch.Tensor | None = None) -> torch.Tensor:
  """``act(x weight^T + bias) + residual``: x (..., in), weight (out, in), bias (out), residual (..., out); activation one of ACTIVATIONS.
  ``out``: a contiguous tensor (..., out) to write (no gradients), which may be ``residual`` itself but shares no other memory
  with the inputs."""
  act, n = _arguments("dense", x, weight, activation)
  lead = tuple(x.shape[:-1])
  if bias is not None:
    _check(bias, "dense: bias", x, (n,))
  if residual is not None:
    _check(residual, "dense: residual", x, (*lead, n))
  if out is not None:
    _check_out("dense", out, x, (*lead, n), (weight, bias), residual)
  return _run(x, weight, None, bias, None, residual, act, lead, out)


def gated(x: torch.Tensor, weight: torch.Tensor, weight_up: torch.Tensor, bias: torch.Tensor | None = None, bias_up: torch.Tensor | None = None,
          activation: str = "silu", out: torch.Tensor | None = None) -> torch.Tensor:
  """``act(x weight^T + bias) * (x weight_up^T + bias_up)``: both products, the activation and the multiplication in one launch; weight and
  weight_up (out, in).  ``out`` as for dense()."""
  act, n = _arguments("gated", x, weight, activation)
  _check(weight_up, "gated: weight_up", x, tuple(weight.shape))
  lead = tuple(x.shape[:-1])
  for b, name in ((bias, "bias"), (bias_up, "bias_up")):
    if b is not None:
      _check(b, f"gated: {name}", x, (n,))
  if out is not None:
    _check_out("gated", out, x, (*lead, n), (weight, weight_up, bias, bias_up))
  return _run(x, weight, weight_up, bias, bias_up, None, act, lead, out)


def _span(t: torch.Tensor) -> tuple:
  """[first, last) byte of the memory that a non-empty tensor's elements lie in."""
  lo = t.data_ptr()
  return lo, lo + (sum((s - 1) * st for s, st in zip(t.shape, t.stride(), strict=True)) + 1) * t.element_size()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
  if not a.numel() or not b.numel():
    return False
  (a0, a1), (b0, b1) = _span(a), _span(b)
  return a0 < b1 and b0 < a1


def _check_out(what: str, out: torch.Tensor, like: torch.Tensor, shape: tuple, others: tuple = (), same_as: torch.Tensor | None = None) -> None:
  """`out` is written while `like` and `others` are still read: it may share no memory with them.  `same_as` may be `out` itself."""
  _check(out, f"{what}: out", like, shape)
  if not out.is_contiguous() or out.requires_grad:
    raise ValueError(f"{what}: out must be contiguous and must not require gradients")
  if same_as is not None and not (same_as.data_ptr() == out.data_ptr() and same_as.stride() == out.stride()):
    others = (*others, same_as)
  if any(t is not None and _overlap(out, t) for t in (like, *others)):
    raise ValueError(f"{what}: out overlaps an input")
