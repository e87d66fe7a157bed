"""Operators of the policy network between an environment's observation rows and its action rows (include/mjlab_policy.h).

  dense(x, weight, bias, activation, residual)   y = act(x W^T + b) + r
  gated(x, weight, weight_up, ...)               y = act(x W^T + b) * (x W_up^T + b_up)
  decay_attention(q, k, v, log_decay, ...)       S_t = decay S_{t-1} + k_t v_t^T, o_t = scale q_t S_t over stored steps, S cut at resets
  decay_attention_step(q, k, v, log_decay, state, ...)  the same for one control step

float32, float16 or bfloat16, the same type everywhere, sums and states in 32 bits, each output and gradient rounded once: what lies between them is held to 2^-15
or better of each term of a sum, and has a float's range (a float16 layer's upstream gradient may be tiny, or its product with the slope beyond 65504).  The first
three are differentiable once, in reverse mode (no vmap, no forward mode), in every tensor argument but log_decay.  Every call enqueues on torch's current stream of
the tensors' device and may be captured into a hipGraph; nothing synchronises.  The last dimension of an argument must be contiguous, rows may
be any distance apart.  No fallback: without the HIP library, or for a tensor that is not on the GPU, these raise.

A backward pass that is captured into a graph must not share leaves with an eager autograd graph that is still alive (torch synchronises
with the eager stream inside the capture): capture from leaves of its own, as for any other torch operation."""

from __future__ import annotations

import ctypes
import struct

import torch

from . import native

_vp, _ll = ctypes.c_void_p, ctypes.c_longlong

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # MJLAB_DTYPE_*
ACTIVATIONS = {"none": 0, "relu": 1, "elu": 2, "tanh": 3, "sigmoid": 4, "silu": 5, "gelu": 6}  # MJLAB_ACT_*; gelu: the exact one (erf)


class Layer(ctypes.Structure):  # mjlab_layer_t
  _fields_ = [("dtype", ctypes.c_int), ("act", ctypes.c_int), ("z_is_y", ctypes.c_int), ("z_bytes", ctypes.c_int), ("rows", _ll), ("inp", _ll), ("out", _ll),
              ("x", _vp), ("w", _vp), ("w_up", _vp), ("b", _vp), ("b_up", _vp), ("r", _vp),
              ("ldx", _ll), ("ldw", _ll), ("ldw_up", _ll), ("ldr", _ll), ("ldy", _ll), ("y", _vp), ("z", _vp), ("z_up", _vp),
              ("workspace", _vp), ("workspace_bytes", _ll)]  # fmt: skip


class LayerGrad(ctypes.Structure):  # mjlab_layer_grad_t
  _fields_ = [("f", Layer), ("dy", _vp), ("ld_dy", _ll), ("dx", _vp), ("dw", _vp), ("dw_up", _vp), ("db", _vp), ("db_up", _vp),
              ("workspace", _vp), ("workspace_bytes", _ll)]  # fmt: skip


class Rows(ctypes.Structure):  # mjlab_decay_rows_t
  _fields_ = [("p", _vp), ("batch", _ll), ("time", _ll), ("head", _ll)]


class Decay(ctypes.Structure):  # mjlab_decay_t
  _fields_ = [("dtype", ctypes.c_int), ("reset_bytes", ctypes.c_int), ("batch", _ll), ("length", _ll), ("heads", ctypes.c_int), ("dk", ctypes.c_int),
              ("dv", ctypes.c_int), ("scale", ctypes.c_float), ("q", Rows), ("k", Rows), ("v", Rows), ("o", Rows), ("log_decay", _vp), ("state", _vp),
              ("state_out", _vp), ("reset", _vp), ("reset_batch", _ll), ("reset_time", _ll), ("lengths", _vp), ("workspace", _vp),
              ("workspace_bytes", _ll)]  # fmt: skip


class DecayGrad(ctypes.Structure):  # mjlab_decay_grad_t
  _fields_ = [("f", Decay), ("d_out", Rows), ("dq", Rows), ("dk", Rows), ("dv", Rows), ("d_state_out", _vp), ("d_state", _vp), ("segments", _vp)]


# A call's argument struct is packed in one go (setting two dozen ctypes fields one by one takes longer than a small layer's kernel): the layouts of the
# mirrors above, which native.policy_lib() holds against the library's.
_LAYER = struct.Struct("@4i3q6P5q3PPq")
_LAYER_GRAD = struct.Struct("@4i3q6P5q3PPq" "Pq5PPq")
_ROWS = "P3q"
_DECAY = struct.Struct("@2i2q3if" + 4 * _ROWS + "3PP2q2Pq")
_DECAY_GRAD = struct.Struct("@2i2q3if" + 4 * _ROWS + "3PP2q2Pq" + 4 * _ROWS + "3P")
assert _LAYER.size == ctypes.sizeof(Layer) and _LAYER_GRAD.size == ctypes.sizeof(LayerGrad)
assert _DECAY.size == ctypes.sizeof(Decay) and _DECAY_GRAD.size == ctypes.sizeof(DecayGrad)

_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None


def _call(fn: str, packed: bytes, dev: torch.device) -> None:
  """Enqueue on torch's current stream of `dev`."""
  lib = native.policy_lib()
  index = dev.index
  stream = _raw_stream(index) if _raw_stream else torch.cuda.current_stream(dev).cuda_stream
  if torch.cuda.current_device() == index:
    rc = getattr(lib, fn)(packed, stream)
  else:
    with torch.cuda.device(dev):
      rc = getattr(lib, fn)(packed, stream)
  if rc:
    native.policy_check(rc, fn)


# A tensor of the caller's that a kernel wrote: autograd is to notice where an earlier operation kept it for its backward pass.
_written = torch.autograd.graph.increment_version


def _ptr(t: torch.Tensor | None) -> int:
  return 0 if t is None else t.data_ptr()


def _check(t: torch.Tensor, what: str, name: str, like: torch.Tensor, shape: tuple) -> torch.Tensor:
  if t.dtype != like.dtype or t.device != like.device:
    raise TypeError(f"{what}: {name}: expected {like.dtype} on {like.device}, got {t.dtype} on {t.device}")
  if t.shape != shape:
    raise ValueError(f"{what}: {name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
  if shape and shape[-1] > 1 and t.stride(-1) != 1:
    raise ValueError(f"{what}: {name}: the last dimension must be contiguous (shape {tuple(t.shape)}, strides {t.stride()})")
  return t


def _rows(t: torch.Tensor, what: str) -> torch.Tensor:
  """(rows, last) over any leading dimensions, without a copy where the strides allow it."""
  if t.shape[-1] > 1 and t.stride(-1) != 1:
    raise ValueError(f"{what}: the last dimension must be contiguous (shape {tuple(t.shape)}, strides {t.stride()})")
  return t if t.dim() == 2 else t.reshape(-1, t.shape[-1])


def _ld(t: torch.Tensor) -> int:
  return t.stride(0) if t.shape[0] > 1 else t.shape[1]


# float32 layers whose slope the output gives store nothing else for the backward pass.  16 bits: 1 + y and 1 - y^2 would cancel, and a rounded sum shows in the
# gradients (tanh: 1.54 times the error of their own rounding, elu 1.14; relu: sums below half of fp16's smallest number have slope 0), so the sums are kept as floats.
_FROM_OUTPUT = {ACTIVATIONS[a] for a in ("relu", "elu", "tanh", "sigmoid")}


def _from_output(x, w_up, r, act: int) -> bool:
  return x.dtype == torch.float32 and w_up is None and r is None and act in _FROM_OUTPUT


def _forward(x, w, w_up, b, b_up, r, act: int, keep: bool, y=None):
  """-> y, z, z_up (z: the sums before the activation where the backward pass will want them)."""
  (m, k), n = x.shape, w.shape[0]
  if y is None:
    y = x.new_empty((m, n))
  z = z_up = None
  if m:
    dtype, lds = DTYPES[x.dtype], (_ld(x), _ld(w), 0 if w_up is None else _ld(w_up), 0 if r is None else _ld(r), _ld(y))
    inputs = (x.data_ptr(), w.data_ptr(), _ptr(w_up), _ptr(b), _ptr(b_up), _ptr(r))
    if keep and w_up is not None:
      if not native.policy_lib().mjlab_layer_recomputes(_LAYER.pack(dtype, act, 0, 0, m, k, n, *inputs, *lds, 0, 0, 0, 0, 0)):
        z, z_up = (torch.empty((m, n), dtype=torch.float32, device=x.device) for _ in range(2))
    elif keep and act and not _from_output(x, w_up, r, act):
      z = torch.empty((m, n), dtype=torch.float32, device=x.device)
    args = (dtype, act, 0, 0 if z is None else z.element_size(), m, k, n, *inputs, *lds, y.data_ptr(), _ptr(z), _ptr(z_up))
    need = native.policy_lib().mjlab_layer_forward_workspace(_LAYER.pack(*args, 0, 0))
    if need < 0:
      native.policy_check(need, "mjlab_layer_forward_workspace")
    ws = torch.empty((need,), dtype=torch.uint8, device=x.device) if need else None
    _call("mjlab_layer_forward", _LAYER.pack(*args, _ptr(ws), need), x.device)
  return y, z, z_up


class _Layer(torch.autograd.Function):
  @staticmethod
  def forward(ctx, x, w, w_up, b, b_up, r, act):
    y, z, z_up = _forward(x, w, w_up, b, b_up, r, act, keep=True)
    ctx.z_is_y = _from_output(x, w_up, r, act)
    again = w_up is not None and z is None
    ctx.save_for_backward(x, w, w_up, y if ctx.z_is_y else z, z_up, b if again else None, b_up if again else None)
    ctx.act = act
    return y

  @staticmethod
  @torch.autograd.function.once_differentiable
  def backward(ctx, dy):
    x, w, w_up, z, z_up, b, b_up = ctx.saved_tensors  # (the biases where the sums are formed again)
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

      def pack(workspace: int, size: int) -> bytes:
        return _LAYER_GRAD.pack(DTYPES[x.dtype], ctx.act, ctx.z_is_y, 0 if z is None else z.element_size(), m, k, n, x.data_ptr(), w.data_ptr(), _ptr(w_up),
                                _ptr(b), _ptr(b_up), 0, _ld(x), _ld(w),
                                _ld(w_up) if gated else 0, 0, 0, 0, _ptr(z), _ptr(z_up), 0, 0, dy.data_ptr(), _ld(dy), _ptr(dx), _ptr(dw), _ptr(dwu), _ptr(db), _ptr(dbu),
                                workspace, size)  # fmt: skip

      need = native.policy_lib().mjlab_layer_backward_workspace(pack(0, 0))
      if need < 0:
        native.policy_check(need, "mjlab_layer_backward_workspace")
      ws = torch.empty((need,), dtype=torch.uint8, device=x.device) if need else None
      _call("mjlab_layer_backward", pack(_ptr(ws), need), x.device)
    return dx, dw if need_w else None, dwu if need_wu else None, db if need_b else None, dbu if need_bu else None, dr, None


def _arguments(what: str, x: torch.Tensor, w: torch.Tensor, activation: str) -> tuple:
  if x.dtype not in DTYPES or not x.is_cuda:
    raise TypeError(f"{what}: x must be a float32, float16 or bfloat16 device tensor, got {x.dtype} on {x.device} (there is no CPU fallback)")
  if activation not in ACTIVATIONS:
    raise ValueError(f"{what}: unknown activation {activation!r} (one of {', '.join(ACTIVATIONS)})")
  if x.dim() < 1 or w.dim() != 2 or x.shape[-1] < 1 or w.shape[0] < 1:
    raise ValueError(f"{what}: x (..., in) and weight (out, in) with in, out >= 1, got {tuple(x.shape)} and {tuple(w.shape)}")
  _check(w, what, "weight", x, (w.shape[0], x.shape[-1]))
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
    _written(out)
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
    _check(bias, "dense", "bias", x, (n,))
  if residual is not None:
    _check(residual, "dense", "residual", x, (*lead, n))
  if out is not None:
    _check_out("dense", out, x, (*lead, n), (weight, bias), residual)
  return _run(x, weight, None, bias, None, residual, act, lead, out)


def gated(x: torch.Tensor, weight: torch.Tensor, weight_up: torch.Tensor, bias: torch.Tensor | None = None, bias_up: torch.Tensor | None = None,
          activation: str = "silu", out: torch.Tensor | None = None) -> torch.Tensor:
  """``act(x weight^T + bias) * (x weight_up^T + bias_up)``: both products, the activation and the multiplication in one launch; weight and
  weight_up (out, in).  ``out`` as for dense()."""
  act, n = _arguments("gated", x, weight, activation)
  _check(weight_up, "gated", "weight_up", x, weight.shape)
  lead = tuple(x.shape[:-1])
  for b, name in ((bias, "bias"), (bias_up, "bias_up")):
    if b is not None:
      _check(b, "gated", name, x, (n,))
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
  _check(out, what, "out", like, shape)
  if not out.is_contiguous() or out.requires_grad:
    raise ValueError(f"{what}: out must be contiguous and must not require gradients")
  if same_as is not None and not (same_as.data_ptr() == out.data_ptr() and same_as.stride() == out.stride()):
    others = (*others, same_as)
  if any(t is not None and _overlap(out, t) for t in (like, *others)):
    raise ValueError(f"{what}: out overlaps an input")


MAX_HEAD_DIM = 128  # MJLAB_DECAY_MAX_DIM


def _decay_arguments(what: str, q, k, v, log_decay, state, reset, lead: tuple) -> None:
  """Checks shared by the chunked form (lead = batch, length) and the step (lead = batch)."""
  if q.dtype not in DTYPES or not q.is_cuda:
    raise TypeError(f"{what}: q must be a float32, float16 or bfloat16 device tensor, got {q.dtype} on {q.device} (there is no CPU fallback)")
  h, dk = q.shape[-2:]
  _check(k, what, "k", q, (*lead, h, dk))
  if v.dim() != q.dim():
    raise ValueError(f"{what}: v must have the dimensions of q, got {tuple(v.shape)}")
  dv = v.shape[-1]
  _check(q, what, "q", q, (*lead, h, dk))
  _check(v, what, "v", q, (*lead, h, dv))
  if h < 1 or not 1 <= dk <= MAX_HEAD_DIM or not 1 <= dv <= MAX_HEAD_DIM:
    raise ValueError(f"{what}: at least one head, and head sizes in [1, {MAX_HEAD_DIM}], got {h} heads of {dk} and {dv}")
  if log_decay.dtype != torch.float32 or log_decay.device != q.device or tuple(log_decay.shape) != (h,) or not log_decay.is_contiguous():
    raise ValueError(f"{what}: log_decay must be a contiguous float32 tensor ({h},) on {q.device}, got {log_decay.dtype} {tuple(log_decay.shape)} on {log_decay.device}")
  if log_decay.requires_grad:
    raise ValueError(f"{what}: the decays are constants; log_decay must not require gradients")
  if state is not None and (state.dtype != torch.float32 or state.device != q.device or tuple(state.shape) != (lead[0], h, dk, dv) or not state.is_contiguous()):
    raise ValueError(f"{what}: state must be a contiguous float32 tensor {(lead[0], h, dk, dv)} on {q.device}, got {state.dtype} {tuple(state.shape)} on {state.device}")
  if reset is not None and (reset.dtype not in (torch.bool, torch.uint8, torch.int32) or reset.device != q.device or tuple(reset.shape) != lead):
    raise ValueError(f"{what}: reset must be a bool, uint8 or int32 tensor {lead} on {q.device}, got {reset.dtype} {tuple(reset.shape)} on {reset.device}")


def _decay_pack(q, k, v, o, log_decay, scale: float, state, state_out, reset, lengths) -> tuple:
  """The values of a mjlab_decay_t up to its workspace; q, k, v, o: (batch, length, heads, d), o None: not used."""
  b, n, h, dk = q.shape
  r = (0, 0, 0, 0) if reset is None else (reset.element_size(), reset.data_ptr(), reset.stride(0), reset.stride(1))
  return (DTYPES[q.dtype], r[0], b, n, h, dk, v.shape[3], scale, *_strided(q), *_strided(k), *_strided(v), *_strided(o), log_decay.data_ptr(), _ptr(state),
          _ptr(state_out), *r[1:], _ptr(lengths))  # fmt: skip


def _strided(t: torch.Tensor | None) -> tuple:
  return (0, 0, 0, 0) if t is None else (t.data_ptr(), *t.stride()[:3])


def _rows_like(t: torch.Tensor, d: int) -> torch.Tensor:
  """A new (batch, length, heads, d) tensor with the batch and time axes in memory in the order they have in `t`."""
  b, n, h, _ = t.shape
  return t.new_empty((n, b, h, d)).transpose(0, 1) if b > 1 and n > 1 and t.stride(1) > t.stride(0) else t.new_empty((b, n, h, d))


def _decay_launch(fn: str, layout: struct.Struct, head: tuple, tail: tuple, dev: torch.device) -> torch.Tensor | None:
  """-> the workspace, which the forward pass leaves the states of its segments in."""
  need = native.policy_lib().mjlab_decay_workspace(_DECAY.pack(*head, 0, 0))
  if need < 0:
    native.policy_check(need, "mjlab_decay_workspace")
  ws = torch.empty((need,), dtype=torch.uint8, device=dev) if need else None
  _call(fn, layout.pack(*head, _ptr(ws), need, *tail), dev)
  return ws


def _decay_forward(q, k, v, state, log_decay, scale, reset, lengths):
  b, n, h, dk = q.shape
  o = _rows_like(q, v.shape[3])
  if b == 0 or n == 0:
    final = q.new_zeros((b, h, dk, v.shape[3]), dtype=torch.float32) if state is None else state.clone()
    return o, final, None
  final = torch.empty((b, h, dk, v.shape[3]), dtype=torch.float32, device=q.device)
  ws = _decay_launch("mjlab_decay_forward", _DECAY, _decay_pack(q, k, v, o, log_decay, scale, state, final, reset, lengths), (), q.device)
  return o, final, ws


class _DecayAttention(torch.autograd.Function):
  @staticmethod
  def forward(ctx, q, k, v, state, log_decay, scale, reset, lengths):
    o, final, segments = _decay_forward(q, k, v, state, log_decay, scale, reset, lengths)
    ctx.save_for_backward(q, k, v, state, log_decay, reset, lengths, segments)
    ctx.scale = scale
    ctx.set_materialize_grads(False)
    return o, final

  @staticmethod
  @torch.autograd.function.once_differentiable
  def backward(ctx, do, dfinal):
    q, k, v, state, log_decay, reset, lengths, segments = ctx.saved_tensors
    need_q, need_k, need_v, need_s = ctx.needs_input_grad[:4]
    if do is None and dfinal is None:
      return (None,) * 8
    b, n, h, dk = q.shape
    if b == 0 or n == 0:
      ds = None
      if need_s:
        ds = torch.zeros_like(state) if dfinal is None else dfinal
      return tuple(torch.zeros_like(t) if need else None for t, need in ((q, need_q), (k, need_k), (v, need_v))) + (ds, None, None, None, None)
    if do is None:
      do = torch.zeros((1, 1, 1, v.shape[3]), dtype=q.dtype, device=q.device).expand(b, n, h, v.shape[3])
    elif v.shape[3] > 1 and do.stride(3) != 1:
      do = do.contiguous()
    dfinal = None if dfinal is None else dfinal.contiguous()
    dq = _rows_like(q, dk) if need_q else None
    dk_ = _rows_like(k, dk) if need_k else None
    dv = _rows_like(v, v.shape[3]) if need_v or need_s else None
    ds = torch.empty_like(state) if need_s else None
    _decay_launch("mjlab_decay_backward", _DECAY_GRAD, _decay_pack(q, k, v, None, log_decay, ctx.scale, state, None, reset, lengths),
                  (*_strided(do), *_strided(dq), *_strided(dk_), *_strided(dv), _ptr(dfinal), _ptr(ds), _ptr(segments)), q.device)
    return dq, dk_, dv if need_v else None, ds, None, None, None, None


def decay_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, scale: float | None = None, state: torch.Tensor | None = None,
                    reset: torch.Tensor | None = None, lengths: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
  """Linear attention with a decay per head over stored steps -> (o (batch, length, heads, dv), final state (batch, heads, dk, dv) float32).

  q, k (batch, length, heads, dk), v (batch, length, heads, dv): any strides with a contiguous last dimension, so a time-major rollout buffer goes in
  as ``buffer.transpose(0, 1)``.  ``log_decay`` (heads,) float32, constants (<= 0; a positive one grows).  ``scale`` defaults to dk ** -0.5.  ``state``: what
  was carried into the first step (zeros if None).  ``reset`` (batch, length), non-zero where a step is the first of an episode: nothing is carried into
  it.  ``lengths`` (batch,) int32: sequence b ends before step lengths[b]; o is zero behind it and the final state is the one at its end.  A NaN or
  infinity of one step does not reach earlier steps or other episodes."""
  if q.dim() != 4:
    raise ValueError(f"decay_attention: q must be (batch, length, heads, dk), got {tuple(q.shape)}")
  lead = tuple(q.shape[:2])
  _decay_arguments("decay_attention", q, k, v, log_decay, state, reset, lead)
  if lengths is not None and (lengths.dtype != torch.int32 or lengths.device != q.device or tuple(lengths.shape) != lead[:1] or not lengths.is_contiguous()):
    raise ValueError(f"decay_attention: lengths must be a contiguous int32 tensor {lead[:1]} on {q.device}, got {lengths.dtype} {tuple(lengths.shape)} on {lengths.device}")
  scale = q.shape[3] ** -0.5 if scale is None else float(scale)
  if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, state)):
    return _DecayAttention.apply(q, k, v, state, log_decay, scale, reset, lengths)
  return _decay_forward(q, k, v, state, log_decay, scale, reset, lengths)[:2]


def decay_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, state: torch.Tensor, scale: float | None = None,
                         reset: torch.Tensor | None = None, out: torch.Tensor | None = None, out_state: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
  """One control step of the same recurrence -> (o (batch, heads, dv), state).  q, k (batch, heads, dk), v (batch, heads, dv); ``state`` (batch, heads, dk, dv) float32 is
  updated in place, or left alone and written to ``out_state``.  ``reset`` (batch,): non-zero where the environment was reset before this step (what
  PhysicsRollout.step() returned).  No gradients: an update replays stored steps through decay_attention()."""
  if q.dim() != 3:
    raise ValueError(f"decay_attention_step: q must be (batch, heads, dk), got {tuple(q.shape)}")
  b, h, dk = q.shape
  _decay_arguments("decay_attention_step", q, k, v, log_decay, state, reset, (b,))
  dv = v.shape[2]
  if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, state)):
    raise ValueError("decay_attention_step takes no part in a graph of gradients: call it under torch.no_grad()")
  if out_state is None:
    out_state = state
  elif out_state is not state:
    if out_state.dtype != torch.float32 or out_state.device != q.device or out_state.shape != state.shape or not out_state.is_contiguous():
      raise ValueError("decay_attention_step: out_state must be like state")
    if out_state.data_ptr() != state.data_ptr() and _overlap(out_state, state):
      raise ValueError("decay_attention_step: out_state overlaps state")
  if any(_overlap(out_state, t) for t in (q, k, v)):
    raise ValueError("decay_attention_step: the state overlaps an input")
  own = out is None
  if own:
    out = q.new_empty((b, h, dv))
  else:
    _check_out("decay_attention_step", out, q, (b, h, dv), (k, v, state, out_state))
  if b:
    r = (0, 0, 0) if reset is None else (reset.element_size(), reset.data_ptr(), reset.stride(0))
    rows = [x for t in (q, k, v, out) for x in (t.data_ptr(), t.stride(0), 0, t.stride(1))]
    _call("mjlab_decay_step", _DECAY.pack(DTYPES[q.dtype], r[0], b, 1, h, dk, dv, dk**-0.5 if scale is None else scale, *rows, log_decay.data_ptr(), state.data_ptr(),
                                          out_state.data_ptr(), r[1], r[2], 0, 0, 0, 0), q.device)  # fmt: skip
    _written(out_state)
    if not own:
      _written(out)
  return out, out_state
