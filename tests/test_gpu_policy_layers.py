"""Dense and gated layers (mjlab_amd/policy_ops.py) against their formulas in 64 bits, element by element.

The bounds are worst cases, from the sizes alone.  u = half a step of the type; sums run in 32 bits (u32 = 2^-24), in any order, so a sum of
n products a_i b_i is off by at most (n + 2) u32 sum |a_i b_i|.  An activation is Lipschitz with constant <= 1.13 (silu, gelu) and its slope with
constant <= 1; evaluating either in 32 bits is off by at most 16 u32 of (1 + |z|).  Forward: error of z, times 1.13, plus evaluation, plus one
rounding.
Backward: the slope is taken at z rounded to the type (not rounded: gated layers, tanh, sigmoid, and elu, silu and gelu up to 2^22 sums), dz is
rounded to the type (up to 2^28 multiplications per product: to two numbers of it, u^2 instead of u), then one product and one rounding more.  The
slope of relu jumps at 0: where |z| is inside its error bound, the whole |dy| may be lost."""

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
U32 = 2.0**-24
TINY = {torch.float32: 2.0**-126, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-126}  # half a step of the subnormals (fp32: flushed)
SHAPES = [(1, 1, 1), (3, 5, 7), (64, 64, 64), (65, 129, 31), (130, 99, 257), (1, 512, 3), (300, 286, 117), (31, 33, 300), (2101, 45, 2103)]


def act(z, name):
  """(value, slope) in 64 bits."""
  if name == "none":
    return z, torch.ones_like(z)
  if name == "relu":
    return z.clamp(min=0), (z > 0).double()
  if name == "elu":
    return torch.where(z > 0, z, z.clamp(max=0).expm1()), z.clamp(max=0).exp()
  if name == "tanh":
    return z.tanh(), 1 - z.tanh() ** 2
  s = torch.sigmoid(z)
  if name == "sigmoid":
    return s, s * (1 - s)
  if name == "silu":
    return z * s, s * (1 + z * (1 - s))
  phi = 0.5 * (1 + torch.erf(z * 0.5**0.5))
  return z * phi, phi + z * torch.exp(-0.5 * z * z) * (2 * torch.pi) ** -0.5


def close(got, want, bound, what):
  err = (got.double() - want).abs()
  worst = (err / bound.clamp(min=1e-300)).max().item() if err.numel() else 0.0
  assert got.isfinite().all() and worst <= 1.0, f"{what}: {worst:.3g} times its bound, error {err.max().item():.3g}"


def rand(gen, *shape, dtype, scale=1.0):
  return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def check_layer(m, k, n, dtype, name, gated, bias, residual, x=None, seed=0):
  from mjlab_amd import policy_ops

  gen = torch.Generator(device="cuda").manual_seed(seed)
  u, tiny = U[dtype], TINY[dtype]
  x = rand(gen, m, k, dtype=dtype) if x is None else x
  w = rand(gen, n, k, dtype=dtype, scale=k**-0.5)
  wu = rand(gen, n, k, dtype=dtype, scale=k**-0.5) if gated else None
  b = rand(gen, n, dtype=dtype) if bias else None
  bu = rand(gen, n, dtype=dtype) if bias and gated else None
  r = rand(gen, m, n, dtype=dtype) if residual else None
  dy = rand(gen, m, n, dtype=dtype)
  leaves = [t for t in (x, w, wu, b, bu, r) if t is not None]
  for t in leaves:
    t.requires_grad_(True)
  call = (lambda: policy_ops.gated(x, w, wu, b, bu, activation=name)) if gated else (lambda: policy_ops.dense(x, w, b, activation=name, residual=r))
  y = call()
  grads = dict(zip([id(t) for t in leaves], torch.autograd.grad(y, leaves, dy), strict=True))
  with torch.no_grad():
    assert torch.equal(call(), y)  # the path that stores nothing for a backward pass computes the same
    X, W, DY = x.double(), w.double(), dy.double()

    def sums(wt, bt):
      B = 0 if bt is None else bt.double()
      return X @ wt.double().t() + B, (k + 2) * U32 * (X.abs() @ wt.double().abs().t() + (0 if bt is None else B.abs()))

    z, ez = sums(w, b)
    f, df = act(z, name)
    ef = 1.13 * ez + 16 * U32 * (1 + z.abs())
    uz, tz = (0, 0) if gated or name in ("tanh", "sigmoid") or (name in ("elu", "silu", "gelu") and m * n <= 1 << 22) else (u, tiny)  # (these sums are not rounded)
    edf = ez + uz * z.abs() + tz + 16 * U32 * (1 + z.abs()) + ((z.abs() <= ez).double() if name == "relu" else 0)
    if name == "none" and not gated:
      edf = torch.zeros_like(z)
    if gated:
      up, eu = sums(wu, bu)
      want, e = f * up, ef * (up.abs() + eu) + f.abs() * eu
      dz = [DY * up * df, DY * f]
      edz = [DY.abs() * (edf * (up.abs() + eu) + df.abs() * eu), DY.abs() * ef]
    else:
      want, e = (f, ef) if r is None else (f + r.double(), ef)
      dz, edz = [DY * df], [DY.abs() * edf]
    e = e + 4 * U32 * (want.abs() + (0 if r is None else r.double().abs()))
    close(y, want, e + u * (want.abs() + e) + tiny, "y")
    rounded = gated or name != "none"
    udz = 0 if not rounded else u if dtype == torch.float32 or (2 if gated else 1) * m * k * n > 1 << 28 else u * u
    edz = [d + (4 * U32 + udz) * (z_.abs() + d) + (tiny if rounded else 0) for z_, d in zip(dz, edz, strict=True)]
    ws = [w, wu] if gated else [w]
    dx = sum(d @ q.double() for d, q in zip(dz, ws, strict=True))
    ex = sum(d @ q.double().abs() + (2 * n + 2) * U32 * ((z_.abs() + d) @ q.double().abs()) for z_, d, q in zip(dz, edz, ws, strict=True))
    close(grads[id(x)], dx, ex + u * (dx.abs() + ex) + tiny, "dx")
    for z_, d, q, bias_ in zip(dz, edz, ws, [b, bu] if gated else [b], strict=True):
      dw, ew = z_.t() @ X, d.t() @ X.abs() + (m + 2) * U32 * ((z_.abs() + d).t() @ X.abs())
      close(grads[id(q)], dw, ew + u * (dw.abs() + ew) + tiny, "dw")
      if bias_ is not None:
        db, eb = z_.sum(0), d.sum(0) + (m + 2) * U32 * (z_.abs() + d).sum(0)
        close(grads[id(bias_)], db, eb + u * (db.abs() + eb) + tiny, "db")
    if r is not None:
      assert torch.equal(grads[id(r)], dy)


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("gated", [False, True])
def test_sizes(m, k, n, dtype, gated):
  check_layer(m, k, n, dtype, "silu", gated, bias=True, residual=not gated)


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("name", ["none", "relu", "elu", "tanh", "sigmoid", "silu", "gelu"])
@pytest.mark.parametrize("gated", [False, True])
def test_activations(name, dtype, gated):
  check_layer(77, 40, 83, dtype, name, gated, bias=False, residual=False, seed=1)
  check_layer(77, 40, 83, dtype, name, gated, bias=True, residual=False, seed=2)


@pytest.mark.parametrize("dtype", list(U))
def test_many_rows_split_the_weight_gradient(dtype):
  check_layer(5003, 70, 33, dtype, "gelu", False, bias=True, residual=True)
  check_layer(5003, 70, 33, dtype, "gelu", True, bias=True, residual=False)


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("m,k,n", [(1, 2048, 1024), (5, 1999, 333), (64, 1031, 517), (300, 1100, 200), (70, 300, 2049)])
@pytest.mark.parametrize("gated", [False, True])
def test_few_rows_split_the_sums(m, k, n, dtype, gated):
  check_layer(m, k, n, dtype, "silu", gated, bias=True, residual=not gated, seed=8)
  check_layer(m, k, n, dtype, "elu", gated, bias=False, residual=False, seed=9)


@pytest.mark.parametrize("dtype", list(U))
def test_row_strides_and_odd_addresses(dtype):
  gen = torch.Generator(device="cuda").manual_seed(3)
  wide = rand(gen, 70, 61, dtype=dtype)
  check_layer(70, 37, 19, dtype, "elu", False, bias=True, residual=True, x=wide[:, 3:40].detach())
  check_layer(70, 37, 19, dtype, "elu", True, bias=True, residual=False, x=wide[:, 3:40].detach())
  one = rand(gen, 1, 37, dtype=dtype).expand(70, 37)
  check_layer(70, 37, 19, dtype, "elu", False, bias=True, residual=False, x=one)


def test_leading_dimensions_and_out():
  from mjlab_amd import policy_ops

  gen = torch.Generator(device="cuda").manual_seed(4)
  x, w, b = rand(gen, 6, 5, 33, dtype=torch.float32), rand(gen, 17, 33, dtype=torch.float32), rand(gen, 17, dtype=torch.float32)
  r = rand(gen, 6, 5, 17, dtype=torch.float32)
  y = policy_ops.dense(x, w, b, activation="tanh", residual=r)
  assert y.shape == (6, 5, 17)
  assert torch.equal(policy_ops.dense(x.reshape(30, 33), w, b, activation="tanh", residual=r.reshape(30, 17)).view(6, 5, 17), y)
  out = torch.empty_like(y)
  assert policy_ops.dense(x, w, b, activation="tanh", residual=r, out=out) is out and torch.equal(out, y)
  assert policy_ops.dense(x, w, b, activation="tanh", residual=r, out=r) is r and torch.equal(r, y)  # the residual's own memory
  one = policy_ops.dense(x[0, 0], w, b)
  assert one.shape == (17,) and torch.equal(one, policy_ops.dense(x, w, b)[0, 0])
  swapped = x.transpose(0, 1)
  assert torch.equal(policy_ops.dense(swapped, w, b), policy_ops.dense(swapped.contiguous(), w, b))


def test_no_rows():
  from mjlab_amd import policy_ops

  x = torch.empty((0, 8), device="cuda", requires_grad=True)
  w = torch.randn((4, 8), device="cuda", requires_grad=True)
  b = torch.randn((4,), device="cuda", requires_grad=True)
  y = policy_ops.dense(x, w, b, activation="elu")
  assert y.shape == (0, 4)
  gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
  assert gx.shape == x.shape and not gw.any() and not gb.any()


def test_nan_and_infinity_stay_in_their_row():
  from mjlab_amd import policy_ops

  for dtype in U:
    x = torch.ones((200, 48), device="cuda", dtype=dtype)
    w = torch.ones((72, 48), device="cuda", dtype=dtype)
    x[7, 3], x[130, 47] = float("nan"), float("inf")
    for name in ("relu", "none", "elu", "silu", "gelu"):
      y = policy_ops.dense(x, w, activation=name)
      assert y[7].isnan().all() and (y[130] == float("inf")).all()
      rest = torch.ones(200, dtype=torch.bool, device="cuda")
      rest[[7, 130]] = False
      assert y[rest].isfinite().all()
    # a row whose sums are infinite in 16 bits has the limit of the slope, not infinity times zero
    xb = torch.full((4, 48), 200.0 if dtype == torch.float16 else 1.0, device="cuda", dtype=dtype, requires_grad=True)
    y = policy_ops.dense(xb, w * 10, activation="silu")
    (gx,) = torch.autograd.grad(y, xb, torch.full_like(y, 2.0**-10))
    assert torch.equal(gx.double(), torch.full_like(gx, 72 * 10 * 2.0**-10).double())


def test_gradient_against_differences():
  from mjlab_amd import policy_ops

  gen = torch.Generator(device="cuda").manual_seed(5)
  x, w, wu = (rand(gen, *s, dtype=torch.float32) for s in ((9, 12), (7, 12), (7, 12)))
  dy = rand(gen, 9, 7, dtype=torch.float32)
  for fn in (lambda a, c, d: policy_ops.dense(a, c, activation="gelu"), lambda a, c, d: policy_ops.gated(a, c, d, activation="tanh")):
    args = [t.clone().requires_grad_(True) for t in (x, w, wu)]
    grads = torch.autograd.grad((fn(*args) * dy).sum(), args, allow_unused=True)
    for i, g in enumerate(grads):
      if g is None:
        continue
      d = rand(gen, *args[i].shape, dtype=torch.float32)
      h = 2.0**-7
      with torch.no_grad():
        hi, lo = ((fn(*[t + s * h * d if j == i else t for j, t in enumerate(args)]).double() * dy.double()).sum() for s in (1, -1))
        got, want = (g.double() * d.double()).sum(), (hi - lo) / (2 * h)
        # central difference: third derivative term h^2 / 6 |f'''| |d|^3-sized plus rounding 2^-24 / h of the sum of magnitudes
        scale = (g.double().abs() * d.double().abs()).sum()
        assert (got - want).abs() <= 2.0**-6 * scale, (i, got.item(), want.item())


def test_graph_replays_equal_eager():
  """A layer's forward and backward captured into a hipGraph, replayed on changing inputs with eager work in between."""
  from mjlab_amd import policy_ops

  gen = torch.Generator(device="cuda").manual_seed(6)
  x, w, wu = (rand(gen, *s, dtype=torch.bfloat16) for s in ((600, 96), (130, 96), (130, 96)))
  b, dy = rand(gen, 130, dtype=torch.bfloat16), rand(gen, 600, 130, dtype=torch.bfloat16)

  def step(leaves):
    y = policy_ops.gated(*leaves[:3], leaves[3], leaves[3], activation="silu")
    return [y, *torch.autograd.grad(y, leaves, dy)]

  static = [t.clone().requires_grad_(True) for t in (x, w, wu, b)]
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    step(static)
  torch.cuda.current_stream().wait_stream(side)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    captured = step(static)
  for k in range(4):
    with torch.no_grad():
      static[0].copy_(x * (1 + k))
    graph.replay()
    torch.cuda.synchronize()
    eager = step([t.detach().clone().requires_grad_(True) for t in static])
    for a, c in zip(captured, eager, strict=True):
      assert torch.equal(a, c)


def test_other_stream():
  from mjlab_amd import policy_ops

  gen = torch.Generator(device="cuda").manual_seed(7)
  x, w = rand(gen, 3000, 512, dtype=torch.float32), rand(gen, 512, 512, dtype=torch.float32)
  want = policy_ops.dense(x, w, activation="elu")
  torch.cuda.synchronize()
  st = torch.cuda.Stream()
  st.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(st):
    got = policy_ops.dense(x * 1.0, w, activation="elu")
  st.synchronize()
  assert torch.equal(got, want)


def test_refusals_on_the_device():
  from mjlab_amd import policy_ops

  x, w = torch.randn((4, 8), device="cuda"), torch.randn((3, 8), device="cuda")
  bad = [
    (ValueError, lambda: policy_ops.dense(x, w, activation="mish")),
    (ValueError, lambda: policy_ops.dense(x, w[:, :7])),
    (TypeError, lambda: policy_ops.dense(x, w.half())),
    (TypeError, lambda: policy_ops.dense(x, w.cpu())),
    (TypeError, lambda: policy_ops.dense(x.double(), w.double())),
    (ValueError, lambda: policy_ops.dense(x, w, torch.randn(4, device="cuda"))),
    (ValueError, lambda: policy_ops.dense(x, w, residual=torch.randn((4, 1), device="cuda"))),
    (ValueError, lambda: policy_ops.dense(torch.randn((8, 4), device="cuda").t(), w)),
    (ValueError, lambda: policy_ops.dense(x, torch.randn((8, 3), device="cuda").t())),
    (ValueError, lambda: policy_ops.dense(x, w, out=torch.empty((3, 4), device="cuda").t())),
    (ValueError, lambda: policy_ops.dense(x, torch.randn((8, 8), device="cuda"), out=x)),
    (ValueError, lambda: policy_ops.gated(x, w, torch.randn((4, 8), device="cuda"))),
    (ValueError, lambda: policy_ops.dense(x.clone().requires_grad_(True), w, out=torch.empty((4, 3), device="cuda"))),
    (ValueError, lambda: policy_ops.dense(torch.empty((4, 0), device="cuda"), torch.empty((3, 0), device="cuda"))),
  ]
  for kind, call in bad:
    with pytest.raises(kind):
      call()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gated", [False, True])
def test_sizes_whose_dz_is_one_number(dtype, gated):
  check_layer(1203, 1001, 1003, dtype, "gelu", gated, bias=True, residual=False, seed=15)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gated", [False, True])
def test_an_infinite_upstream_gradient_stays_infinite(dtype, gated):
  """... in its row of dx: its rounding leaves nothing, not a NaN."""
  from mjlab_amd import policy_ops

  x, w, wu = (torch.rand((n, 24), device="cuda").to(dtype).add_(0.5).requires_grad_(True) for n in (40, 30, 30))
  y = policy_ops.gated(x, w, wu, activation="sigmoid") if gated else policy_ops.dense(x, w, activation="sigmoid")
  dy = torch.ones_like(y)
  dy[7, 3] = float("inf")
  dx, dw = torch.autograd.grad(y, [x, w], dy)
  bad = torch.zeros((40,), dtype=torch.bool, device="cuda")
  bad[7] = True
  assert (dx[7] == float("inf")).all() and dx[~bad].isfinite().all()
  assert (dw[3] == float("inf")).all() and dw[:3].isfinite().all() and dw[4:].isfinite().all()


def test_an_output_over_a_kept_input_is_noticed():
  from mjlab_amd import policy_ops

  x, w = torch.randn((6, 8), device="cuda"), torch.randn((8, 8), device="cuda", requires_grad=True)
  y = policy_ops.dense(x, w)
  with torch.no_grad():
    policy_ops.dense(torch.ones_like(x), w, out=x)
  with pytest.raises(RuntimeError, match="modified by an inplace operation"):
    y.sum().backward()
