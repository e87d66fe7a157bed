"""What 16-bit operators keep on the way to their outputs: nothing of it is rounded to 16 bits, and none of it leaves the range of a float.

Layers: bounds, element by element, from the sizes alone (u: half a step of the type; u32 = 2^-24).  The sums before the activation are floats: off by at most
(k + 2) u32 sum |x w|, and the slope by that (Lipschitz with constant <= 1) and its evaluation, 16 u32 (1 + |z|).  dz is a float, formed with at most four
roundings.  The matrix cores read it as two bfloat16, which leaves at most 2^-8 of 2^-8 of it; a float16 that it meets is two bfloat16 as well (exactly), and the
product of the two second parts, another 2^-16, is not formed.  Three such products per term are summed in 32 bits, in any order.  Then one rounding to the type."""

import pytest
import torch
from test_gpu_policy_layers import TINY, U, U32, act, close, rand
from test_gpu_policy_memory import inputs, recurrence

pytestmark = pytest.mark.gpu

HALVES = [torch.float16, torch.bfloat16]
READ = {torch.float16: 2.0**-15, torch.bfloat16: 2.0**-16}


def check_gradients(m, k, n, dtype, name, gated, seed, dy_scale=1.0, x_scale=1.0, w_scale=1.0, shift=0.0, shift_up=0.0, want_bias=True, dy=None):
  from mjlab_amd import policy_ops

  gen = torch.Generator(device="cuda").manual_seed(seed)
  u, tiny, read = U[dtype], TINY[dtype], READ[dtype]
  x, w = rand(gen, m, k, dtype=dtype, scale=x_scale), rand(gen, n, k, dtype=dtype, scale=w_scale * k**-0.5)
  b = (rand(gen, n, dtype=torch.float32, scale=0.3) + shift).to(dtype)
  wu, bu = (rand(gen, n, k, dtype=dtype, scale=w_scale * k**-0.5), (rand(gen, n, dtype=torch.float32, scale=0.3) + shift_up).to(dtype)) if gated else (None, None)
  dy = rand(gen, m, n, dtype=torch.float32).mul(dy_scale).to(dtype) if dy is None else dy(gen)
  leaves = [t for t in (x, w, wu, *((b, bu) if want_bias else ())) if t is not None]
  for t in leaves:
    t.requires_grad_(True)
  y = policy_ops.gated(x, w, wu, b, bu, activation=name) if gated else policy_ops.dense(x, w, b, activation=name)
  grads = dict(zip([id(t) for t in leaves], torch.autograd.grad(y, leaves, dy), strict=True))
  with torch.no_grad():
    X, DY = x.double(), dy.double()

    def sums(wt, bt):
      return X @ wt.double().t() + bt.double(), (k + 2) * U32 * (X.abs() @ wt.double().abs().t() + bt.double().abs())

    z, ez = sums(w, b)
    f, df = act(z, name)
    ef, edf = 1.13 * ez + 16 * U32 * (1 + z.abs()), ez + 16 * U32 * (1 + z.abs()) + ((z.abs() <= ez).double() if name == "relu" else 0)
    if gated:
      up, eu = sums(wu, bu)
      dz, edz = [DY * up * df, DY * f], [DY.abs() * (edf * (up.abs() + eu) + df.abs() * eu), DY.abs() * ef]
    else:
      dz, edz = [DY * df], [DY.abs() * edf]
    edb = [d + 4 * U32 * (q.abs() + d) for q, d in zip(dz, edz, strict=True)]
    edz = [d + read * (q.abs() + d) for q, d in zip(dz, edb, strict=True)]
    ws = [w, wu] if gated else [w]
    dx = sum(d @ q.double() for d, q in zip(dz, ws, strict=True))
    ex = sum(d @ q.double().abs() + (6 * n + 2) * U32 * ((z_.abs() + d) @ q.double().abs()) for z_, d, q in zip(dz, edz, ws, strict=True))
    close(grads[id(x)], dx, ex + u * (dx.abs() + ex) + tiny, "dx")
    for z_, d, e, q, bias in zip(dz, edz, edb, ws, (b, bu), strict=False):
      dw, ew = z_.t() @ X, d.t() @ X.abs() + (3 * m + 2) * U32 * ((z_.abs() + d).t() @ X.abs())
      close(grads[id(q)], dw, ew + u * (dw.abs() + ew) + tiny, "dw")
      if want_bias:
        db, eb = z_.sum(0), e.sum(0) + (m + 2) * U32 * (z_.abs() + e).sum(0)
        close(grads[id(bias)], db, eb + u * (db.abs() + eb) + tiny, "db")
    return dz


SIZES = [(70, 40, 83), (5, 1999, 333), (1203, 1001, 1003)]  # small, few rows (split sums), more than 2^28 multiplications


@pytest.mark.parametrize("m,k,n", [(70, 40, 83), (6007, 70, 33), (1203, 1001, 1003)])
@pytest.mark.parametrize("name,gated", [("tanh", False), ("silu", False), ("silu", True)])
@pytest.mark.parametrize("scale", [2.0**-14, 2.0**-20])
def test_small_upstream_gradients_in_fp16(m, k, n, name, gated, scale):
  """As of a mean over many rows.  Weights of 16 keep dx inside fp16's normal numbers."""
  check_gradients(m, k, n, torch.float16, name, gated, seed=1, dy_scale=scale, x_scale=1 / 16, w_scale=16.0)


@pytest.mark.parametrize("m,k,n", SIZES)
def test_dz_of_a_gated_layer_beyond_fp16(m, k, n):
  """dg = dy * up * slope: about 1e5 and up to several 1e5, while dx and dw are finite."""
  dz = check_gradients(m, k, n, torch.float16, "silu", True, seed=2, dy_scale=200.0, x_scale=2.0**-9, w_scale=2.0**-9 * k**0.5, shift_up=1000.0, want_bias=False)
  assert dz[0].abs().max() > 65504


@pytest.mark.parametrize("m,k,n", SIZES)
def test_dz_of_a_dense_layer_beyond_fp16(m, k, n):
  """The slope of gelu is 1.13 at 1.41: dy = +-62000 gives dz = +-70000."""
  dz = check_gradients(m, k, n, torch.float16, "gelu", False, seed=3, x_scale=2.0**-9, w_scale=2.0**-9 * k**0.5, shift=1.41, want_bias=False,
                       dy=lambda gen: 62000 * (rand(gen, m, n, dtype=torch.float32).sign()).half())
  assert dz[0].abs().max() > 65504


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("name,gated", [("relu", False), ("silu", False), ("gelu", True)])
@pytest.mark.parametrize("m,k,n", [*SIZES, (2101, 45, 2103), (64, 1031, 517), (1, 1, 1), (131, 257, 65)])
def test_gradients(m, k, n, name, gated, dtype):
  check_gradients(m, k, n, dtype, name, gated, seed=4)


def only_rounded(got, want, e2, what):
  """The 2-norm of the error is that of rounding the exact result once, and what the roundings before it leave: `e2`, the expected square of that for each output,
  in all, with a factor of 4 for the spread."""
  own, err = (want.to(got.dtype).double() - want).norm(), (got.double() - want).norm()
  assert err <= own + 4 * e2.sum().sqrt(), f"{what}: off by {float(err / want.norm()):.3g} of its norm, rounding alone by {float(own / want.norm()):.3g}"


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("name,gated", [("elu", False), ("silu", False), ("gelu", False), ("tanh", False), ("sigmoid", False), ("silu", True)])
@pytest.mark.parametrize("m,k,n", [(1203, 1001, 1003), (2101, 45, 2103), (701, 333, 405)])
def test_gradients_are_as_exact_as_their_own_rounding(m, k, n, name, gated, dtype):
  """Roundings are independent, so a sum of terms t_i that are each off by at most r |t_i| is off by r sqrt(sum t_i^2) in the mean, and one of n additions in 32 bits
  by sqrt(n) u32 times the same (its partial sums are no larger in the mean)."""
  from mjlab_amd import policy_ops

  gen = torch.Generator(device="cuda").manual_seed(5)
  x, w, wu = rand(gen, m, k, dtype=dtype), *(rand(gen, n, k, dtype=dtype, scale=k**-0.5) for _ in range(2))
  dy = rand(gen, m, n, dtype=dtype)
  leaves = [t.requires_grad_(True) for t in ((x, w, wu) if gated else (x, w))]
  y = policy_ops.gated(*leaves, activation=name) if gated else policy_ops.dense(*leaves, activation=name)
  grads = torch.autograd.grad(y, leaves, dy)
  with torch.no_grad():
    X, DY, ws = x.double(), dy.double(), [t.double() for t in leaves[1:]]
    z = [X @ q.t() for q in ws]
    ez = [k**0.5 * U32 * ((X * X) @ (q * q).t()).sqrt() for q in ws]
    f, df = act(z[0], name)
    edf = ez[0] + 16 * U32 * (1 + z[0].abs())
    dz = [DY * z[1] * df, DY * f] if gated else [DY * df]
    edz = [DY.abs() * (edf * z[1].abs() + df.abs() * ez[1]), DY.abs() * edf * 1.13] if gated else [DY.abs() * edf]
    off = [(READ[dtype] + 4 * U32) * q.abs() + d for q, d in zip(dz, edz, strict=True)]
    only_rounded(grads[0], sum(d @ q for d, q in zip(dz, ws, strict=True)), sum((o * o + 6 * n * U32**2 * d * d) @ (q * q) for o, d, q in zip(off, dz, ws, strict=True)), "dx")
    for g, d, o in zip(grads[1:], dz, off, strict=True):
      only_rounded(g, d.t() @ X, (o * o + 3 * m * U32**2 * d * d).t() @ (X * X), "dw")


@pytest.mark.parametrize("name,slope", [("relu", 1.0), ("silu", 0.5), ("elu", 1.0)])
@pytest.mark.parametrize("m,n", [(3, 5), (2100, 2102)])
def test_the_slope_at_sums_that_fp16_cannot_hold(name, slope, m, n):
  """2^-15 * 2^-15 is 0 in fp16; its slope is that of a positive number."""
  from mjlab_amd import policy_ops

  x, w = (torch.full((s, 1), 2.0**-15, device="cuda", dtype=torch.float16, requires_grad=True) for s in (m, n))
  dx, dw = torch.autograd.grad(policy_ops.dense(x, w, activation=name), (x, w), torch.ones((m, n), device="cuda", dtype=torch.float16))
  assert torch.equal(dx.double(), torch.full_like(dx, slope * n * 2.0**-15).double()) and torch.equal(dw.double(), torch.full_like(dw, slope * m * 2.0**-15).double())


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("name", ["silu", "none"])
@pytest.mark.parametrize("m,k,n", [(40, 24, 30), (1203, 1001, 1003), (5, 1999, 333)])
def test_an_infinite_input_or_weight_stays_infinite(m, k, n, name, dtype):
  """Positive weights: the sums that the infinite number is in are infinite, so the slope there is 1 and dz = dy; dw has infinities of dy's sign in the infinite
  input's column, dx in the infinite weight's, and numbers elsewhere."""
  from mjlab_amd import policy_ops

  gen = torch.Generator(device="cuda").manual_seed(6)
  x, w = (torch.rand(s, generator=gen, device="cuda").add_(0.5).to(dtype) for s in ((m, k), (n, k)))
  dy = torch.where(torch.rand((m, n), generator=gen, device="cuda") < 0.5, -1.0, 1.0).to(dtype)
  for inputs_bad, (row, col) in ((True, (m - 2, 7)), (False, (n - 4, 11))):
    leaves = [x.clone(), w.clone()]
    leaves[0 if inputs_bad else 1][row, col] = float("inf")
    for t in leaves:
      t.requires_grad_(True)
    g = torch.autograd.grad(policy_ops.dense(*leaves, activation=name), leaves, dy)[1 if inputs_bad else 0]
    rest = torch.ones((k,), dtype=torch.bool, device="cuda")
    rest[col] = False
    assert torch.equal(g[:, col].float(), (dy[row, :] if inputs_bad else dy[:, row]).float() * float("inf")) and g[:, rest].isfinite().all()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("b,t,h,dk,dv", [(2, 1100, 2, 128, 128), (2, 1100, 3, 64, 64), (2, 1100, 2, 127, 33), (2, 300, 2, 128, 128), (3, 150, 2, 48, 80), (2, 200, 2, 32, 128), (2, 200, 2, 128, 32)])
def test_memory_is_as_exact_as_its_own_rounding(b, t, h, dk, dv, dtype):
  """Linear attention: a weighted key, a pair and the state are each read as two bfloat16 at least, 2^-16 of them left out; two of them are on the way to an output, 2^-15
  in all.  The sum of the terms' squares is the recurrence on squares.  What is wanted in the end as floats (the state, its gradient) is made of weighted keys as three bfloat16: off by roundings of
  32 bits alone, as many as there are steps and terms of a dot product, their root in the mean."""
  from mjlab_amd import policy_ops

  x = inputs(b, t, h, dk, dv, dtype, seed=18, resets=0.005, carry=True)
  leaves = [x[n].requires_grad_(True) for n in ("q", "k", "v", "state")]
  o, final = policy_ops.decay_attention(*leaves[:3], x["log_decay"], state=leaves[3], reset=x["reset"])
  got = [o, final, *torch.autograd.grad([o, final], leaves, [x["do"], x["dstate"]])]
  with torch.no_grad():
    lam, scale = x["log_decay"].double().exp(), dk**-0.5
    want = recurrence(*leaves[:3], lam, scale, leaves[3], x["reset"], None, x["do"], x["dstate"])
    squares = recurrence(*(z.double() ** 2 for z in leaves[:3]), lam**2, scale**2, leaves[3].double() ** 2, x["reset"], None, x["do"].double() ** 2, x["dstate"].double() ** 2)
    for name, g, w, s in zip(("o", "final", "dq", "dk", "dv", "dstate"), got, want, squares, strict=True):
      floats = name in ("final", "dstate")
      only_rounded(g, w, s * (4 * (t + max(dk, dv)) * U32**2 if floats else 2.0**-30), name)
