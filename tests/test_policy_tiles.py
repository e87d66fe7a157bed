"""Every kernel that a layer's sizes can choose -- tile, epilogue, sums split or not, for each product and type -- at sizes that are odd in all three dimensions.

The first test holds the sizes to what they are here for, without a GPU; the others run them.  Errors are held against what independent roundings leave (u: half a step of
the type, u32 = 2^-24): a sum of terms t_i that are each off by at most r |t_i| is off by r sqrt(sum t_i^2) in the mean, one of n additions in 32 bits by
sqrt(n) u32 times the same, a matrix instruction's terms are off by READ (float32: as three bfloat16 whose last products are left out; dz in 16 bits: as two bfloat16;
what has 16 bits itself: not at all), and 16 u32 (1 + |z|) for an activation or its slope.  All outputs together: four times that besides their own rounding; each one
by itself: twelve times."""

import ctypes
import sys
from pathlib import Path

import pytest
import torch
from test_gpu_policy_layers import TINY, U, U32, act, rand

from mjlab_amd import native, policy_ops

SHAPES = [(35, 137, 133), (37, 2091, 2987), (16199, 393, 203), (4715, 645, 2821), (263, 805, 2345), (16563, 619, 333), (13853, 1739, 193), (10307, 1699, 135), (17207, 67, 2869)]
KINDS = [("none", False), ("silu", False), ("silu", True)]  # (activation, gated): without an activation the backward products read dy itself


def chosen(m, k, n, dtype, name, gated):
  f = policy_ops.Layer()
  f.dtype, f.act, f.rows, f.inp, f.out, f.x, f.w, f.ldx, f.ldw = policy_ops.DTYPES[dtype], policy_ops.ACTIVATIONS[name], m, k, n, 64, 64, k, k
  if gated:
    f.w_up, f.ldw_up = 64, k
  return tuple(native.policy_lib().mjlab_layer_tile(ctypes.byref(f), product) for product in range(3))


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("name,gated", KINDS)
def test_these_sizes_reach_every_kernel(dtype, name, gated):
  wide = dtype == torch.float32
  want = [
    {64, 128, -64, -128} if wide else {64, 128, 256, -64},  # y
    {64, 128, -64, -128, 256, -256} if not wide and name == "none" else {64, 128, -64, -128},  # dx
    {-64, -128} if gated else {64, 128, -64, -128},  # dw (a gated layer's two are always joined by a second launch)
  ]
  tiles = [chosen(*s, dtype, name, gated) for s in SHAPES]
  for product in range(3):
    assert {t[product] for t in tiles} == want[product], product
  if gated and not wide:  # up to 1024 inputs the sums are formed again, in the tile of an unsplit forward product; beyond, they are stored
    assert {t[0] for s, t in zip(SHAPES, tiles, strict=True) if s[1] <= 1024 and t[0] > 0} == {64, 128, 256} and any(s[1] > 1024 for s in SHAPES)
  bad = policy_ops.Layer()
  assert native.policy_lib().mjlab_layer_tile(ctypes.byref(bad), 0) == 0 and native.policy_lib().mjlab_layer_tile(None, 0) == 0


READ = {torch.float32: (2.0**-22, 2.0**-22), torch.float16: (0.0, 2.0**-15), torch.bfloat16: (0.0, 2.0**-16)}  # (forward and without dz, with dz)


def near(got, want, e2, dtype, what):
  """`e2`: the expected square of each output's error before its own rounding."""
  err, own = (got.double() - want).abs(), (want.to(dtype).double() - want).abs()
  assert got.isfinite().all() and err.norm() <= own.norm() + 4 * e2.sum().sqrt(), f"{what}: off by {float(err.norm() / want.norm()):.3g} of its norm"
  worst = (err / (U[dtype] * want.abs() + 12 * (1 + U[dtype]) * e2.sqrt() + TINY[dtype])).max()
  assert worst <= 1, f"{what}: {float(worst):.3g} times its bound"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("name,gated", KINDS)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_every_kernel(m, k, n, name, gated, dtype):
  gen = torch.Generator(device="cuda").manual_seed(m)
  ahead, behind = READ[dtype]
  behind = ahead if name == "none" else behind
  x, ws = rand(gen, m, k, dtype=dtype), [rand(gen, n, k, dtype=dtype, scale=k**-0.5) for _ in range(2 if gated else 1)]
  bs = [rand(gen, n, dtype=dtype, scale=0.3) for _ in ws]
  r = None if gated else rand(gen, m, n, dtype=dtype)
  dy = rand(gen, m, n, dtype=dtype)
  leaves = [t.requires_grad_(True) for t in (x, *ws, *bs, *(() if gated else (r,)))]
  y = policy_ops.gated(x, *ws, *bs, activation=name) if gated else policy_ops.dense(x, *ws, *bs, activation=name, residual=r)
  gx, *rest = torch.autograd.grad(y, leaves, dy)
  with torch.no_grad():
    X, DY, W = x.double(), dy.double(), [w.double() for w in ws]
    zs = [X @ w.t() + b.double() for w, b in zip(W, bs, strict=True)]
    ezs = [(ahead + k**0.5 * U32) * ((X * X) @ (w * w).t() + b.double() ** 2).sqrt() for w, b in zip(W, bs, strict=True)]
    f, df = act(zs[0], name)
    ef, edf = 1.13 * ezs[0] + 16 * U32 * (1 + zs[0].abs()), ezs[0] + 16 * U32 * (1 + zs[0].abs())
    if name == "none":
      ef, edf = ezs[0], torch.zeros_like(f)
    if gated:
      near(y, f * zs[1], (ef * zs[1]) ** 2 + (f * ezs[1]) ** 2 + (4 * U32 * f * zs[1]) ** 2, dtype, "y")
      dz, edz = [DY * zs[1] * df, DY * f], [DY.abs() * (edf * zs[1].abs() + df.abs() * ezs[1]), DY.abs() * ef]
    else:
      near(y, f + r.double(), ef**2 + (4 * U32 * (f.abs() + r.double().abs())) ** 2, dtype, "y")
      dz, edz = [DY * df], [DY.abs() * edf]
      assert torch.equal(rest.pop(), dy)
    off = [e + 4 * U32 * d.abs() for d, e in zip(dz, edz, strict=True)]
    mul = [(o + behind * d.abs()) ** 2 for d, o in zip(dz, off, strict=True)]
    near(gx, sum(d @ w for d, w in zip(dz, W, strict=True)), sum((o + 6 * n * U32**2 * d * d) @ (w * w) for o, d, w in zip(mul, dz, W, strict=True)), dtype, "dx")
    for i, (d, o, e) in enumerate(zip(dz, mul, off, strict=True)):
      near(rest[i], d.t() @ X, (o + 3 * m * U32**2 * d * d).t() @ (X * X), dtype, "dw")
      near(rest[len(ws) + i], d.sum(0), (e * e + m * U32**2 * d * d).sum(0), dtype, "db")


def test_no_product_kernel_spills():
  sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "tools"))
  import code_object

  if not (code_object.LLVM / "llvm-objdump").exists():
    pytest.skip("ROCm LLVM tools not installed")
  native.policy_lib()
  kernels = {n: md for n, md in code_object.kernels(native.POLICY_LIB_PATH).items() if "k_product" in n}
  assert len(kernels) >= 78  # 16 bits: 8 products and epilogues x 3 tiles and 4 of dz x 2, of each of two types; float: 7 x 2
  for name, md in kernels.items():
    assert md["private_segment_fixed_size"] == 0, (name, md)
