"""Norm, weight and rotation of query and key heads against a float64 form.

Tolerances: float32 results come from one sum over a head and a handful of
rounded products (1e-6 covers head sizes up to 1000); 16-bit results add one
rounding (2^-8 for bfloat16 and 2^-11 for float16 at most per element); weight gradients sum thousands of
float32 terms (1e-5) before their own rounding.
"""

from __future__ import annotations

import math

import pytest
import torch

import associative_scan_triton as ast

DEV = "cuda"
gpu = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TOL = {F32: 1e-6, F16: 2.0**-11, BF16: 2.0**-8}


def oracle(x, w, cos, sin, pos, eps, interleaved):
  """float64; pos < 0 gives zero rows."""
  half, dim = cos.shape[1], x.shape[2]
  n = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * w
  i = torch.arange(half) * (2 if interleaved else 1)
  j = i + (1 if interleaved else half)
  c, s = cos[pos.clamp(min=0)][:, None], sin[pos.clamp(min=0)][:, None]
  matrix_i = n[..., i] * c - n[..., j] * s
  matrix_j = n[..., j] * c + n[..., i] * s
  y = n.clone()
  y = y.index_copy(2, i, matrix_i).index_copy(2, j, matrix_j)
  assert y.shape[2] == dim
  return torch.where((pos >= 0)[:, None, None], y, torch.zeros_like(y))


def tables(rows, half, seed=4):
  angle = torch.rand(rows, half, generator=torch.Generator().manual_seed(seed)) * 6.3
  return angle.cos(), angle.sin()


def close(name, got, want, tol):
  got, want = got.detach().double().cpu(), want.detach().double().cpu()
  assert got.shape == want.shape and torch.isfinite(got).all(), name
  rms = float(want.square().mean().sqrt()) if want.numel() else 0.0
  assert float((got - want).norm()) <= tol * float(want.norm()) + 1e-30, (
    name, float((got - want).norm() / want.norm()), tol)
  if rms:
    assert float(((got - want).abs() / want.abs().clamp(min=rms)).max()) <= 16 * tol, name


def make(tokens, hq, hk, dim, dtype, seed=0, wtype=None):
  gen = torch.Generator().manual_seed(seed)
  size = torch.rand(hq + hk, 1, generator=gen) * 4 + 0.1
  both = (torch.randn(tokens, hq + hk, dim, generator=gen) * size).to(dtype)
  w = [(1 + 0.3 * torch.randn(dim, generator=gen)).to(wtype or dtype) for _ in range(2)]
  d = [torch.randn(tokens, h, dim, generator=gen).to(dtype) for h in (hq, hk)]
  return both[:, :hq], both[:, hq:], *w, *d


def check(tokens, hq, hk, dim, half, dtype, interleaved=False, positions=None, lengths=None, wtype=None,
          first=0, eps=1e-6):
  q, k, wq, wk, dq, dk = make(tokens, hq, hk, dim, dtype, wtype=wtype)
  rows = 61
  cos, sin = tables(rows, half)
  if lengths is None:
    pos = torch.randint(0, rows, (tokens,), generator=torch.Generator().manual_seed(7)).to(positions)
    where = {"positions": pos.to(DEV)}
  else:
    cu = torch.tensor([first + sum(lengths[:i]) for i in range(len(lengths) + 1)])
    pos = torch.cat([torch.full((first,), -1)] + [torch.arange(m) for m in lengths])
    where = {"args": {"cu_seqlens": cu.to(torch.int32).to(DEV)}}
  both = torch.cat((q, k), 1).to(DEV)
  ours = [both[:, :hq].detach().requires_grad_(True), both[:, hq:].detach().requires_grad_(True),
          wq.to(DEV).requires_grad_(True), wk.to(DEV).requires_grad_(True)]
  yq, yk = ast.qk_norm_rotate(*ours, cos.to(DEV), sin.to(DEV), eps=eps, interleaved=interleaved, **where)
  assert yq.is_contiguous() and yq.dtype == dtype and yk.shape == k.shape
  grads = torch.autograd.grad([yq, yk], ours, [dq.to(DEV), dk.to(DEV)])
  gold = [x.double().requires_grad_(True) for x in (q, k, wq, wk)]
  want = [oracle(gold[i], gold[i + 2], cos.double(), sin.double(), pos.long(), eps, interleaved) for i in (0, 1)]
  want_grads = torch.autograd.grad(want, gold, [dq.double(), dk.double()])
  close("queries", yq, want[0], TOL[dtype])
  close("keys", yk, want[1], TOL[dtype])
  for name, a, b in zip(("d_queries", "d_keys"), grads, want_grads):
    close(name, a, b, TOL[dtype] + 2e-6)
  for name, a, b in zip(("d_query_weight", "d_key_weight"), grads[2:], want_grads[2:]):
    close(name, a, b, 1e-5 + (0 if a.dtype == F32 else TOL[a.dtype]))


@gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,half", [(128, 64), (128, 16), (64, 32), (64, 0), (80, 16), (96, 48), (48, 24), (256, 128),
                                      (8, 4), (6, 3), (1, 0), (33, 7), (130, 65), (600, 300)])
def test_head_sizes(dim, half, interleaved, dtype):
  check(37, 3, 2, dim, half, dtype, interleaved, positions=torch.int64)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tokens", [1, 2, 15, 1000])
@pytest.mark.parametrize("heads", [(1, 1), (12, 12), (16, 4), (5, 1)], ids=str)
def test_tokens_and_heads(heads, tokens, dtype):
  check(tokens, *heads, 64, 32, dtype, positions=torch.int32, wtype=F32)


@gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [64, 33])
def test_sequences(dim, dtype):
  check(130, 3, 2, dim, 16, dtype, lengths=[1, 0, 60, 58], first=11)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_tokens_take_several_heads_a_group(dtype):
  check(30000, 6, 2, 64, 32, dtype, positions=torch.int64)


@gpu
@pytest.mark.parametrize("dim", [64, 33])
def test_zero_rows_eps_and_large_values(dim):
  q, k, wq, wk, _, _ = make(4, 2, 1, dim, F32)
  both = torch.cat((q, k), 1).clone()
  both[0] = 0.0  # nothing to norm: eps alone
  both[1] *= 1e15
  cos, sin = tables(4, 8)
  where = torch.arange(4)
  yq, yk = ast.qk_norm_rotate(both[:, :2].to(DEV), both[:, 2:].to(DEV), wq.to(DEV), wk.to(DEV), cos.to(DEV),
                              sin.to(DEV), positions=where.to(DEV), eps=1e-5)
  assert not yq[0].any() and not yk[0].any()
  for got, x, w in ((yq, both[:, :2], wq), (yk, both[:, 2:], wk)):
    close("y", got, oracle(x.double(), w.double(), cos.double(), sin.double(), where, 1e-5, False), 1e-6)


@gpu
def test_views_strides_and_alignment():
  # the same numbers through aligned and misaligned views of a projection
  gen = torch.Generator().manual_seed(2)
  flat = torch.randn(50 * (5 * 64 + 8) + 1, generator=gen).to(BF16).to(DEV)
  w = torch.ones(64, dtype=BF16, device=DEV)
  cos, sin = (x.to(DEV) for x in tables(61, 32))
  pos = torch.arange(50, device=DEV)
  for shift in (0, 1):
    wide = flat[shift:shift + 50 * (5 * 64 + 8)].view(50, -1)
    q, k = wide[:, :192].view(50, 3, 64), wide[:, 192:320].view(50, 2, 64)
    yq, yk = ast.qk_norm_rotate(q, k, w, w, cos, sin, positions=pos)
    for got, x in ((yq, q), (yk, k)):
      close("y", got, oracle(x.double().cpu(), w.double().cpu(), cos.double().cpu(), sin.double().cpu(), pos.cpu(), 1e-6,
                             False), TOL[BF16])


@gpu
@pytest.mark.parametrize("dim", [64, 33])
def test_positions_outside_the_table_are_reported(dim):
  q, k, wq, wk, _, _ = (x.to(DEV) for x in make(3, 2, 2, dim, F32))
  cos, sin = (x.to(DEV) for x in tables(5, 8))
  for bad in (5, -1, 2**40):
    pos = torch.tensor([1, bad, 2], device=DEV)
    with pytest.raises(ast.ScanError, match="position"):
      ast.qk_norm_rotate(q, k, wq, wk, cos, sin, positions=pos)
      ast.check_device_error()
  with pytest.raises(ast.ScanError, match="cu_seqlens"):
    ast.qk_norm_rotate(q, k, wq, wk, cos, sin, {"cu_seqlens": torch.tensor([0, 2], device=DEV)})
    ast.check_device_error()


@gpu
def test_values_that_are_not_finite_stay_in_their_head():
  for dim in (64, 33):
    q, k, wq, wk, _, _ = make(40, 3, 2, dim, F32)
    cos, sin = tables(40, 8)
    pos = torch.arange(40)
    want = oracle(q.double(), wq.double(), cos.double(), sin.double(), pos, 1e-6, False)
    q = q.clone()
    q[7, 1, 3] = math.nan
    q[9, 2, 0] = math.inf
    got, _ = ast.qk_norm_rotate(q.to(DEV), k.to(DEV), wq.to(DEV), wk.to(DEV), cos.to(DEV), sin.to(DEV),
                                positions=pos.to(DEV))
    keep = torch.ones(40, 3, dtype=torch.bool)
    keep[7, 1] = keep[9, 2] = False
    close("y", got.cpu()[keep], want[keep], TOL[F32])


@gpu
def test_weight_gradients_repeat_bit_for_bit():
  q, k, wq, wk, dq, dk = (x.to(DEV) for x in make(5000, 6, 2, 64, BF16))
  cos, sin = (x.to(DEV) for x in tables(5000, 32))
  pos = torch.arange(5000, device=DEV)
  found = []
  for _ in range(2):
    leaves = [x.detach().clone().requires_grad_(True) for x in (q, k, wq, wk)]
    y = ast.qk_norm_rotate(*leaves, cos, sin, positions=pos)
    found.append(torch.autograd.grad(y, leaves, (dq, dk)))
  for a, b in zip(*found):
    assert torch.equal(a, b)


@gpu
def test_gradient_by_differences():
  # central differences in float64: truncation ~ h^2 = 1e-10, our own 1e-6; 1e-5
  q, k, wq, wk, dq, dk = make(9, 2, 1, 16, F32)
  cos, sin = tables(9, 6)
  pos = torch.arange(9)
  leaves = [x.to(DEV).requires_grad_(True) for x in (q, k, wq, wk)]
  y = ast.qk_norm_rotate(*leaves, cos.to(DEV), sin.to(DEV), positions=pos.to(DEV))
  ours = torch.autograd.grad(y, leaves, (dq.to(DEV), dk.to(DEV)))

  def loss(p):
    a = oracle(p[0], p[2], cos.double(), sin.double(), pos, 1e-6, False)
    b = oracle(p[1], p[3], cos.double(), sin.double(), pos, 1e-6, False)
    return float((a * dq.double()).sum() + (b * dk.double()).sum())

  base = [x.double() for x in (q, k, wq, wk)]
  gen = torch.Generator().manual_seed(3)
  for i in range(4):
    direction = torch.randn(base[i].shape, generator=gen, dtype=torch.float64)
    moved = [[x + s * 1e-5 * direction if j == i else x for j, x in enumerate(base)] for s in (1, -1)]
    slope = (loss(moved[0]) - loss(moved[1])) / 2e-5
    assert abs(slope - float((ours[i].double().cpu() * direction).sum())) <= 1e-5 * float(ours[i].norm()) * 16


@gpu
def test_refusals():
  q = torch.randn(4, 2, 16, device=DEV)
  w = torch.ones(16, device=DEV)
  cos, sin = (x.to(DEV) for x in tables(4, 8))
  pos = torch.arange(4, device=DEV)

  def refused(error, match, q=q, k=q, wq=w, wk=w, cos=cos, sin=sin, **kw):
    with pytest.raises(error, match=match):
      ast.qk_norm_rotate(q, k, wq, wk, cos, sin, **({"positions": pos} | kw))

  refused(ValueError, "CUDA tensors only", q=q.cpu())
  refused(ValueError, "either positions or args", positions=None)
  refused(ValueError, "either positions or args", args={"cu_seqlens": pos})
  refused(ValueError, "entries", positions=pos[:3])
  refused(TypeError, "int32 or int64", positions=pos.float())
  refused(TypeError, "weights must be", wk=w.half())
  refused(ValueError, "query_weight must be", wq=w[:8])
  refused(ValueError, "half <=", cos=torch.ones(4, 9, device=DEV), sin=torch.ones(4, 9, device=DEV))
  refused(ValueError, "both tables alike", sin=sin[:3].contiguous())
  refused(TypeError, "cos must be float32", cos=cos.half())
  refused(ValueError, "rows", k=q[:3])
  refused(ValueError, "unit stride", q=q.transpose(1, 2).contiguous().transpose(1, 2))


def test_cpu_tensors_are_refused():
  q = torch.zeros(4, 1, 8)
  with pytest.raises(ValueError, match="CUDA tensors only"):
    ast.qk_norm_rotate(q, q, torch.ones(8), torch.ones(8), torch.ones(4, 4), torch.ones(4, 4),
                       positions=torch.arange(4))


@gpu
def test_empty():
  q = torch.empty(0, 2, 16, device=DEV, requires_grad=True)
  w = torch.ones(16, device=DEV, requires_grad=True)
  cos, sin = (x.to(DEV) for x in tables(4, 8))
  yq, yk = ast.qk_norm_rotate(q, q, w, w, cos, sin, positions=torch.empty(0, dtype=torch.int64, device=DEV))
  (yq.sum() + yk.sum()).backward()
  assert not w.grad.any()


@gpu
@pytest.mark.parametrize("changed", ["cos", "sin", "positions", "cu_seqlens"])
def test_backward_refuses_tables_and_positions_changed_since(changed):
  q, k, wq, wk, dq, dk = (x.to(DEV) for x in make(9, 2, 1, 16, F32))
  cos, sin = (x.to(DEV) for x in tables(20, 8))
  at = {"positions": torch.arange(9, device=DEV), "cu_seqlens": torch.tensor([0, 4, 9], device=DEV)}
  where = {"args": {"cu_seqlens": at["cu_seqlens"]}} if changed == "cu_seqlens" else {"positions": at["positions"]}
  y = ast.qk_norm_rotate(q.requires_grad_(True), k, wq, wk, cos, sin, **where)
  {"cos": cos, "sin": sin, **at}[changed].add_(0 if changed == "cu_seqlens" else 1)
  with pytest.raises(RuntimeError, match="inplace operation"):
    torch.autograd.backward(y, (dq, dk))


@gpu
def test_forward_mode_derivatives_are_refused():
  import torch.autograd.forward_ad as forward_ad
  q, k, wq, wk, _, _ = (x.to(DEV) for x in make(9, 2, 1, 16, F32))
  cos, sin = (x.to(DEV) for x in tables(9, 8))
  pos = torch.arange(9, device=DEV)
  want = ast.qk_norm_rotate(q, k, wq, wk, cos, sin, positions=pos)
  with forward_ad.dual_level():
    for i in range(6):
      x = [q, k, wq, wk, cos, sin]
      x[i] = forward_ad.make_dual(x[i], torch.ones_like(x[i]))
      with pytest.raises(NotImplementedError):
        ast.qk_norm_rotate(*x, positions=pos)
      with pytest.raises(NotImplementedError):
        ast.qk_norm_rotate_compiled(*x, positions=pos)
    for a, b in zip(ast.qk_norm_rotate(q, k, wq, wk, cos, sin, positions=pos), want):
      assert torch.equal(a, b)


@gpu
def test_tables_that_want_a_gradient_are_refused():
  q, k, wq, wk, _, _ = (x.to(DEV) for x in make(9, 2, 1, 16, F32))
  cos, sin = (x.to(DEV) for x in tables(9, 8))
  pos = torch.arange(9, device=DEV)
  for name in ("cos", "sin"):
    leaf = {"cos": cos, "sin": sin}[name].clone().requires_grad_(True)
    for queries in (q, q.clone().requires_grad_(True)):
      with pytest.raises(ValueError, match="no gradient"):
        ast.qk_norm_rotate(queries, k, wq, wk, **{"cos": cos, "sin": sin, name: leaf}, positions=pos)
      with pytest.raises(ValueError, match="no gradient"):
        ast.qk_norm_rotate_compiled(queries, k, wq, wk, **{"cos": cos, "sin": sin, name: leaf}, positions=pos)
    with torch.no_grad():
      ast.qk_norm_rotate(q, k, wq, wk, **{"cos": cos, "sin": sin, name: leaf}, positions=pos)
