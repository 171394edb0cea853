"""qk_norm_rotate with a position on each of several axes, against float64.

Tolerances as for one axis: float32 sums of a head's squares, 1e-6; 16-bit
results one rounding, at most 2^-8 (bfloat16) or 2^-11 (float16) of each value;
gradients of weights are sums over all tokens in float32, 1e-5 of their norm.
"""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import associative_scan_triton as ast
from associative_scan_triton import _lib

DEV = "cuda"
gpu = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TOL = {F32: 1e-6, F16: 2.0**-11, BF16: 2.0**-8}
ROWS = 50


def oracle(x, w, cos, sin, positions, sections, interleaved, eps=1e-6):
  half = sum(sections)
  axis = [a for a, n in enumerate(sections) for _ in range(n)]
  rows = positions[axis].t()  # [tokens, half]
  c, s = cos[rows, torch.arange(half)][:, None], sin[rows, torch.arange(half)][:, None]
  n = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w
  if interleaved:
    a, b = n[..., 0:2 * half:2], n[..., 1:2 * half:2]
    turned = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
  else:
    a, b = n[..., :half], n[..., half:2 * half]
    turned = torch.cat((a * c - b * s, b * c + a * s), -1)
  return torch.cat((turned, n[..., 2 * half:]), -1)


def make(tokens, heads, dim, sections, dtype, seed=0):
  gen = torch.Generator().manual_seed(seed)
  q, k, dq, dk = (torch.randn(tokens, h, dim, generator=gen).to(dtype) for h in (*heads, *heads))
  wq, wk = ((1 + 0.2 * torch.randn(dim, generator=gen)).to(dtype) for _ in range(2))
  angle = torch.rand(ROWS, sum(sections), generator=gen) * 6.3
  positions = torch.randint(0, ROWS, (len(sections), tokens), generator=gen)
  return q, k, wq, wk, angle.cos(), angle.sin(), positions, dq, dk


def near(name, got, want, tol):
  got, want = got.detach().double().cpu(), want.detach().double()
  err, rms = (got - want).abs(), float(want.square().mean().sqrt())
  assert float(err.norm()) <= tol * float(want.norm()) + 1e-30, name
  assert float((err / want.abs().clamp(min=rms)).max()) <= 4 * tol, name


def check(tokens, heads, dim, sections, dtype, interleaved, index=torch.int64, views=False):
  q, k, wq, wk, cos, sin, positions, dq, dk = make(tokens, heads, dim, sections, dtype)
  x = [t.to(DEV) for t in (q, k, wq, wk)]
  if views:
    both = torch.cat(x[:2], 1)
    x[0], x[1] = both[:, :heads[0]], both[:, heads[0]:]
  x = [t.detach().requires_grad_(True) for t in x]
  out = ast.qk_norm_rotate(*x, cos.to(DEV), sin.to(DEV), positions=positions.to(index).to(DEV),
                           interleaved=interleaved, sections=sections)
  ref = [t.double().requires_grad_(True) for t in (q, k, wq, wk)]
  want = [oracle(a, w, cos.double(), sin.double(), positions, sections, interleaved)
          for a, w in ((ref[0], ref[2]), (ref[1], ref[3]))]
  for name, a, b in zip(("queries", "keys"), out, want):
    near(name, a, b, TOL[dtype])
  found = torch.autograd.grad(out, x, (dq.to(DEV), dk.to(DEV)))
  exact = torch.autograd.grad(want, ref, (dq.double(), dk.double()))
  for name, a, b in zip(("d_queries", "d_keys", "d_query_weight", "d_key_weight"), found, exact):
    near(name, a, b, max(TOL[dtype], 1e-5 if "weight" in name else 0.0) * (2 if dtype == F32 else 1))


@gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,sections", [(128, (16, 24, 24)), (64, (8, 12, 12)), (80, (8, 16, 16)), (96, (24, 24)),
                                          (128, (8, 8, 8, 8)), (72, (11, 13, 12)), (48, (0, 24)), (10, (1, 1, 3)),
                                          (300, (20, 30)), (64, (32,)), (128, (32, 0, 0, 32))], ids=str)
def test_sections(dim, sections, interleaved, dtype):
  check(37, (4, 2), dim, sections, dtype, interleaved)


@gpu
@pytest.mark.parametrize("tokens", [1, 2, 700])
def test_tokens_and_strides(tokens):
  check(tokens, (16, 4), 128, (16, 24, 24), BF16, False, index=torch.int32, views=True)


@gpu
@pytest.mark.parametrize("dim", [64, 10])
def test_equal_positions_are_one_axis(dim):
  q, k, wq, wk, cos, sin, positions, _, _ = (t.to(DEV) for t in make(33, (3, 1), dim, (1, dim // 2 - 1), F32))
  same = positions[:1].expand(2, -1).contiguous()
  many = ast.qk_norm_rotate(q, k, wq, wk, cos, sin, positions=same, sections=(1, dim // 2 - 1))
  one = ast.qk_norm_rotate(q, k, wq, wk, cos, sin, positions=same[0].contiguous())
  for a, b in zip(many, one):
    near("one axis", a, b.cpu(), TOL[F32])


@gpu
@pytest.mark.parametrize("dim", [64, 10])
@pytest.mark.parametrize("axis", [0, 2])
@pytest.mark.parametrize("place", [-1, ROWS, 2**31 - 1])
def test_a_position_outside_the_table_is_reported(place, axis, dim, monkeypatch):
  sections = (1, 1, dim // 2 - 2)
  q, k, wq, wk, cos, sin, positions, _, _ = (t.to(DEV) for t in make(9, (3, 1), dim, sections, F32))
  positions[axis, 4] = place
  monkeypatch.setattr(_lib, "_finish", lambda *args: None)  # the call would raise by itself
  out = ast.qk_norm_rotate(q, k, wq, wk, cos, sin, positions=positions, sections=sections)
  with pytest.raises(ast.ScanError, match="position"):
    ast.check_device_error()
  for y in out:
    assert (y[4] == 0).all() and (y[[0, 1, 2, 3, 5, 6, 7, 8]] != 0).any(-1).all()


@gpu
def test_compiled_matches_eager():
  q, k, wq, wk, cos, sin, positions, dq, dk = (t.to(DEV) for t in make(33, (3, 1), 64, (8, 12, 12), BF16))
  results = []
  for fn in (ast.qk_norm_rotate, torch.compile(ast.qk_norm_rotate_compiled, fullgraph=True)):
    x = [t.detach().requires_grad_(True) for t in (q, k, wq, wk)]
    out = fn(*x, cos, sin, positions=positions, sections=(8, 12, 12))
    results.append((*out, *torch.autograd.grad(out, x, (dq, dk))))
  for a, b in zip(*results):
    assert torch.equal(a, b)


def test_refusals():
  with FakeTensorMode():
    q, w, cos = (torch.empty(*s, device=DEV) for s in ((9, 2, 64), (64,), (50, 32)))
    positions = torch.empty(3, 9, dtype=torch.int64, device=DEV)

    def refused(match, sections=(8, 12, 12), **kw):
      kw = {"positions": positions, **kw}
      with pytest.raises(ValueError, match=match):
        ast.qk_norm_rotate(q, q, w, w, cos, cos, sections=sections, **kw)

    refused("add up", sections=(8, 12, 13))
    refused("add up", sections=(-8, 20, 20))
    refused("between 1 and 4", sections=(8, 8, 8, 4, 4))
    refused("between 1 and 4", sections=())
    refused("a row for each", positions=positions[:2])
    refused("a row for each", positions=positions[0])
    refused("a row for each", positions=positions[:, :8])
    refused("a row for each", positions=torch.empty(9, 3, dtype=torch.int64, device=DEV).t())
    refused("need positions", positions=None, args={"cu_seqlens": positions[0]})
    refused("CUDA tensors only", positions=torch.empty(3, 9, dtype=torch.int64))
