"""Causal softmax attention over packed sequences against a float64 oracle.

Tolerances (relative 2-norm per output, then the largest error over the larger
of the value and the output's root mean square) follow from the arithmetic:

* float32: sums of at most a few hundred float32 products and exponentials,
  each off by a few 2^-24: 1e-5, ten times the root of the count.
* 16-bit results: one rounding of the result, at most half a step (2^-8 for
  bfloat16, 2^-11 for float16) and as a root mean square less than 0.6 of it,
  and one of an operand inside each product (probabilities, or their
  derivatives), which averages to as much again: together below 2^-8 and
  2^-11; single elements may cancel, so 16 times that for those.
"""

from __future__ import annotations

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import associative_scan_triton as ast
from associative_scan_triton import _lib

DEV = "cuda"
gpu = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
TOL = {F32: 1e-5, F16: 2.0**-11, BF16: 2.0**-8}


def oracle(q, k, v, lengths, scale, first=0):
  """Sequence by sequence in float64; leaves may require gradients."""
  share = q.shape[1] // k.shape[1]
  outs, at = [q.new_zeros(first, q.shape[1], v.shape[2])], first
  for n in lengths:
    qs, ks, vs = (x[at:at + n].transpose(0, 1) for x in (q, k, v))
    ks, vs = ks.repeat_interleave(share, 0), vs.repeat_interleave(share, 0)
    score = (qs @ ks.transpose(1, 2)) * scale
    later = torch.ones(n, n, dtype=torch.bool).triu(1)
    p = torch.softmax(score.masked_fill(later, float("-inf")), -1)
    outs.append((p @ vs).transpose(0, 1))
    at += n
  outs.append(q.new_zeros(q.shape[0] - at, q.shape[1], v.shape[2]))
  return torch.cat(outs)


def close(name, got, want, tol):
  got, want = got.detach().double().cpu(), want.detach().double().cpu()
  assert got.shape == want.shape, (name, got.shape, want.shape)
  assert torch.isfinite(got).all(), f"{name} has values that are not finite"
  rms = float(want.square().mean().sqrt()) if want.numel() else 0.0
  err = (got - want).abs()
  norm = float(want.norm())
  assert float(err.norm()) <= tol * norm + 1e-30, (name, float(err.norm()) / max(norm, 1e-30), tol)
  if want.numel():
    worst = float((err / torch.clamp(want.abs(), min=rms)).max()) if rms else float(err.max())
    assert worst <= 16 * tol, (name, worst, 16 * tol)


def make(lengths, heads, dims, dtype, seed=0, first=0):
  gen = torch.Generator().manual_seed(seed)
  n, (h, hk), (dk, dv) = first + sum(lengths), heads, dims

  def normal(*shape):
    return torch.randn(shape, generator=gen).to(dtype)

  return normal(n, h, dk), normal(n, hk, dk), normal(n, hk, dv), normal(n, h, dv)


def cu_of(lengths, first=0, dtype=torch.int32):
  ends = [first]
  for m in lengths:
    ends.append(ends[-1] + m)
  return torch.tensor(ends, dtype=dtype, device=DEV)


def check(lengths, heads, dims, dtype, grad=True, scale=None, seed=0, cu_dtype=torch.int32):
  q, k, v, do = make(lengths, heads, dims, dtype, seed)
  args = {"cu_seqlens": cu_of(lengths, dtype=cu_dtype)}
  ours = [x.to(DEV).requires_grad_(grad) for x in (q, k, v)]
  out = ast.attention_causal(*ours, args, scale=scale)
  assert out.dtype == dtype and out.is_contiguous()
  ref = [x.double().requires_grad_(grad) for x in (q, k, v)]
  want = oracle(*ref, lengths, dims[0]**-0.5 if scale is None else scale)
  close("out", out, want, TOL[dtype])
  if grad:
    found = torch.autograd.grad(out, ours, do.to(DEV))
    exact = torch.autograd.grad(want, ref, do.double())
    for name, a, b in zip(("queries", "keys", "values"), found, exact):
      assert a.dtype == dtype
      if float(b.norm()) > 1e-9:
        close(name, a, b, TOL[dtype])
      else:  # sequences of one token have no gradient to queries and keys at all
        assert (a == 0).all(), name


LENGTHS = [[1], [2], [0, 1, 0, 2, 0], [31, 32, 33], [127, 128, 129], [64, 0, 257, 5], [300, 1, 511]]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_lengths(lengths, dtype):
  check(lengths, (2, 2), (64, 64), dtype)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dims", [(128, 128), (64, 128), (128, 64), (16, 8), (1, 1), (40, 72), (96, 33),
                                  (127, 80), (3, 128), (128, 1), (80, 80), (8, 120)], ids=str)
def test_head_sizes(dims, dtype):
  check([150, 3, 140], (3, 3), dims, dtype)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads", [(1, 1), (4, 1), (6, 3), (5, 5), (24, 1), (16, 4)], ids=str)
def test_shared_heads(heads, dtype):
  check([130, 70, 260], heads, (64, 64), dtype, cu_dtype=torch.int64)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths", [[1300], [512, 640], [100, 900, 3]], ids=str)
def test_many_tiles(lengths, dtype):
  check(lengths, (4, 2), (128, 128), dtype)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dims", [(128, 128), (40, 33)], ids=str)
def test_first_tokens_have_no_gradient_to_queries(dims, dtype):
  # they see one key, whatever the scores are
  lengths = [1, 1, 200, 1, 3]
  q, k, v, do = (x.to(DEV) for x in make(lengths, (4, 2), dims, dtype))
  x = [t.requires_grad_(True) for t in (q, k, v)]
  d_q, d_k, _ = torch.autograd.grad(ast.attention_causal(*x, {"cu_seqlens": cu_of(lengths)}), x, do)
  assert (d_q[[0, 1, 2, 202, 203]] == 0).all() and (d_k[[0, 1, 202]] == 0).all()
  assert (d_q[3:202].abs().amax((1, 2)) > 0).all()


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_query_gradients_of_keys_with_a_common_part(dtype):
  # what all keys share does not reach the queries' gradients, nor does it weigh
  # the roundings of ds: with and without it the error is that of two roundings
  n = 400
  q, k, v, do = make([n], (4, 2), (128, 128), dtype)
  common = 3.0 * torch.randn(2, 128, generator=torch.Generator().manual_seed(7))
  q = (0.3 * q.float()).to(dtype)
  k = (k.float() + common).to(dtype)
  ours = [x.to(DEV).requires_grad_(True) for x in (q, k, v)]
  found, = torch.autograd.grad(ast.attention_causal(*ours, {"cu_seqlens": cu_of([n])}), ours[:1], do.to(DEV))
  ref = q.double().requires_grad_(True)
  want, = torch.autograd.grad(oracle(ref, k.double(), v.double(), [n], 128**-0.5), ref, do.double())
  # two roundings of 3**-0.5 half steps at most, as a root mean square: 0.82 half
  # steps of the norm (rows of few keys are ten times as large as the others, so
  # no single element is held against all elements' root mean square here)
  assert float((found.double().cpu() - want).norm()) <= TOL[dtype] * float(want.norm())


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_many_short_sequences(dtype):
  check([1 + i % 7 for i in range(400)], (2, 1), (64, 64), dtype)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_thousands_of_sequences(dtype):
  # more than a CTA keeps the ends of, and than a warp looks through in one step
  check([i % 3 for i in range(2600)], (1, 1), (32, 32), dtype)


@gpu
@pytest.mark.parametrize("size", [2.0**-12, 2.0**-3, 2.0**8])
def test_float16_gradients_of_any_size(size):
  # ds of 700 keys lies a thousandth below do, where float16 has no steps left
  # for the small ones, while the results are inside its range
  n = 700
  q, k, v, do = make([n], (2, 2), (64, 64), F16)
  q, k, v = q * 2.0**-4, k * 2.0**4, v * 2.0**4
  do = (do.float() * size).half()
  ours = [x.to(DEV).requires_grad_(True) for x in (q, k, v)]
  found = torch.autograd.grad(ast.attention_causal(*ours, {"cu_seqlens": cu_of([n])}), ours[:1], do.to(DEV))
  ref = [x.double().requires_grad_(True) for x in (q, k, v)]
  exact = torch.autograd.grad(oracle(*ref, [n], 0.125), ref[:1], do.double())
  # as everywhere, and half of float16's last step for results that reach it;
  # results beyond its largest number are infinite
  got, want = found[0].double().cpu(), exact[0]
  fits = want.abs() < 65504 * (1 - 2.0**-8)
  assert torch.isinf(got[want.abs() > 65536 * (1 + 2.0**-8)]).all()
  err = float((got - want)[fits].norm())
  assert err <= TOL[F16] * float(want.norm()) + 2.0**-25 * want.numel()**0.5


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_far_below_the_largest(dtype):
  # a sequence whose upstream gradients are 2^-8 of another's, and rows of no
  # sequence with huge ones: ds of its 700 keys is about 2^-17 of the largest
  lengths, first = [100, 700], 5
  q, k, v, do = make(lengths, (2, 2), (64, 64), dtype, first=first)
  q = q * 2.0**-3
  do[105:] *= 2.0**-8
  do[:5] = 2.0**15
  ours = [x.to(DEV).requires_grad_(True) for x in (q, k, v)]
  found = torch.autograd.grad(ast.attention_causal(*ours, {"cu_seqlens": cu_of(lengths, first)}), ours, do.to(DEV))
  ref = [x.double().requires_grad_(True) for x in (q, k, v)]
  exact = torch.autograd.grad(oracle(*ref, lengths, 0.125, first), ref, do.double())
  for name, a, b in zip(("queries", "keys", "values"), found, exact):
    assert not a[:5].any(), name
    # float16: results of 2^-13 and more, whose steps stop shrinking at 2^-14
    last = 2.0**-25 * b[105:].numel()**0.5 if dtype == F16 else 0.0
    err = float((a[105:].double().cpu() - b[105:]).norm())
    assert err <= TOL[dtype] * float(b[105:].norm()) + last, name


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_value_gradients_of_keys_with_small_weights(dtype):
  # the first 100 keys have weights of about e^-12 / 200 = 2^-25 for all queries
  # that an upstream gradient reaches
  q, k, v, do = make([300], (2, 2), (64, 64), dtype)
  q[..., 0], k[..., 0] = 8.0, 0.0
  k[:100, :, 0] = -12.0
  do = do * 2.0**12
  do[:100] = 0.0
  ours = [x.to(DEV).requires_grad_(True) for x in (q, k, v)]
  found, = torch.autograd.grad(ast.attention_causal(*ours, {"cu_seqlens": cu_of([300])}), ours[2:], do.to(DEV))
  ref = [x.double().requires_grad_(True) for x in (q, k, v)]
  exact, = torch.autograd.grad(oracle(*ref, [300], 0.125), ref[2:], do.double())
  close("values", found[:100], exact[:100], TOL[dtype])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [0.5, 1.0, 2.0**-8])
def test_scales(scale, dtype):
  # at 0.5 and more rows are sharp: probabilities near 1, ds a small difference
  check([260, 77], (2, 2), (64, 64), dtype, scale=scale)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_scores_that_grow_along_the_row(dtype):
  # every key outweighs all before it: the softmax's reference moves in each tile
  n = 700
  q, k, v, _ = make([n], (2, 2), (64, 64), dtype)
  k[..., 0] = torch.linspace(-30, 30, n)[:, None].to(dtype)
  q[..., 0] = 8.0
  out = ast.attention_causal(q.to(DEV), k.to(DEV), v.to(DEV), {"cu_seqlens": cu_of([n])})
  close("out", out, oracle(q.double(), k.double(), v.double(), [n], 0.125), TOL[dtype])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_sharp_rows_keep_their_gradients(dtype):
  # probabilities within 1e-3 of 1: do.v - do.o cancels all but the last digits,
  # and a do.o from the rounded out alone would leave nothing of them.
  # An element is off by what its roundings leave, weighed by what they meet.
  # The forward's weights are rounded by half a step h each and add up to 1 as
  # rounded: do.o is off by h times the spread of do.v over the row.  p and ds are
  # rounded by h, as the result is; do.v - do.o loses 1e-5 of its float32 terms
  # and h^2 of out (kept with the rest of its rounding); float16's steps end at
  # 2^-24.
  n, h = 256, {F32: 2.0**-24, F16: 2.0**-11, BF16: 2.0**-8}[dtype]
  q, k, v, do = make([n], (2, 2), (64, 64), dtype, seed=5)
  mark = torch.zeros(n, 64)
  mark[torch.arange(n), torch.arange(n) % 64] = 9.0
  k = (0.1 * k.float() + mark[:, None]).to(dtype)
  q = (0.1 * q.float() + mark[:, None]).to(dtype)
  ours = [x.to(DEV).requires_grad_(True) for x in (q, k, v)]
  found = torch.autograd.grad(ast.attention_causal(*ours, {"cu_seqlens": cu_of([n])}), ours, do.to(DEV))
  Q, K, V, G = (x.double().transpose(0, 1) for x in (q, k, v, do))
  score = (0.125 * Q @ K.transpose(1, 2)).masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), float("-inf"))
  p = torch.softmax(score, -1)
  o = p @ V
  spread = G @ V.transpose(1, 2) - (G * o).sum(-1, keepdim=True)
  ds = p * spread
  lost = G.abs() @ V.abs().transpose(1, 2) + (G * o).abs().sum(-1, keepdim=True)
  fine = 2.0**-25 if dtype == F16 else 0.0
  e_ds = h * ds.abs() + 2 * h * p * ds.abs().sum(-1, keepdim=True) + (1e-5 + h * h) * p * lost + fine * (p > 0)
  e_p = (h + 1e-5) * p + fine * (p > 0)
  want = (0.125 * ds @ K, 0.125 * ds.transpose(1, 2) @ Q, p.transpose(1, 2) @ G)
  # dq is summed over the keys less their mean (of the first 128; a row's ds add
  # up to nothing), so that is what its ds meet
  c = K[:, :128].mean(1, keepdim=True) if dtype != F32 else 0 * K[:, :1]
  room = (0.125 * e_ds @ (K - c).abs(), 0.125 * e_ds.transpose(1, 2) @ Q.abs(), e_p.transpose(1, 2) @ G.abs())
  for name, a, b, e in zip(("queries", "keys", "values"), found, want, room):
    err = (a.double().cpu() - b.transpose(0, 1)).abs()
    assert (err <= (e + (h + 1e-6) * b.abs() + fine).transpose(0, 1)).all(), name


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_tokens_of_no_sequence(dtype):
  # rows before cu_seqlens[0] hold NaN: they are not read, and come out zero
  lengths, first = [60, 90], 37
  q, k, v, do = make(lengths, (4, 2), (64, 64), dtype, first=first)
  for x in (q, k, v, do):
    x[:first] = float("nan")
  ours = [x.to(DEV).requires_grad_(True) for x in (q, k, v)]
  out = ast.attention_causal(*ours, {"cu_seqlens": cu_of(lengths, first)})
  found = torch.autograd.grad(out, ours, do.to(DEV))
  ref = [x[first:].double().requires_grad_(True) for x in (q, k, v)]
  want = oracle(*ref, lengths, 0.125)
  exact = torch.autograd.grad(want, ref, do[first:].double())
  for name, a, b in zip(("out", "queries", "keys", "values"), (out, *found), (want, *exact)):
    assert (a[:first] == 0).all(), name
    close(name, a[first:], b, TOL[dtype])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_sequences_do_not_meet(dtype):
  # the second sequence is NaN throughout: nothing of it reaches its neighbours
  lengths = [70, 50, 200]
  q, k, v, do = make(lengths, (4, 2), (64, 64), dtype)
  for x in (q, k, v, do):
    x[70:120] = float("nan")
  ours = [x.to(DEV).requires_grad_(True) for x in (q, k, v)]
  out = ast.attention_causal(*ours, {"cu_seqlens": cu_of(lengths)})
  found = torch.autograd.grad(out, ours, do.to(DEV))
  ref = [x.double().requires_grad_(True) for x in (q, k, v)]
  want = oracle(*ref, lengths, 0.125)
  exact = torch.autograd.grad(want, ref, do.double())
  keep = torch.cat((torch.arange(70), torch.arange(120, 320)))
  for name, a, b in zip(("out", "queries", "keys", "values"), (out, *found), (want, *exact)):
    close(name, a.cpu()[keep], b[keep], TOL[dtype])
    assert not torch.isfinite(a[70:120]).any(), name


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")], ids=str)
@pytest.mark.parametrize("where", ["values", "keys"])
@pytest.mark.parametrize("at", [0, 5, 130, 139, 299])
def test_what_is_not_finite_stays_behind_the_mask(at, where, bad, dtype):
  n = 300
  q, k, v, do = make([n], (2, 1), (64, 64), dtype)
  (v if where == "values" else k)[at, 0, 3] = bad
  ours = [x.to(DEV).requires_grad_(True) for x in (q, k, v)]
  out = ast.attention_causal(*ours, {"cu_seqlens": cu_of([n])})
  do[at:] = 0  # no gradient comes from the rows that saw it
  d_q, = torch.autograd.grad(out, ours[:1], do.to(DEV))
  if at:
    ref = q.double().requires_grad_(True)
    want = oracle(ref, k.double(), v.double(), [n], 0.125)
    clean = oracle(ref[:at], k[:at].double(), v[:at].double(), [at], 0.125)
    close("out", out[:at], clean, TOL[dtype])
    exact, = torch.autograd.grad(clean, ref, do[:at].double())
    close("queries", d_q[:at], exact[:at], TOL[dtype])
  else:
    want = oracle(q.double(), k.double(), v.double(), [n], 0.125)
  if where == "values":
    got, ref = out[at:].cpu().double(), want[at:].detach()
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    assert torch.equal(torch.isinf(got), torch.isinf(ref)) and (got[torch.isinf(got)] == ref[torch.isinf(ref)]).all()
  elif bad != bad:
    assert torch.isnan(out[at:]).all()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(dtype):
  lengths, n = [140, 33], 173
  q, k, v, do = make(lengths, (4, 2), (64, 64), dtype)
  packed = torch.cat((q, k, v), 1).to(DEV)  # views of a packed projection
  odd = torch.zeros(n, 8, 67, dtype=dtype, device=DEV)  # rows off 16 bytes
  odd[..., 1:65] = packed
  turned = packed.transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost
  args = {"cu_seqlens": cu_of(lengths)}
  want = oracle(q.double(), k.double(), v.double(), lengths, 0.125)
  for x in (packed, odd[..., 1:65], turned):
    x = x.detach().requires_grad_(True)
    out = ast.attention_causal(x[:, :4], x[:, 4:6], x[:, 6:], args)
    close("out", out, want, TOL[dtype])
    wide = torch.zeros(n, 4, 70, dtype=dtype, device=DEV)
    wide[..., 3:67] = do.to(DEV)
    found, = torch.autograd.grad(out, x, wide[..., 3:67])
    ref = [y.double().requires_grad_(True) for y in (q, k, v)]
    exact = torch.autograd.grad(oracle(*ref, lengths, 0.125), ref, do.double())
    for a, b in zip((found[:, :4], found[:, 4:6], found[:, 6:]), exact):
      close("gradient", a, b, TOL[dtype])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_broadcast_inputs_and_gradients(dtype):
  # one key head expanded over heads and an upstream gradient of stride 0
  lengths = [90, 41]
  q, k, v, _ = make(lengths, (4, 1), (64, 64), dtype)
  ours = [x.to(DEV).requires_grad_(True) for x in (q, k, v)]
  out = ast.attention_causal(ours[0], ours[1].expand(-1, 4, -1), ours[2].expand(-1, 4, -1),
                             {"cu_seqlens": cu_of(lengths)})
  found = torch.autograd.grad(out.sum(), ours)
  ref = [x.double().requires_grad_(True) for x in (q, k, v)]
  exact = torch.autograd.grad(oracle(*ref, lengths, 0.125).sum(), ref)
  for name, a, b in zip(("queries", "keys", "values"), found, exact):
    # four gradients, each rounded to the type, are added and rounded again
    close(name, a, b, (2 if name != "queries" else 1) * TOL[dtype])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_by_differences(dtype):
  lengths = [70, 131]
  q, k, v, do = make(lengths, (2, 1), (32, 32), dtype, seed=3)
  ours = [x.to(DEV).requires_grad_(True) for x in (q, k, v)]
  found = torch.autograd.grad(ast.attention_causal(*ours, {"cu_seqlens": cu_of(lengths)}), ours, do.to(DEV))
  gen = torch.Generator().manual_seed(9)
  for i, g in enumerate(found):
    x = [t.double() for t in (q, k, v)]
    u = torch.randn(x[i].shape, generator=gen, dtype=torch.float64)
    u = u + g.double().cpu() / g.double().cpu().norm() * u.norm()  # not a direction that averages away
    h = 1e-4

    def loss(e):
      y = list(x)
      y[i] = y[i] + e * u
      return float((oracle(*y, lengths, 32**-0.5) * do.double()).sum())

    slope = (loss(h) - loss(-h)) / (2 * h)
    assert abs(float((g.double().cpu() * u).sum()) - slope) <= 2 * TOL[dtype] * abs(slope) + 1e-6


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_repeats_bit_for_bit_on_another_stream_and_in_a_graph(dtype):
  lengths = [200, 57]
  q, k, v, do = (x.to(DEV) for x in make(lengths, (4, 2), (64, 64), dtype))
  args = {"cu_seqlens": cu_of(lengths)}

  def step(q, k, v):
    x = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = ast.attention_causal(*x, args)
    return (out.detach(), *torch.autograd.grad(out, x, do))

  first = [t.clone() for t in step(q, k, v)]
  s = torch.cuda.Stream()
  s.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(s):
    other = step(q, k, v)
  s.synchronize()
  for a, b in zip(first, other):
    assert torch.equal(a, b)
  graph = torch.cuda.CUDAGraph()
  held = [t.clone() for t in (q, k, v)]
  sync = _lib.sync_check_enabled()
  ast.set_sync_check(False)
  try:
    with torch.cuda.graph(graph):
      captured = step(*held)
  finally:
    ast.set_sync_check(sync)
  for t in held:
    t.mul_(0.5)
  graph.replay()
  torch.cuda.synchronize()
  for a, b in zip(captured, step(q * 0.5, k * 0.5, v * 0.5)):
    assert torch.equal(a, b)


@gpu
def test_empty_inputs():
  for tokens, cu in ((0, [0]), (0, [0, 0]), (3, None)):
    q = torch.randn(tokens, 2, 16, device=DEV, requires_grad=True)
    k, v = (torch.randn(tokens, 1, d, device=DEV, requires_grad=True) for d in (16, 8))
    if cu is None:  # tokens, but no sequence
      cu = [0]
    out = ast.attention_causal(q, k, v, {"cu_seqlens": torch.tensor(cu, dtype=torch.int32, device=DEV)})
    assert out.shape == (tokens, 2, 8) and (out == 0).all()
    for g in torch.autograd.grad(out.sum(), (q, k, v)):
      assert (g == 0).all()


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cu", [[0, 5, 3, 10], [0, 4, 9], [0, 4, 200], [-3, 10]], ids=str)
def test_malformed_sequences_are_reported(cu, dtype):
  q, k, v, _ = (x.to(DEV) for x in make([10], (2, 2), (64, 64), dtype))
  with pytest.raises(ast.ScanError, match="cu_seqlens"):
    ast.attention_causal(q, k, v, {"cu_seqlens": torch.tensor(cu, dtype=torch.int32, device=DEV)})


def test_refusals():
  with FakeTensorMode():
    q = torch.empty(10, 4, 32, device=DEV)
    k = torch.empty(10, 2, 32, device=DEV)
    args = {"cu_seqlens": torch.empty(2, dtype=torch.int32, device=DEV)}

    def refused(error, match, q=q, k=k, v=k, args=args, **kw):
      with pytest.raises(error, match=match):
        ast.attention_causal(q, k, v, args, **kw)

    refused(ValueError, "CUDA tensors only", q=torch.empty(10, 4, 32))
    refused(TypeError, "keys has dtype", k=k.half())
    refused(TypeError, "values has dtype", v=k.half())
    refused(TypeError, "unsupported dtype", q=q.double())
    refused(ValueError, "3 dimensions", v=k[0])
    refused(ValueError, "rows", v=k[:9])
    refused(ValueError, "head size", k=k[..., :16])
    refused(ValueError, "empty head", v=k[..., :0])
    refused(ValueError, "unit stride", v=k.transpose(1, 2).contiguous().transpose(1, 2))
    refused(ValueError, "same number of heads", v=k[:, :1])
    refused(ValueError, "divisor", q=q[:, :3])
    refused(ValueError, "heads", k=k[:, :0], v=k[:, :0])
    refused(ValueError, "head sizes up to 128", v=torch.empty(10, 2, 129, device=DEV))
    refused(TypeError, "int32 or int64", args={"cu_seqlens": args["cu_seqlens"].float()})
    refused(ValueError, "one dimension", args={"cu_seqlens": args["cu_seqlens"][None]})
    refused(ValueError, "at least one entry", args={"cu_seqlens": args["cu_seqlens"][:0]})
    for scale in (0.0, -1.0, float("nan"), float("inf")):
      refused(ValueError, "scale must be", scale=scale)


def test_abi_rejects_bad_arguments_without_a_gpu():
  lib = _lib.load()
  data = torch.zeros(64)

  def call(heads=(2, 2, 2), strides=(4, 4, 4), dims=(4, 4), dtype=0, scale=1.0, tokens=4, seqs=1, index=0):
    rows = [ctypes.byref(_lib.Rows(data.data_ptr(), 8, s, h)) for h, s in zip(heads, strides)]
    return lib.ascan_attention_forward(*rows, data.data_ptr(), index, seqs, tokens, *dims, dtype, scale,
                                       data.data_ptr(), None, None, None)

  for bad in ({"heads": (3, 2, 2)}, {"heads": (2, 2, 1)}, {"heads": (2, 0, 0)}, {"strides": (-4, 4, 4)},
              {"dims": (0, 4)}, {"dims": (4, 129)}, {"dtype": 3}, {"scale": 0.0}, {"scale": float("nan")},
              {"tokens": -1}, {"tokens": 1 << 31}, {"seqs": -1}, {"index": 2}):
    assert call(**bad) == -1, bad
  assert call(tokens=0) == 0 and call(seqs=0) == 0


def test_custom_op_has_a_fake_kernel():
  with FakeTensorMode():
    q, k = torch.empty(10, 4, 32, device=DEV, dtype=BF16), torch.empty(10, 2, 32, device=DEV, dtype=BF16)
    v = torch.empty(10, 2, 24, device=DEV, dtype=BF16)
    out = ast.attention_causal_compiled(q, k, v, {"cu_seqlens": torch.empty(2, dtype=torch.int32, device=DEV)})
    assert out.shape == (10, 4, 24) and out.dtype == BF16


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_compiled_matches_eager(dtype):
  q, k, v, do = (x.to(DEV) for x in make([60, 30], (4, 2), (64, 64), dtype))
  args = {"cu_seqlens": cu_of([60, 30])}
  results = []
  for fn in (ast.attention_causal, torch.compile(ast.attention_causal_compiled, fullgraph=True)):
    x = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = fn(*x, args)
    results.append((out.detach(), *torch.autograd.grad(out, x, do)))
  for a, b in zip(*results):
    assert torch.equal(a, b)


@gpu
def test_backward_refuses_inputs_changed_since():
  q, k, v, do = (x.to(DEV) for x in make([60], (2, 2), (64, 64), BF16))
  q.requires_grad_(True)
  args = {"cu_seqlens": cu_of([60])}
  for change in (k, args["cu_seqlens"]):
    out = ast.attention_causal(q, k, v, args)
    change.add_(0)
    with pytest.raises(RuntimeError, match="inplace operation"):
      torch.autograd.grad(out, q, do)
