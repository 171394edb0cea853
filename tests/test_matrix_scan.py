"""The matrix-state scan and its one-token step against a token-by-token float64 oracle.

Tolerances (relative 2-norm per output, then largest error over the output's
root mean square) follow from the arithmetic:

* float32: sums of at most a few hundred float32 products, each rounded by
  2^-24: 1e-5, ten times the root of the count.
* 16-bit outputs: one rounding of the result (2^-8 for bfloat16, 2^-11 for
  float16 at most, less than half of it as a root mean square) and at most one
  of an operand inside each product, which averages to as much again: 2^-8 and
  2^-11; single elements may cancel, so 16 times that against the root mean
  square.
* float32 outputs of 16-bit inputs (states, gate gradients): the inputs are
  exact, operands that are computed keep at least 16 bits: 2e-5.
"""

from __future__ import annotations

import math

import pytest
import torch

import associative_scan_triton as ast
from associative_scan_triton import _lib

DEV = "cuda"
gpu = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TOL = {F32: 1e-5, F16: 2.0**-11, BF16: 2.0**-8}
STATE_TOL = 2e-5


def oracle(q, k, v, g, lengths, scale, s0=None, first=0):
  """Token by token in float64; leaves may require gradients.  (out, final)."""
  heads = max(x.shape[1] for x in (q, k, v, g))
  q, k, v, g = (x.repeat_interleave(heads // x.shape[1], 1) for x in (q, k, v, g))
  outs = [q.new_zeros(first, heads, v.shape[2])]
  finals, at = [], first
  for n, length in enumerate(lengths):
    state = s0[n] if s0 is not None else q.new_zeros(heads, q.shape[2], v.shape[2])
    for t in range(at, at + length):
      state = state * torch.exp(g[t])[:, None, None] + k[t][:, :, None] * v[t][:, None, :]
      outs.append(scale * (q[t][:, :, None] * state).sum(1)[None])
    finals.append(state)
    at += length
  return torch.cat(outs), torch.stack(finals)


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


def make(lengths, heads, dims, dtype, seed=0, gate_dtype=F32, carry=False, first=0, rate=0.3):
  """Inputs on the CPU in their type: q, k, v, g, s0, d_out, d_final."""
  gen = torch.Generator().manual_seed(seed)
  hq, hk, hv, hg = heads
  h, (dk, dv), n = max(heads), dims, first + sum(lengths)

  def normal(*shape):
    return torch.randn(shape, generator=gen)

  q = normal(n, hq, dk).to(dtype)
  k = normal(n, hk, dk).to(dtype)
  v = normal(n, hv, dv).to(dtype)
  g = (-rate * torch.rand(n, hg, generator=gen)**2).to(gate_dtype)
  s0 = normal(len(lengths), h, dk, dv) * 2 if carry else None
  d_out = normal(n, h, dv).to(dtype)
  d_final = normal(len(lengths), h, dk, dv) if carry else None
  return q, k, v, g, s0, d_out, d_final


def cu_of(lengths, first=0, dtype=torch.int32):
  ends = [first]
  for m in lengths:
    ends.append(ends[-1] + m)
  return torch.tensor(ends, dtype=dtype, device=DEV)


def check_forward(lengths, heads, dims, dtype, **kw):
  q, k, v, g, s0, _, _ = make(lengths, heads, dims, dtype, **kw)
  first = kw.get("first", 0)
  out, final = ast.matrix_scan_causal(
    q.to(DEV), k.to(DEV), v.to(DEV), g.to(DEV), {"cu_seqlens": cu_of(lengths, first)},
    initial_state=None if s0 is None else s0.to(DEV), return_final_state=True)
  assert out.dtype == dtype and final.dtype == F32
  want, want_final = oracle(q.double(), k.double(), v.double(), g.double(), lengths,
                            dims[0]**-0.5, None if s0 is None else s0.double(), first)
  close("out", out, want, TOL[dtype])
  close("final_state", final, want_final, STATE_TOL)


LENGTHS = [[1], [2], [0, 1, 0, 2, 0], [31, 32, 33], [127, 128, 129], [64, 0, 257, 5], [700, 1, 511]]


@gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_forward_lengths(lengths, dtype):
  check_forward(lengths, (2, 2, 2, 2), (64, 64), dtype, carry=True)


@gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dims", [(128, 128), (64, 128), (128, 64), (16, 8), (1, 1), (40, 72), (96, 33),
                                  (127, 80), (3, 128), (128, 1)], ids=str)
def test_forward_head_sizes(dims, dtype):
  check_forward([150, 3], (3, 3, 3, 3), dims, dtype)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads", [(1, 1, 1, 1), (4, 1, 1, 1), (2, 2, 4, 4), (1, 2, 4, 1), (6, 3, 2, 6),
                                   (4, 4, 1, 4)], ids=str)
def test_forward_shared_heads(heads, dtype):
  check_forward([130, 70], heads, (64, 64), dtype, gate_dtype=dtype)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lengths", [[2600], [1024, 1024, 512], [100, 2300, 3]], ids=str)
def test_forward_across_segments(lengths, dtype):
  # one head of few tokens per SM: the packed axis is cut into many segments
  check_forward(lengths, (1, 1, 1, 1), (64, 64), dtype, carry=True, rate=0.02)


@gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_tokens_of_no_sequence(dtype):
  # rows before cu_seqlens[0] hold NaN: they are not read, and come out zero
  q, k, v, g, _, _, _ = make([60, 90], (2, 2, 2, 2), (64, 64), dtype, first=37)
  clean = [x.clone() for x in (q, k, v, g)]
  for x in (q, k, v, g):
    x[:37] = math.nan
  out = ast.matrix_scan_causal(*(x.to(DEV) for x in (q, k, v, g)),
                               {"cu_seqlens": cu_of([60, 90], 37, torch.int64)})
  want, _ = oracle(*(x.double() for x in clean), [60, 90], 64**-0.5, first=37)
  assert not out[:37].any()
  close("out", out, want, TOL[dtype])


@gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("gates", ["drop", "one", "steep", "mixed", "growing"])
def test_gates(gates, dtype):
  lengths = [200, 77]
  q, k, v, g, s0, _, _ = make(lengths, (2, 2, 2, 2), (64, 64), dtype, carry=True)
  if gates == "drop":  # nothing is kept anywhere: every row sees itself alone
    g.fill_(-math.inf)
  elif gates == "one":
    g.zero_()
  elif gates == "steep":  # sums of thousands inside a chunk
    g.fill_(-37.5)
    g[::3] = -0.01
  elif gates == "mixed":
    g[torch.randperm(277, generator=torch.Generator().manual_seed(3))[:60]] = -math.inf
  else:
    g = g * -0.1
  out, final = ast.matrix_scan_causal(*(x.to(DEV) for x in (q, k, v, g)),
                                      {"cu_seqlens": cu_of(lengths)}, initial_state=s0.to(DEV),
                                      return_final_state=True)
  want, want_final = oracle(q.double(), k.double(), v.double(), g.double(), lengths, 64**-0.5,
                            s0.double())
  close("out", out, want, TOL[dtype])
  close("final_state", final, want_final, STATE_TOL)


@gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("where", [0, 1, 2])
def test_values_that_are_not_finite_stay_behind_the_mask(where, bad, dtype):
  # a bad query, key or value at token t touches no earlier token of its
  # sequence and no token of another
  lengths = [90, 150, 40]
  tensors = list(make(lengths, (2, 2, 2, 2), (64, 64), dtype)[:4])
  want, _ = oracle(*(x.double() for x in tensors), lengths, 64**-0.5)
  t = 90 + 71
  tensors[where][t, 1, 5] = bad
  out = ast.matrix_scan_causal(*(x.to(DEV) for x in tensors), {"cu_seqlens": cu_of(lengths)})
  keep = torch.ones(280, 2, dtype=torch.bool)
  keep[t if where == 0 else slice(t, 240), 1] = False
  close("out", out.cpu()[keep], want[keep], TOL[dtype])
  assert not torch.isfinite(out[t, 1]).all()


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strided_and_misaligned_inputs(dtype):
  # views of one packed projection, and the same shifted by one element
  lengths, h, d = [100, 61], 3, 64
  gen = torch.Generator().manual_seed(5)
  flat = torch.randn(161 * (3 * h * d + h) + 1, generator=gen).to(dtype).to(DEV)
  gates = (-0.2 * torch.rand(h, 161, generator=gen)).to(DEV).t()
  for shift in (0, 1):
    packed = flat[shift:shift + 161 * (3 * h * d + h)].view(161, -1)
    q, k, v = (packed[:, i * h * d:(i + 1) * h * d].view(161, h, d) for i in range(3))
    out = ast.matrix_scan_causal(q, k, v, gates, {"cu_seqlens": cu_of(lengths)})
    want, _ = oracle(*(x.double().cpu() for x in (q, k, v, gates)), lengths, d**-0.5)
    close(f"out shifted by {shift}", out, want, TOL[dtype])


def run_gradients(tensors, lengths, scale=None, first=0, use=("out", "final")):
  """(our gradients, the oracle's) of sum(out*d_out) + sum(final*d_final)."""
  q, k, v, g, s0, d_out, d_final = tensors
  leaves = [x.to(DEV).requires_grad_(True) for x in (q, k, v, g)]
  init = None if s0 is None else s0.to(DEV).requires_grad_(True)
  out, final = ast.matrix_scan_causal(*leaves, {"cu_seqlens": cu_of(lengths, first)}, scale=scale,
                                      initial_state=init, return_final_state=True)
  ends = [x for x, name in ((out, "out"), (final, "final")) if name in use]
  grads = [x.to(DEV) for x, name in ((d_out, "out"), (d_final, "final")) if name in use]
  wrt = leaves + ([init] if init is not None else [])
  ours = torch.autograd.grad(ends, wrt, grads)
  leaves = [x.double().requires_grad_(True) for x in (q, k, v, g)]
  init = None if s0 is None else s0.double().requires_grad_(True)
  out, final = oracle(*leaves, lengths, scale if scale is not None else q.shape[2]**-0.5, init, first)
  ends = [x for x, name in ((out, "out"), (final, "final")) if name in use]
  wrt = leaves + ([init] if init is not None else [])
  gold = torch.autograd.grad(ends, wrt, [x.cpu().double() for x in grads], allow_unused=True)
  return ours, [torch.zeros_like(w) if x is None else x for x, w in zip(gold, wrt)]


NAMES = ("d_queries", "d_keys", "d_values", "d_log_gates", "d_initial_state")


def check_gradients(tensors, lengths, dtype, gate_dtype=F32, **kw):
  ours, gold = run_gradients(tensors, lengths, **kw)
  for name, a, b in zip(NAMES, ours, gold):
    tol = TOL[dtype]
    if name == "d_initial_state" or (name == "d_log_gates" and gate_dtype == F32):
      tol = STATE_TOL
    assert a.dtype == (F32 if name == "d_initial_state" else
                       gate_dtype if name == "d_log_gates" else dtype)
    close(name, a, b, tol)


@gpu
@pytest.mark.parametrize("lengths,heads,dims", [([244], 5, (128, 64)), ([130, 200, 1, 180], 5, (64, 128)),
                                                ([700, 556], 4, (128, 128)), ([206], 8, (40, 72))], ids=str)
def test_float32_gate_gradients_of_bfloat16_inputs(lengths, heads, dims):
  # computed operands keep 16 bits, 2^-17 = 7.6e-6 of a term at most, and the
  # stretch of rows that a gradient sums is a chunk: below 1e-5 of its norm
  ours, gold = run_gradients(make(lengths, (heads,) * 4, dims, BF16, carry=True), lengths)
  at = NAMES.index("d_log_gates")
  want = gold[at].double()
  error = ((ours[at].double().cpu() - want).norm() / want.norm()).item()
  assert error <= 1e-5, error


@gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_gradient_lengths(lengths, dtype):
  check_gradients(make(lengths, (2, 2, 2, 2), (64, 64), dtype, carry=True), lengths, dtype)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dims", [(128, 128), (64, 128), (128, 64), (40, 72), (5, 1)], ids=str)
def test_gradient_head_sizes(dims, dtype):
  check_gradients(make([140, 9], (2, 2, 2, 2), dims, dtype), [140, 9], dtype, use=("out",))


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads", [(4, 1, 1, 1), (2, 2, 4, 4), (1, 2, 4, 1), (6, 3, 2, 6)], ids=str)
def test_gradient_shared_heads(heads, dtype):
  tensors = make([90, 50], heads, (64, 64), dtype, gate_dtype=dtype)
  check_gradients(tensors, [90, 50], dtype, gate_dtype=dtype, use=("out",))


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rate", [0.002, 0.3, 6.0])
def test_gradient_across_segments_and_stored_states(rate, dtype):
  lengths = [100, 2500]
  tensors = make(lengths, (1, 1, 1, 1), (64, 64), dtype, carry=True, rate=rate)
  check_gradients(tensors, lengths, dtype)


@gpu
def test_gradient_of_the_final_state_alone():
  tensors = make([70, 0, 200], (2, 2, 2, 2), (64, 64), F32, carry=True)
  check_gradients(tensors, [70, 0, 200], F32, use=("final",))


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradient_scale_gates_and_outside_tokens(dtype):
  tensors = list(make([80, 75], (2, 1, 2, 2), (64, 64), dtype, first=11))
  tensors[3][30::17] = -math.inf
  ours, gold = run_gradients(tensors, [80, 75], scale=0.3, first=11, use=("out",))
  for name, a, b in zip(NAMES, ours, gold):
    if name == "d_log_gates":  # exp's own gradient at -inf is 0; so is ours
      b = torch.where(torch.isfinite(tensors[3].double()), b, torch.zeros_like(b))
    close(name, a, b, STATE_TOL if name == "d_log_gates" else TOL[dtype])
    assert not a[:11].any()


@gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_gates_that_nothing_passes_have_no_gradient(dtype):
  # the first token of a sequence without an initial state, and a dropped gate:
  # zero, not what rounding leaves of sums that cancel
  lengths = [1, 1, 300, 1]
  q, k, v, g, _, d_out, _ = make(lengths, (2, 2, 2, 2), (64, 64), dtype)
  g[50] = -math.inf
  g[77] = -150.0
  leaf = g.to(DEV).requires_grad_(True)
  out = ast.matrix_scan_causal(q.to(DEV), k.to(DEV), v.to(DEV), leaf, {"cu_seqlens": cu_of(lengths)})
  (d_gates,) = torch.autograd.grad(out, leaf, d_out.to(DEV))
  for t in (0, 1, 2, 50, 77, 302):
    assert not d_gates[t].any(), t
  assert d_gates[3:50].any() and torch.isfinite(d_gates).all()


@gpu
def test_gradient_by_differences():
  # central differences of a float64 evaluation of the loss at float32 inputs
  # moved by +-h: truncation h^2 ~ 1e-8, so only our own 1e-5 remains; 1e-4
  lengths = [50, 90]
  tensors = make(lengths, (2, 1, 2, 2), (32, 32), F32, carry=True)
  q, k, v, g, s0, d_out, d_final = tensors
  ours, _ = run_gradients(tensors, lengths)
  gen = torch.Generator().manual_seed(9)
  base = [x.double() for x in (q, k, v, g, s0)]

  def loss(parts):
    out, final = oracle(*parts[:4], lengths, 32**-0.5, parts[4])
    return float((out * d_out.double()).sum() + (final * d_final.double()).sum())

  for i, name in enumerate(NAMES):
    direction = torch.randn(base[i].shape, generator=gen, dtype=torch.float64)
    h = 1e-4
    up = [x + h * direction if j == i else x for j, x in enumerate(base)]
    down = [x - h * direction if j == i else x for j, x in enumerate(base)]
    slope = (loss(up) - loss(down)) / (2 * h)
    ours_slope = float((ours[i].double().cpu() * direction).sum())
    size = float(ours[i].double().norm())
    assert abs(slope - ours_slope) <= 1e-4 * size, (name, slope, ours_slope)


@gpu
@pytest.mark.parametrize("lengths,heads,dims", [([300], (2, 2, 2, 2), (128, 128)), ([130, 0, 71, 400], (4, 2, 4, 4), (64, 128)),
                                                ([1100], (1, 1, 1, 1), (40, 72)), ([5], (3, 3, 3, 3), (64, 64))], ids=str)
def test_bfloat16_results_are_rounded_once(lengths, heads, dims):
  # Computed operands (masked scores, the state, what enters it) keep 16 bits,
  # so a result is within 2^-16 of its size before its rounding, d = 1.5e-5.  It
  # then differs from the rounded exact value where a rounding boundary lies
  # between: in a share d / ulp of the elements, by one ulp (2^-7 of a value at
  # most), so by sqrt(d * 2^-7) = 3.5e-4 of the norm.  One operand of 8 bits
  # gives 2^-9 and more.
  tensors = make(lengths, heads, dims, BF16, seed=2, carry=True)
  ours, gold = run_gradients(tensors, lengths)
  q, k, v, g, s0, _, _ = tensors
  out = ast.matrix_scan_causal(q.to(DEV), k.to(DEV), v.to(DEV), g.to(DEV), {"cu_seqlens": cu_of(lengths)},
                               initial_state=s0.to(DEV))
  want, _ = oracle(q.double(), k.double(), v.double(), g.double(), lengths, dims[0]**-0.5, s0.double())
  for name, a, b in zip(("out",) + NAMES[:3], (out, *ours), (want, *gold)):
    rounded = b.to(BF16).double()
    apart = float((a.double().cpu() - rounded).norm() / rounded.norm())
    assert apart <= 2.0**-11, (name, apart)


@gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("gate", [-1.0, -4.0, -8.0, -12.0])
@pytest.mark.parametrize("lengths,heads,dims", [([300], 2, (64, 64)), ([70, 1, 401], 2, (128, 128)), ([190], 3, (40, 24))],
                         ids=str)
def test_gate_gradients_at_strong_decay(lengths, heads, dims, gate, dtype):
  # every term of a gate's gradient carries the decay e^gate, and so must the
  # terms that are summed for it: the usual bounds hold at any gate
  tensors = list(make(lengths, (heads,) * 4, dims, dtype, seed=6))
  tensors[3].fill_(gate)
  ours, gold = run_gradients(tensors, lengths, use=("out",))
  at = NAMES.index("d_log_gates")
  close("d_log_gates", ours[at], gold[at], STATE_TOL if dtype != F32 else TOL[F32])


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gate_gradients_at_strong_decay_with_states_and_shared_heads(dtype):
  lengths = [150, 260]
  tensors = list(make(lengths, (2, 4, 1, 4), (64, 64), dtype, seed=8, carry=True))
  tensors[3].fill_(-8.0)
  tensors[3][140:160] = -0.1  # some of the state leaves the first sequence, and enters the second
  check_gradients(tensors, lengths, dtype)


@gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("at", [0, 1, 2, 3, 31, 32, 127, 130, 257])
def test_gates_that_are_not_finite_stay_behind_the_mask(at, bad, dtype):
  # a bad gate at token t reaches no earlier output, no gradient of a later
  # key or value (their paths start behind it), no earlier query's gradient,
  # and nothing of another sequence or head
  lengths = [90, 300, 40]
  q, k, v, g, _, d_out, _ = make(lengths, (2, 2, 2, 2), (64, 64), dtype)
  ours_g = g.clone()
  t = 90 + at
  ours_g[t, 1] = bad
  leaves = [x.to(DEV).requires_grad_(True) for x in (q, k, v, ours_g)]
  out = ast.matrix_scan_causal(*leaves, {"cu_seqlens": cu_of(lengths)})
  d_q, d_k, d_v, d_g = (x.cpu() for x in torch.autograd.grad(out, leaves, d_out.to(DEV)))
  gold = [x.double().requires_grad_(True) for x in (q, k, v, g)]
  want, _ = oracle(*gold, lengths, 64**-0.5)
  want_q, want_k, want_v, want_g = torch.autograd.grad(want, gold, d_out.double())
  before = torch.ones(430, 2, dtype=torch.bool)
  before[t:390, 1] = False  # what the bad gate is not before
  after = torch.ones(430, 2, dtype=torch.bool)
  after[90:t, 1] = False
  apart = before & after  # ... nor its gradient's terms
  apart[90:390, 1] = False
  if at > 0:
    assert not torch.isfinite(out[t, 1]).all()
  for name, got, gold, keep in (("out", out.detach().cpu(), want, before), ("d_queries", d_q, want_q, before),
                                ("d_keys", d_k, want_k, after), ("d_values", d_v, want_v, after)):
    close(name, got[keep], gold[keep], TOL[dtype])
  close("d_log_gates", d_g[apart], want_g[apart], STATE_TOL)


@gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("where", [0, 1, 2, 3])
def test_gradients_of_values_that_are_not_finite_stay_behind_the_mask(where, bad, dtype):
  # queries and upstream gradients reach their own and earlier tokens' key and
  # value gradients, keys and values the later queries' and each other's row
  lengths = [90, 150, 40]
  q, k, v, g, _, d_out, _ = make(lengths, (2, 2, 2, 2), (64, 64), dtype)
  gold = [x.double().requires_grad_(True) for x in (q, k, v)]
  want, _ = oracle(*gold, g.double(), lengths, 64**-0.5)
  want = torch.autograd.grad(want, gold, d_out.double())
  inputs = [q, k, v, d_out]
  t = 90 + 71
  inputs[where] = inputs[where].clone()
  inputs[where][t, 1, 5] = bad
  leaves = [x.to(DEV).requires_grad_(True) for x in inputs[:3]]
  out = ast.matrix_scan_causal(*leaves, g.to(DEV), {"cu_seqlens": cu_of(lengths)})
  found = torch.autograd.grad(out, leaves, inputs[3].to(DEV))
  row, earlier, later, none = slice(t, t + 1), slice(90, t + 1), slice(t, 240), slice(0, 0)
  reached = ((none, earlier, earlier), (later, none, row), (later, row, none), (row, earlier, earlier))[where]
  for name, got, gold, rows in zip(NAMES, found, want, reached):
    keep = torch.ones(280, 2, dtype=torch.bool)
    keep[rows, 1] = False
    close(name, got.cpu()[keep], gold[keep], TOL[dtype])


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lengths", [[2048] * 8, [16384]], ids=["2048x8", "16384"])
def test_states_of_long_memory_do_not_drift(lengths, dtype):
  # positive operands and gates of 0: a state only grows, and every chunk adds
  # to one that is larger than itself.  A chunk's own sums are good to 2^-22,
  # and the states that they are added to in float32 round 128 times at most,
  # by 2^-25 on average and either way: 2^-21 of the norm together
  heads, d = 12, 128
  total, n = sum(lengths), len(lengths)
  gen = torch.Generator(device=DEV).manual_seed(4)
  q, k, v, d_out = (torch.randn(total, heads, d, generator=gen, device=DEV).abs().to(dtype) for _ in range(4))
  gates = torch.zeros(total, heads, device=DEV)
  s0 = torch.zeros(n, heads, d, d, device=DEV, requires_grad=True)
  out, final = ast.matrix_scan_causal(q, k, v, gates, {"cu_seqlens": cu_of(lengths)}, scale=1.0, initial_state=s0,
                                      return_final_state=True)
  (d_initial,) = torch.autograd.grad(out, s0, d_out)
  for name, got, a, b in (("final_state", final, k, v), ("d_initial_state", d_initial, q, d_out)):
    want = torch.einsum("nthi,nthj->nhij", *(x.double().view(n, -1, heads, d) for x in (a, b)))
    apart = float((got.double() - want).norm() / want.norm())
    assert apart <= 2.0**-21, (name, apart)


@gpu
@pytest.mark.parametrize("rate", [0.01, 0.3, 6.0])
@pytest.mark.parametrize("lengths,heads,dims", [([257], 2, (128, 128)), ([130, 0, 71, 400], 3, (64, 128)), ([1300], 1, (128, 64)),
                                                ([5], 2, (40, 72))], ids=str)
def test_float32_states_of_bfloat16_inputs(lengths, heads, dims, rate):
  # what enters a state keeps 24 bits, its decay two factors good to 2^-22, and
  # it is summed and scaled in float32: 2^-20 of its norm, as float32 inputs have
  tensors = make(lengths, (heads,) * 4, dims, BF16, seed=3, carry=True, rate=rate)
  q, k, v, g, s0, _, _ = tensors
  _, final = ast.matrix_scan_causal(q.to(DEV), k.to(DEV), v.to(DEV), g.to(DEV), {"cu_seqlens": cu_of(lengths)},
                                    initial_state=s0.to(DEV), return_final_state=True)
  _, want = oracle(q.double(), k.double(), v.double(), g.double(), lengths, dims[0]**-0.5, s0.double())
  ours, gold = run_gradients(tensors, lengths)
  for name, a, b in (("final_state", final, want), (NAMES[4], ours[4], gold[4])):
    apart = float((a.double().cpu() - b).norm() / b.norm())
    assert apart <= 2.0**-20, (name, apart)


@gpu
@pytest.mark.parametrize("lengths,dims", [([2600], (64, 64)), ([100, 2300, 3], (128, 128)), ([1024, 1024, 512], (40, 72))], ids=str)
def test_bfloat16_across_segments_without_float32_results(lengths, dims):
  # nothing float32 is asked for: what enters a state keeps 16 bits, and the
  # outputs and gradients are held to the same bounds
  tensors = make(lengths, (1, 1, 1, 1), dims, BF16, seed=15, gate_dtype=BF16, rate=0.02)
  q, k, v, g, _, d_out, _ = tensors
  leaves = [x.to(DEV).requires_grad_(True) for x in (q, k, v, g)]
  out = ast.matrix_scan_causal(*leaves, {"cu_seqlens": cu_of(lengths)})
  ours = torch.autograd.grad(out, leaves, d_out.to(DEV))
  gold = [x.double().requires_grad_(True) for x in (q, k, v, g)]
  want, _ = oracle(*gold, lengths, dims[0]**-0.5)
  close("out", out, want, TOL[BF16])
  for name, a, b in zip(NAMES, ours, torch.autograd.grad(want, gold, d_out.double())):
    close(name, a, b, TOL[BF16])


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_repeats_bit_for_bit_on_another_stream_and_in_a_graph(dtype):
  lengths = [300, 1000]
  q, k, v, g, s0, _, _ = (x if x is None else x.to(DEV)
                          for x in make(lengths, (2, 2, 2, 2), (64, 64), dtype, carry=True))
  args = {"cu_seqlens": cu_of(lengths)}

  def call():
    return ast.matrix_scan_causal(q, k, v, g, args, initial_state=s0, return_final_state=True)

  first = call()
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    second = call()
  torch.cuda.current_stream().wait_stream(side)
  sync_check = _lib.sync_check_enabled()
  _lib.set_sync_check(False)  # a synchronisation is not allowed while capturing
  try:
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      third = call()
    for x in third:
      x.zero_()
    graph.replay()
    torch.cuda.synchronize()
  finally:
    _lib.set_sync_check(sync_check)
  for a, b, c in zip(first, second, third):
    assert torch.equal(a, b) and torch.equal(a, c)


@gpu
@pytest.mark.parametrize("backward", [False, True])
def test_a_thread_without_a_cuda_context(backward):
  # a new thread whose first CUDA work is this call, every buffer coming from
  # torch's cache: nothing has made a context current in it yet
  import threading

  from associative_scan_triton import matrix_scan
  q, k, v, g, _, d_out, _ = (x if x is None else x.to(DEV)
                             for x in make([70], (2, 2, 2, 2), (64, 64), BF16))
  cu = cu_of([70])

  def call():
    if backward:
      return matrix_scan._scan_backward(q, k, v, g, cu, 0.125, None, None, d_out, None)[:4]
    return matrix_scan._scan_forward(q, k, v, g, cu, 0.125, None, True)

  want = call()
  found = []
  for x in want:  # leaves free blocks of every size that the call needs
    found.append(x.clone())
  want, found = found, []
  torch.cuda.synchronize()
  sync_check = _lib.sync_check_enabled()
  _lib.set_sync_check(False)
  try:
    thread = threading.Thread(target=lambda: found.append(call()))
    thread.start()
    thread.join()
  finally:
    _lib.set_sync_check(sync_check)
  assert found, "the call failed in the new thread"
  for a, b in zip(found[0], want):
    assert torch.equal(a, b)


@gpu
def test_empty_inputs():
  q = torch.empty(0, 2, 16, device=DEV, requires_grad=True)
  g = torch.empty(0, 2, device=DEV)
  s0 = torch.randn(2, 2, 16, 16, device=DEV)
  out, final = ast.matrix_scan_causal(q, q, q, g, {"cu_seqlens": cu_of([0, 0])}, initial_state=s0,
                                      return_final_state=True)
  assert out.shape == (0, 2, 16) and torch.equal(final, s0)
  out.sum().backward()
  assert q.grad.shape == q.shape


@gpu
def test_malformed_sequences_are_reported():
  q = torch.randn(50, 1, 32, device=DEV)
  g = torch.zeros(50, 1, device=DEV)
  for cu in ([0, 49], [0, 60], [0, 30, 20, 50], [-3, 50]):
    with pytest.raises(ast.ScanError, match="cu_seqlens"):
      ast.matrix_scan_causal(q, q, q, g, {"cu_seqlens": torch.tensor(cu, device=DEV)})
      ast.check_device_error()


@gpu
def test_refusals():
  q = torch.randn(10, 2, 32, device=DEV)
  g = torch.zeros(10, 2, device=DEV)
  args = {"cu_seqlens": cu_of([10])}

  def refused(error, match, q=q, k=q, v=q, g=g, **kw):
    with pytest.raises(error, match=match):
      ast.matrix_scan_causal(q, k, v, g, {**args, **kw.pop("args", {})}, **kw)

  refused(ValueError, "CUDA tensors only", q=q.cpu())
  refused(TypeError, "keys has dtype", k=q.half())
  refused(TypeError, "unsupported dtype", q=q.double())
  refused(TypeError, "log_gates must be", g=g.half())
  refused(ValueError, "3 dimensions", v=q[0])
  refused(ValueError, "2 dimensions", g=q)
  refused(ValueError, "rows", v=q[:9])
  refused(ValueError, "head size", k=q[..., :16])
  refused(ValueError, "unit stride", v=q.transpose(1, 2).contiguous().transpose(1, 2))
  refused(ValueError, "divide", v=torch.randn(10, 3, 32, device=DEV))
  refused(ValueError, "head sizes up to 128", v=torch.randn(10, 2, 129, device=DEV))
  refused(TypeError, "int32 or int64", args={"cu_seqlens": args["cu_seqlens"].float()})
  refused(ValueError, "one dimension", args={"cu_seqlens": args["cu_seqlens"][None]})
  refused(ValueError, "initial_state has shape", initial_state=torch.zeros(1, 2, 32, 31, device=DEV))
  refused(TypeError, "initial_state must be float32",
          initial_state=torch.zeros(1, 2, 32, 32, device=DEV, dtype=F16))


def test_cpu_tensors_are_refused():
  q = torch.zeros(4, 1, 8)
  g = torch.zeros(4, 1)
  cu = torch.tensor([0, 4])
  with pytest.raises(ValueError, match="CUDA tensors only"):
    ast.matrix_scan_causal(q, q, q, g, {"cu_seqlens": cu})
  with pytest.raises(ValueError, match="CUDA tensors only"):
    ast.matrix_scan_step(q, q, q, g, torch.zeros(4, 1, 8, 8))


def test_abi_rejects_bad_arguments_without_a_gpu():
  import ctypes
  lib = _lib.load()
  r = ctypes.byref(_lib.Rows(1 << 20, 8, 8, 1))
  three = ctypes.byref(_lib.Rows(1 << 20, 8, 8, 3))
  none = ctypes.byref(_lib.Rows(None, 8, 8, 1))
  ok = [r, r, r, r, 0, 1 << 20, 0, 1, 4, 2, 8, 8, 0, 1.0, None, 1 << 20, None, None, 0, None]

  def rc(**changes):
    a = list(ok)
    for at, value in changes.items():
      a[int(at[1:])] = value
    return lib.ascan_matrix_scan_forward(*a)

  assert rc() == -2  # everything in order but the workspace
  for changes in ({"_0": three}, {"_1": none}, {"_4": 3}, {"_5": None}, {"_6": 2}, {"_7": -1},
                  {"_8": -1}, {"_9": 0}, {"_10": 129}, {"_11": 0}, {"_12": 5}, {"_15": None}):
    assert rc(**changes) == -1, changes
  assert rc(_8=0) == 0 and rc(_7=0) == 0
  assert lib.ascan_matrix_scan_workspace(0, 0, 0, 0, 0, 0, 0, 0, 0, 0) >= 256
  small = lib.ascan_matrix_scan_workspace(4096, 1, 2, 2, 2, 2, 2, 64, 64, 0)
  assert lib.ascan_matrix_scan_workspace(4096, 1, 2, 2, 2, 2, 2, 64, 64, 1) > small


@gpu
def test_backward_refuses_cu_seqlens_changed_since():
  # a loop that packs into one buffer: the backward must not read the next batch's ends
  q, k, v, g, _, d_out, _ = (x if x is None else x.to(DEV) for x in make([30, 20], (2, 2, 2, 2), (16, 16), F32))
  cu = cu_of([30, 20])
  out = ast.matrix_scan_causal(q.requires_grad_(True), k, v, g, {"cu_seqlens": cu})
  cu[1] = 10
  with pytest.raises(RuntimeError, match="inplace operation"):
    out.backward(d_out)


def test_workspace_holds_the_states_that_the_types_store():
  # both directions' states: every 128 tokens for float32 gates on the tensor
  # cores, every 256 in float32 arithmetic, every 1024 for gates of 16 bits
  lib = _lib.load()
  f32, f16, bf16 = 0, 1, 2
  tokens, heads, dims = 65536, 12, (128, 128)
  sizes = (tokens, 1, heads, heads, heads, heads, heads, *dims)
  state = 4 * heads * dims[0] * dims[1]
  every = lambda n: 2 * (tokens // n + 1) * state
  fine, coarse = (lib.ascan_matrix_scan_workspace_of(*sizes, bf16, g, 1) for g in (f32, bf16))
  assert fine - coarse == every(128) - every(1024)
  fine, coarse = (lib.ascan_matrix_scan_workspace_of(*sizes, f16, g, 1) for g in (f32, f16))
  assert fine - coarse == every(256) - every(1024)
  # all else: row dots of both directions in halves, carries of at most 64 segments
  assert coarse <= every(1024) + 4 * 4 * tokens * heads + 3 * 64 * state + 2**20
  for backward in (0, 1):
    most = lib.ascan_matrix_scan_workspace(*sizes, backward)
    assert most == max(lib.ascan_matrix_scan_workspace_of(*sizes, d, g, backward)
                       for d in (f32, f16, bf16) for g in (f32, f16, bf16))


# ---------------------------------------------------------------------------
# one token
# ---------------------------------------------------------------------------


def step_oracle(q, k, v, g, state, scale):
  heads = state.shape[1]
  q, k, v, g = (x.double().repeat_interleave(heads // x.shape[1], 1) for x in (q, k, v, g))
  new = state.double() * torch.exp(g)[..., None, None] + k[..., :, None] * v[..., None, :]
  return scale * (q[..., None] * new).sum(-2), new


@gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dims", [(128, 128), (64, 32), (40, 72), (7, 5), (200, 260)], ids=str)
@pytest.mark.parametrize("batch", [1, 3, 170])
def test_step(batch, dims, dtype):
  heads, (dk, dv) = (2, 1, 4, 4), dims
  q, k, v, g, _, _, _ = (x if x is None else x.to(DEV) for x in make([batch], heads, dims, dtype))
  gen = torch.Generator().manual_seed(1)
  pool = torch.randn(batch + 5, 4, dk, dv, generator=gen).to(DEV)
  slots = torch.randperm(batch + 5, generator=gen)[:batch].to(torch.int32).to(DEV)
  want, new = step_oracle(q, k, v, g, pool[slots.long()], 0.5)
  before = pool.clone()
  other = torch.full_like(pool, 7.0)
  out = ast.matrix_scan_step(q, k, v, g, pool, slots=slots, scale=0.5, state_out=other)
  assert torch.equal(pool, before)
  close("out", out, want, TOL[dtype])
  close("state", other[slots.long()], new, 1e-6)
  idle = torch.ones(batch + 5, dtype=torch.bool, device=DEV)
  idle[slots.long()] = False
  assert (other[idle] == 7.0).all()
  again = ast.matrix_scan_step(q, k, v, g, pool, slots=slots, scale=0.5)
  assert torch.equal(out, again) and torch.equal(pool[slots.long()], other[slots.long()])
  assert torch.equal(pool[idle], before[idle])


@gpu
def test_step_idle_rows_and_slots_outside_the_pool():
  q, k, v, g, _, _, _ = (x if x is None else x.to(DEV) for x in make([3], (2, 2, 2, 2), (32, 32), F32))
  pool = torch.randn(4, 2, 32, 32, device=DEV)
  before = pool.clone()
  q[1] = k[1] = v[1] = math.nan
  slots = torch.tensor([2, -1, 0], dtype=torch.int32, device=DEV)
  want, new = step_oracle(q, k, v, g, before[slots.long()], 32**-0.5)
  out = ast.matrix_scan_step(q, k, v, g, pool, slots=slots)
  assert not out[1].any()
  close("out", out[[0, 2]], want[[0, 2]], 1e-5)
  assert torch.equal(pool[[1, 3]], before[[1, 3]])
  with pytest.raises(ast.ScanError, match="slot"):
    ast.matrix_scan_step(q, k, v, g, pool, slots=slots + 2)
    ast.check_device_error()


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_step_continues_the_scan(dtype):
  lengths = [40, 3]
  q, k, v, g, s0, _, _ = (x if x is None else x.to(DEV)
                          for x in make(lengths, (2, 2, 2, 2), (64, 64), dtype, carry=True))
  whole, final = ast.matrix_scan_causal(q, k, v, g, {"cu_seqlens": cu_of(lengths)}, initial_state=s0,
                                        return_final_state=True)
  head = torch.cat((torch.arange(39), torch.arange(40, 42))).to(DEV)
  _, state = ast.matrix_scan_causal(*(x[head] for x in (q, k, v, g)), {"cu_seqlens": cu_of([39, 2])},
                                    initial_state=s0, return_final_state=True)
  last = torch.tensor([39, 42], device=DEV)
  out = ast.matrix_scan_step(*(x[last] for x in (q, k, v, g)), state)
  close("out", out, whole[last].double(), 2 * TOL[dtype])
  close("state", state, final.double(), 2 * STATE_TOL)


@gpu
def test_step_refusals():
  q = torch.randn(3, 2, 16, device=DEV)
  g = torch.zeros(3, 2, device=DEV)
  pool = torch.zeros(4, 2, 16, 16, device=DEV)
  slots = torch.arange(3, dtype=torch.int32, device=DEV)

  def refused(error, match, g=g, state=pool, **kw):
    with pytest.raises(error, match=match):
      ast.matrix_scan_step(q, q, q, g, state, **kw)

  refused(ValueError, "state has shape", state=pool[:, :1])
  refused(TypeError, "state must be float32", state=pool.half())
  refused(ValueError, "slots must be", slots=slots.long())
  refused(ValueError, "slots must be", slots=slots[:2])
  refused(ValueError, "need 3 states", state=pool[:2].contiguous())
  both = torch.zeros(5, 2, 16, 16, device=DEV)
  refused(ValueError, "overlaps", state=both[:4], state_out=both[1:])
  refused(ValueError, "no backward", g=g.clone().requires_grad_(True))


@gpu
@pytest.mark.slow
def test_step_pool_beyond_32_bit_offsets():
  slots_total = 2**31 // (128 * 128) + 3
  pool = torch.empty(slots_total, 1, 128, 128, device=DEV)
  q, k, v, g, _, _, _ = (x if x is None else x.to(DEV) for x in make([2], (1, 1, 1, 1), (128, 128), F32))
  slots = torch.tensor([slots_total - 1, 0], dtype=torch.int32, device=DEV)
  pool[slots.long()] = torch.randn(2, 1, 128, 128, device=DEV)
  want, new = step_oracle(q, k, v, g, pool[slots.long()], 128**-0.5)
  out = ast.matrix_scan_step(q, k, v, g, pool, slots=slots)
  close("out", out, want, 1e-5)
  close("state", pool[slots.long()], new, 1e-6)


@gpu
@pytest.mark.parametrize("stepped", ["final_state", "initial_state", "other"])
def test_backward_refuses_a_state_that_a_step_has_overwritten(stepped):
  # the scan's gradients need the states as they were; a step in place shows in
  # the tensor's version like any of torch's own writes
  q, k, v, g, s0, _, d_final = (x.to(DEV) for x in make([20, 9], (2, 2, 2, 2), (16, 16), F32, carry=True))
  out, final = ast.matrix_scan_causal(q.clone().requires_grad_(True), k, v, g, {"cu_seqlens": cu_of([20, 9])},
                                      initial_state=s0, return_final_state=True)
  pool = {"final_state": final.detach(), "initial_state": s0, "other": torch.zeros_like(s0)}[stepped]
  version = pool._version
  ast.matrix_scan_step(q[:2], k[:2], v[:2], g[:2], pool)
  assert pool._version > version
  if stepped == "other":
    torch.autograd.backward([out, final], [out.detach(), d_final])
  else:
    with pytest.raises(RuntimeError, match="inplace operation"):
      torch.autograd.backward([out, final], [out.detach(), d_final])


@gpu
def test_step_marks_only_what_it_writes():
  q, k, v, g, _, _, _ = (x if x is None else x.to(DEV) for x in make([3], (2, 2, 2, 2), (16, 16), F32))
  pool, other = torch.zeros(3, 2, 16, 16, device=DEV), torch.zeros(3, 2, 16, 16, device=DEV)
  was = pool._version, other._version
  ast.matrix_scan_step(q, k, v, g, pool, state_out=other)
  assert pool._version == was[0] and other._version > was[1]
  with torch.inference_mode():  # such tensors have no version to mark
    made = torch.zeros(3, 2, 16, 16, device=DEV)
    out = ast.matrix_scan_step(q, k, v, g, made)
    assert torch.equal(made, other)
    assert torch.equal(ast.matrix_scan_step(q, k, v, g, pool), out)


@gpu
def test_step_with_an_empty_pool():
  # slots are checked against a pool of no states like any other
  q, k, v, g, _, _, _ = (x if x is None else x.to(DEV) for x in make([3], (2, 2, 2, 2), (16, 16), F32))
  pool = torch.empty(0, 2, 16, 16, device=DEV)
  idle = torch.full((3,), -1, dtype=torch.int32, device=DEV)
  assert not ast.matrix_scan_step(q, k, v, g, pool, slots=idle).any()
  with pytest.raises(ast.ScanError, match="slot"):
    ast.matrix_scan_step(q, k, v, g, pool, slots=idle + 1)
    ast.check_device_error()


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------


@gpu
def test_example_trains_and_decodes(capsys):
  import importlib.util

  from conftest import REPO
  spec = importlib.util.spec_from_file_location("gla_example",
                                                REPO / "examples" / "gated_linear_attention.py")
  example = importlib.util.module_from_spec(spec)
  spec.loader.exec_module(example)
  assert example.main(["--steps", "12", "--dim", "128", "--heads", "2"]) == 0
  assert "step by step" in capsys.readouterr().out


def test_custom_ops_have_fake_kernels():
  from torch._subclasses.fake_tensor import FakeTensorMode
  ops = torch.ops.associative_scan_triton
  with FakeTensorMode():
    q = torch.empty(9, 2, 16, device="cuda")
    v = torch.empty(9, 4, 8, device="cuda", dtype=torch.float32)
    g = torch.empty(9, 4, device="cuda")
    cu = torch.empty(3, dtype=torch.int32, device="cuda")
    out, final = ops.matrix_scan_fwd(q, q, v, g, cu, 1.0, None)
    assert out.shape == (9, 4, 8) and final.shape == (2, 4, 16, 8) and final.dtype == F32
    grads = ops.matrix_scan_bwd(q, q, v, g, cu, 1.0, None, final, out, None)
    assert [x.shape for x in grads[:4]] == [q.shape, q.shape, v.shape, g.shape]
    assert grads[4].numel() == 0
    state = torch.empty(12, 4, 16, 8, device="cuda")
    assert ops.matrix_scan_step(q, q, v, g, state, None, 1.0).shape == (9, 4, 8)
    w, t = torch.empty(16, device="cuda"), torch.empty(5, 8, device="cuda")
    yq, yk = ops.qk_norm_rotate_fwd(q, v[..., :4].new_empty(9, 1, 16), w, w, t, t, cu, None, 1e-6, False)
    assert yq.shape == q.shape and yk.shape == (9, 1, 16)


@gpu
def test_compiled_layer_matches_eager():
  # forward, gradients and a step traced in one piece
  lengths, h, d = [70, 0, 131], 2, 32
  gen = torch.Generator().manual_seed(11)
  packed = torch.randn(201, 3 * h * d, generator=gen).to(DEV).requires_grad_(True)
  gates = (-0.1 * torch.rand(201, h, generator=gen)).to(DEV).requires_grad_(True)
  weight = torch.ones(d, device=DEV, requires_grad=True)
  angle = torch.rand(140, d // 2, generator=gen).to(DEV)
  cos, sin, args = angle.cos(), angle.sin(), {"cu_seqlens": cu_of(lengths)}

  def layer(packed, gates, weight, scan, rotate):
    q, k, v = packed.view(-1, 3, h, d).unbind(1)
    q, k = rotate(q, k, weight, weight, cos, sin, args)
    out, final = scan(q, k, v, gates, args, return_final_state=True)
    return (out * 2.0).sum(-1), final

  def compiled(packed, gates, weight):
    return layer(packed, gates, weight, ast.matrix_scan_causal_compiled, ast.qk_norm_rotate_compiled)

  found = []
  for run in (lambda: layer(packed, gates, weight, ast.matrix_scan_causal, ast.qk_norm_rotate),
              lambda: torch.compile(compiled, fullgraph=True, backend="aot_eager")(packed, gates, weight)):
    out, final = run()
    found.append((out, final, *torch.autograd.grad((out.square().sum() + final.sum()), (packed, gates, weight))))
  for a, b in zip(*found):
    assert torch.equal(a, b)

  q, k, v = (torch.randn(3, h, d, generator=gen).to(DEV) for _ in range(3))
  g = torch.zeros(3, h, device=DEV)
  pools = [torch.ones(4, h, d, d, device=DEV) for _ in range(2)]
  slots = torch.tensor([2, -1, 0], dtype=torch.int32, device=DEV)
  step = torch.compile(ast.matrix_scan_step_compiled, fullgraph=True, backend="aot_eager")
  a = ast.matrix_scan_step(q, k, v, g, pools[0], slots=slots)
  b = step(q, k, v, g, pools[1], slots)
  assert torch.equal(a, b) and torch.equal(*pools)


@gpu
def test_forward_mode_derivatives_are_refused():
  # a dual tensor's tangent is not dropped without a word
  import torch.autograd.forward_ad as forward_ad
  q, k, v, g, s0, _, _ = (x if x is None else x.to(DEV) for x in make([9], (2, 2, 2, 2), (16, 16), F32, carry=True))
  args = {"cu_seqlens": cu_of([9])}
  want = ast.matrix_scan_causal(q, k, v, g, args, initial_state=s0)
  stepped = ast.matrix_scan_step(q[:1], k[:1], v[:1], g[:1], s0.clone())
  with forward_ad.dual_level():
    for i in range(5):
      x = [q, k, v, g, s0]
      x[i] = forward_ad.make_dual(x[i], torch.ones_like(x[i]))
      with pytest.raises(NotImplementedError):
        ast.matrix_scan_causal(*x[:4], args, initial_state=x[4])
      with torch.no_grad(), pytest.raises(NotImplementedError):
        ast.matrix_scan_causal(*x[:4], args, initial_state=x[4])
      with pytest.raises(NotImplementedError):
        ast.matrix_scan_causal_compiled(*x[:4], args, initial_state=x[4])
      with pytest.raises(ValueError, match="no derivatives"):
        ast.matrix_scan_step(*(forward_ad.make_dual(y[:1], torch.ones_like(y[:1])) if j == i else y[:1]
                               for j, y in enumerate((q, k, v, g, s0))))
    # tensors without a tangent are taken as ever
    assert torch.equal(ast.matrix_scan_causal(q, k, v, g, args, initial_state=s0), want)
    assert torch.equal(ast.matrix_scan_step(q[:1], k[:1], v[:1], g[:1], s0.clone()), stepped)


@gpu
@pytest.mark.parametrize("dtype,gate_dtype", [(F32, F32), (F16, F32), (F16, F16), (BF16, F32), (BF16, BF16)], ids=str)
@pytest.mark.parametrize("lengths", [[2500], [77, 2300, 123]], ids=str)
def test_gradients_across_stored_states(lengths, dtype, gate_dtype):
  # 50 heads fill the SMs with one or two segments of the packed axis, so a
  # piece of a sequence is longer than the stretch (128 to 1024 tokens) over
  # which a gate's gradient is summed, and states are stored inside it
  tensors = make(lengths, (50,) * 4, (16, 16), dtype, seed=12, gate_dtype=gate_dtype, carry=True, rate=0.02)
  check_gradients(tensors, lengths, dtype, gate_dtype=gate_dtype)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradients_of_shared_heads_across_stored_states(dtype):
  lengths = [40, 1500]
  tensors = make(lengths, (10, 5, 50, 50), (16, 24), dtype, seed=13, carry=True, rate=0.05)
  check_gradients(tensors, lengths, dtype)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_step_rotation_and_gradients_in_a_graph(dtype):
  lengths = [130, 60]
  q, k, v, g, s0, d_out, d_final = (x.to(DEV) for x in make(lengths, (2, 1, 2, 2), (64, 64), dtype, carry=True))
  args = {"cu_seqlens": cu_of(lengths)}
  angle = torch.rand(130, 32, generator=torch.Generator().manual_seed(1)).to(DEV)
  cos, sin, weight = angle.cos(), angle.sin(), torch.ones(64, device=DEV, dtype=dtype)
  pool, other = torch.randn(5, 2, 64, 64, device=DEV), torch.zeros(5, 2, 64, 64, device=DEV)
  slots = torch.tensor([3, -1, 0], dtype=torch.int32, device=DEV)

  def call():
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v, g, s0, weight)]
    yq, yk = ast.qk_norm_rotate(leaves[0], leaves[1], leaves[5], leaves[5], cos, sin, args)
    out, final = ast.matrix_scan_causal(yq, yk, *leaves[2:4], args, initial_state=leaves[4], return_final_state=True)
    grads = torch.autograd.grad([out, final], leaves, [d_out, d_final])
    new = ast.matrix_scan_step(q[:3], k[:3], v[:3], g[:3], pool, slots=slots, state_out=other)
    return [out, final, new, other, *grads]

  first = [x.detach().clone() for x in call()]
  sync_check = _lib.sync_check_enabled()
  _lib.set_sync_check(False)  # a synchronisation is not allowed while capturing
  try:
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
      call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      captured = call()
    for x in captured:
      x.detach().zero_()
    graph.replay()
    torch.cuda.synchronize()
  finally:
    _lib.set_sync_check(sync_check)
  for a, b in zip(first, captured):
    assert torch.equal(a, b)
