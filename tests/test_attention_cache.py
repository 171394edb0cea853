"""The 8-bit cache of keys and values, and the attention of single tokens over it.

What a write leaves is known exactly: scales are powers of two, so a value is
rounded once, and the oracle's e4m3 (float64 arithmetic) has to agree bit for
bit.  The attention reads the same bytes as its oracle: float32 results within
1e-5 (float32 sums; operands keep 22 bits), 16-bit ones within one rounding,
2^-8 and 2^-11, which weights of 11 bits hardly add to; single elements 16
times that, as they may cancel.
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import associative_scan_triton as ast
from associative_scan_triton import _lib
from test_attention import BF16, DEV, F16, F32, TOL, TYPES, close, cu_of, oracle

gpu = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def ints(x, dtype=torch.int32):
  return torch.tensor(x, dtype=dtype, device=DEV)


def round_e4m3(y):
  """To the nearest e4m3, ties to even, in float64."""
  _, e = torch.frexp(y)
  step = torch.ldexp(torch.ones_like(y), (e - 1).clamp(min=-6) - 3)
  return torch.round(y / step) * step


def scale_for(top: float) -> float:
  if top == 0:
    return 2.0**-64
  m, e = math.frexp(top)  # 448 = 0.875 * 2^9
  return 2.0**max(-64, min(64, e - 8 if m > 0.875 else e - 9))


class Model:
  """A cache in float64 on the CPU."""

  def __init__(self, cache):
    self.x = [t.double().cpu() for t in cache[:2]]  # elements, not values
    self.s = [t.double().cpu() for t in cache[2:]]

  def write(self, keys, values, pages, starts, lengths):
    page, at = self.x[0].shape[2], 0
    for b, n in enumerate(lengths):
      for pos in range(starts[b], starts[b] + n):
        i, r = int(pages[b][pos // page]), pos % page
        # what this call writes to the page, from its first row on
        first = max(starts[b], pos // page * page)
        if pos != first:
          continue
        m = min(starts[b] + n, (pos // page + 1) * page) - pos
        for x, s, new in zip(self.x, self.s, (keys, values)):
          rows = new[at + pos - starts[b]:at + pos - starts[b] + m].double().transpose(0, 1)
          for h in range(x.shape[1]):
            y = rows[h]
            fits = y[torch.isfinite(y)].abs()
            need = scale_for(float(fits.max()) if fits.numel() else 0.0)
            if r:
              need = max(need, float(s[i, h]))
              x[i, h, :r] = round_e4m3(x[i, h, :r] * (float(s[i, h]) / need))
            z = round_e4m3(torch.nan_to_num(y, 0.0, 0.0, 0.0) / need).clamp(-448, 448)
            x[i, h, r:r + m] = torch.where(torch.isfinite(y), z, torch.full_like(z, float("nan")))
            s[i, h] = need
      at += n

  def check(self, cache):
    for want, got in zip(self.x + self.s, cache):
      got = got.double().cpu()
      assert torch.equal(torch.isnan(got), torch.isnan(want))
      assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))

  def values(self, which):
    return self.x[which] * self.s[which][..., None, None]


def filled(pages, heads, page, dk, dv, seed=0):
  """A cache of random pages."""
  gen = torch.Generator().manual_seed(seed)
  x = [torch.randn(pages, heads, page, d, generator=gen) * (0.2 + 3 * torch.rand(pages, heads, 1, 1, generator=gen))
       for d in (dk, dv)]
  s = [torch.tensor([[scale_for(float(t[i, h].abs().max())) for h in range(heads)] for i in range(pages)]) for t in x]
  e = [(t / f[..., None, None]).to(E4M3) for t, f in zip(x, s)]
  return ast.AttentionCache(*(t.to(DEV) for t in e), *(t.float().to(DEV) for t in s))


def tokens(n, heads, dk, dv, dtype, seed=1, size=1.0):
  gen = torch.Generator().manual_seed(seed)
  return ((size * torch.randn(n, heads, dk, generator=gen)).to(dtype),
          (size * torch.randn(n, heads, dv, generator=gen)).to(dtype))


def table(pool, counts, seed=2):
  """A row of pages for each request, in random order; -1 behind its last."""
  order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).tolist()
  rows = [[order.pop() for _ in range(c)] for c in counts]
  width = max(counts)
  return [r + [-1] * (width - len(r)) for r in rows]


def check_write(lengths, starts, page, dims, dtype, heads=2, size=1.0, start_dtype=torch.int32):
  counts = [max(1, -(-(s + n) // page)) for s, n in zip(starts, lengths)]
  cache = filled(sum(counts) + 2, heads, page, *dims)
  model = Model(cache)
  pages = table(sum(counts) + 2, counts)
  k, v = tokens(sum(lengths), heads, *dims, dtype, size=size)
  ast.attention_cache_write(k.to(DEV), v.to(DEV), cache, ints(pages), ints(starts, start_dtype),
                            {"cu_seqlens": cu_of(lengths)})
  model.write(k, v, pages, starts, lengths)
  model.check(cache)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [16, 48, 64, 128])
def test_write_prompts_and_continuations(page, dtype):
  check_write([1, 0, 130, 64, 17, 33], [0, 5, 0, 64, 200, 15], page, (64, 64), dtype)


@gpu
@pytest.mark.parametrize("size", [1.0, 300.0, 1e-3])
@pytest.mark.parametrize("dtype", TYPES)
def test_write_one_token_each(dtype, size):
  # larger tokens move what their pages hold to a larger scale
  check_write([1] * 37, [3 * i for i in range(37)], 16, (128, 64), dtype, size=size, start_dtype=torch.int64)


@gpu
@pytest.mark.parametrize("dims", [(16, 16), (80, 48), (96, 128), (112, 32)], ids=str)
def test_write_head_sizes(dims):
  check_write([40, 3], [7, 0], 32, dims, BF16, heads=3)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_write_extremes(dtype):
  # powers of two, ties, the format's smallest steps, zeros, and what is not finite
  page, n = 16, 12
  cache = ast.attention_cache(3, 1, page, 16, device=DEV)
  model = Model(cache)
  k, v = tokens(n, 1, 16, 16, dtype)
  k[0, 0] = torch.tensor([448, -448, 0, 2.0**-9, 2.0**-10, 3 * 2.0**-11, 17, 19, 1.0625, 1.1875, 0.0625, 240, 232, -1,
                          2.0**-6, 2.0**-7]).to(dtype)
  k[5, 0, 3], k[6, 0, 2], k[7, 0, 1] = float("nan"), float("inf"), float("-inf")
  v.zero_()
  pages = [[2]]
  ast.attention_cache_write(k.to(DEV), v.to(DEV), cache, ints(pages), ints([0]), {"cu_seqlens": cu_of([n])})
  model.write(k, v, pages, [0], [n])
  model.check(cache)
  assert float(cache.key_scales[2, 0]) == 1.0 and float(cache.value_scales[2, 0]) == 2.0**-64
  if dtype != F16:
    big = torch.full((1, 1, 16), 1e30, dtype=dtype)  # beyond the largest scale: its largest value
    ast.attention_cache_write(big.to(DEV), big.to(DEV), cache, ints(pages), ints([n]), {"cu_seqlens": cu_of([1])})
    assert float(cache.key_scales[2, 0]) == 2.0**64 and (cache.keys[2, 0, n].float() == 448).all()


@gpu
def test_write_leaves_the_rest_alone():
  cache = filled(6, 2, 32, 64, 64)
  before = [t.clone() for t in cache]
  k, v = (t.to(DEV) for t in tokens(7, 2, 64, 64, BF16, size=100.0))
  ast.attention_cache_write(k, v, cache, ints([[4, -1], [1, 3]]), ints([-1, 40]), {"cu_seqlens": cu_of([3, 4])})
  changed = torch.zeros(6, 32, dtype=torch.bool)
  changed[3, :12] = True  # what the request holds of the page, and its new tokens
  for a, b in zip(cache[:2], before[:2]):
    same = (a.view(torch.uint8) == b.view(torch.uint8)).all(-1).all(1).cpu()
    assert same[~changed].all() and not same[3, 8:12].any()
  for a, b in zip(cache[2:], before[2:]):
    assert torch.equal(a[:3], b[:3]) and torch.equal(a[4:], b[4:]) and (a[3] > b[3]).all()


@gpu
@pytest.mark.parametrize("pages,start", [([[7]], 0), ([[-1]], 0), ([[2]], 32)], ids=str)
def test_write_outside_the_pool_is_reported(pages, start):
  cache = filled(3, 1, 32, 16, 16)
  before = [t.clone() for t in cache]
  k, v = (t.to(DEV) for t in tokens(2, 1, 16, 16, F32))
  with pytest.raises(ast.ScanError, match="page"):
    ast.attention_cache_write(k, v, cache, ints(pages), ints([start]), {"cu_seqlens": cu_of([2])})
  for a, b in zip(cache, before):
    assert torch.equal(a.float(), b.float())


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------


def step_oracle(q, model, pages, lengths, scale):
  k, v = model.values(0), model.values(1)
  share, out = q.shape[1] // k.shape[1], []
  for b, n in enumerate(lengths):
    if n <= 0:
      out.append(torch.zeros(q.shape[1], v.shape[3], dtype=torch.float64))
      continue
    at = torch.tensor(pages[b][:-(-n // k.shape[2])])
    kb, vb = (x[at].transpose(0, 1).flatten(1, 2)[:, :n].repeat_interleave(share, 0) for x in (k, v))
    p = torch.softmax((q[b].double()[:, None] * kb).sum(-1) * scale, -1)
    out.append((p[..., None] * vb).sum(1))
  return torch.stack(out)


def check_step(lengths, heads, dims, page, dtype, scale=None, spare=2, length_dtype=torch.int32, q_size=1.0):
  h, hk = heads
  counts = [max(1, -(-n // page)) for n in lengths]
  pool = sum(counts) + spare
  cache = filled(pool, hk, page, *dims)
  pages = table(pool, counts)
  q = (q_size * torch.randn(len(lengths), h, dims[0], generator=torch.Generator().manual_seed(4))).to(dtype)
  out = ast.attention_cache_step(q.to(DEV), cache, ints(pages), ints(lengths, length_dtype), scale=scale)
  assert out.dtype == dtype
  want = step_oracle(q, Model(cache), pages, lengths, dims[0]**-0.5 if scale is None else scale)
  close("out", out, want, TOL[dtype])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [16, 48, 64, 128])
def test_step_lengths(page, dtype):
  check_step([1, 15, 16, 17, 0, 63, 64, 65, 200, -3, 129, 1000], (4, 2), (64, 64), page, dtype,
             length_dtype=torch.int64)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dims", [(128, 128), (128, 64), (64, 128), (96, 96), (80, 48), (16, 16), (112, 80)], ids=str)
def test_step_head_sizes(dims, dtype):
  check_step([300, 77], (3, 3), dims, 32, dtype)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads", [(1, 1), (16, 1), (24, 1), (40, 2), (12, 3), (5, 5)], ids=str)
def test_step_shared_heads(heads, dtype):
  check_step([130, 400], heads, (128, 128), 64, dtype)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_step_long_context(dtype):
  check_step([30000], (4, 1), (128, 128), 64, dtype)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_step_many_requests(dtype):
  check_step([1 + 37 * i % 300 for i in range(300)], (2, 1), (64, 64), 16, dtype)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("q_size", [1e-4, 30.0])
def test_step_sizes_of_queries(q_size, dtype):
  check_step([500, 40], (4, 2), (64, 64), 32, dtype, q_size=q_size)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_step_pages_of_very_different_scales(dtype):
  page, n = 16, 16 * 12
  cache = filled(12, 1, page, 64, 64)
  spread = torch.tensor([2.0**(7 * (i % 5) - 20) for i in range(12)], device=DEV)[:, None]
  cache.value_scales.mul_(spread)
  cache.key_scales.mul_(spread.sqrt().log2().round().exp2() * 2.0**3)
  q = torch.randn(1, 2, 64, generator=torch.Generator().manual_seed(4)).to(dtype)
  pages = [list(range(12))]
  out = ast.attention_cache_step(q.to(DEV), cache, ints(pages), ints([n]))
  close("out", out, step_oracle(q, Model(cache), pages, [n], 0.125), TOL[dtype])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_step_does_not_read_what_lies_behind_the_last_token(dtype):
  # rows behind it, and pages of no request, hold NaN; requests share pages
  cache = filled(5, 1, 64, 64, 64)
  bytes_ = [t.view(torch.uint8) for t in cache[:2]]
  for t in bytes_:
    t[3, :, 21:] = 0x7F
    t[4] = 0x7F
  pages, lengths = [[1, 3], [1, 2], [3, 0]], [64 + 21, 100, 21]
  q = torch.randn(3, 2, 64, generator=torch.Generator().manual_seed(4)).to(dtype)
  out = ast.attention_cache_step(q.to(DEV), cache, ints(pages), ints(lengths))
  close("out", out, step_oracle(q, Model(cache), pages, lengths, 0.125), TOL[dtype])


@gpu
def test_step_values_that_are_not_finite():
  cache = filled(2, 2, 32, 32, 32)
  cache.values.view(torch.uint8)[0, 1, 3, 7] = 0x7F
  q = torch.randn(1, 2, 32, device=DEV)
  out = ast.attention_cache_step(q, cache, ints([[0, 1]]), ints([50]))
  nan = torch.isnan(out[0])
  assert nan[1, 7] and int(nan.sum()) == 1


@gpu
@pytest.mark.parametrize("pages,length", [([[5]], 10), ([[-2]], 10), ([[1]], 33)], ids=str)
def test_step_outside_the_pool_is_reported(pages, length):
  cache = filled(3, 1, 32, 16, 16)
  with pytest.raises(ast.ScanError, match="page"):
    ast.attention_cache_step(torch.randn(1, 2, 16, device=DEV), cache, ints(pages), ints([length]))


@gpu
def test_step_pool_beyond_32_bit_offsets():
  page, pages = 4096, 4200  # 2.2 GB of keys
  cache = ast.attention_cache(pages, 1, page, 128, 16, device=DEV)
  k, v = tokens(5, 1, 128, 16, BF16)
  last = ints([[pages - 1]])
  ast.attention_cache_write(k.to(DEV), v.to(DEV), cache, last, ints([0]), {"cu_seqlens": cu_of([5])})
  q = torch.randn(1, 1, 128, generator=torch.Generator().manual_seed(4)).to(BF16)
  out = ast.attention_cache_step(q.to(DEV), cache, last, ints([5]))
  small = Model([t[-1:] for t in cache])
  close("out", out, step_oracle(q, small, [[0]], [5], 128**-0.5), TOL[BF16])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_a_conversation(dtype):
  """A prompt through the rotation and the attention, its cache written, then
  token by token: as the whole conversation at once over the cached values."""
  h, hk, d, page, n, more = 4, 2, 64, 32, 70, 9
  gen = torch.Generator().manual_seed(8)
  x = [torch.randn(n + more, m, d, generator=gen).to(dtype).to(DEV) for m in (h, hk, hk)]
  w = torch.ones(d, dtype=dtype, device=DEV)
  angle = torch.arange(200, device=DEV)[:, None] * torch.logspace(0, -3, d // 2, device=DEV)
  place = torch.stack((torch.arange(n + more), torch.arange(n + more) // 8, torch.arange(n + more) % 8)).to(DEV)
  rotate = dict(cos=angle.cos(), sin=angle.sin(), sections=(8, 12, 12))
  cache = ast.attention_cache(8, hk, page, d, device=DEV)
  pages = ints([[6, 1, 4]])
  q, k = ast.qk_norm_rotate(x[0][:n], x[1][:n], w, w, positions=place[:, :n].contiguous(), **rotate)
  prompt = ast.attention_causal(q, k, x[2][:n], {"cu_seqlens": ints([0, n])})
  ast.attention_cache_write(k, x[2][:n], cache, pages, ints([0]), {"cu_seqlens": ints([0, n])})
  outs, keys, queries = [], [k], [q]
  for t in range(n, n + more):
    q, k = ast.qk_norm_rotate(x[0][t:t + 1], x[1][t:t + 1], w, w, positions=place[:, t:t + 1].contiguous(), **rotate)
    ast.attention_cache_write(k, x[2][t:t + 1], cache, pages, ints([t]), {"cu_seqlens": ints([0, 1])})
    outs.append(ast.attention_cache_step(q, cache, pages, ints([t + 1])))
    keys.append(k)
    queries.append(q)
  q, k = torch.cat(queries).cpu().double(), torch.cat(keys).cpu().double()
  whole = oracle(q, k, x[2].cpu().double(), [n + more], 0.125)
  close("prompt", prompt, whole[:n], TOL[dtype])
  close("step", outs[-1], step_oracle(queries[-1].cpu(), Model(cache), [[6, 1, 4]], [n + more], 0.125), TOL[dtype])
  # against the unrounded keys and values: each is off by at most 2^-4 of
  # itself, 2^-4 / sqrt(3) as a root mean square; a score of norm-1 parts by as
  # much, and the mean of the values by both
  got = torch.cat(outs).cpu().double()
  assert float((got - whole[n:]).norm()) <= 2 * 2.0**-4 / 3**0.5 * float(whole[n:].norm())


@gpu
def test_write_and_step_in_a_graph_and_on_another_stream():
  cache = filled(6, 2, 32, 64, 64)
  k, v = (t.to(DEV) for t in tokens(2, 2, 64, 64, BF16))
  q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(4)).to(BF16).to(DEV)
  pages, starts, lengths, args = ints([[0, 3], [5, 1]]), ints([40, 7]), ints([41, 8]), {"cu_seqlens": cu_of([1, 1])}
  twin = ast.AttentionCache(*(t.clone() for t in cache))

  def step(c):
    ast.attention_cache_write(k, v, c, pages, starts, args)
    return ast.attention_cache_step(q, c, pages, lengths)

  want = step(twin)
  s = torch.cuda.Stream()
  s.wait_stream(torch.cuda.current_stream())
  third = ast.AttentionCache(*(t.clone() for t in cache))
  s.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(s):
    other = step(third)
  s.synchronize()
  assert torch.equal(other, want)
  graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
  ast.set_sync_check(False)
  try:
    with torch.cuda.graph(graph):
      out = step(cache)
    with torch.cuda.graph(graph2, pool=graph.pool()):  # its workspace may be the first one's
      out2 = ast.attention_cache_step(q, cache, pages, lengths)
  finally:
    ast.set_sync_check(True)
  for _ in range(2):
    graph.replay()
    graph2.replay()
  torch.cuda.synchronize()
  assert torch.equal(out2, want)
  graph.replay()
  torch.cuda.synchronize()
  assert torch.equal(out, want)
  for a, b in zip(cache, twin):
    assert torch.equal(a.float(), b.float())


@gpu
def test_write_counts_as_a_change():
  cache = filled(2, 1, 32, 16, 16)
  k, v = (t.to(DEV) for t in tokens(1, 1, 16, 16, F32))
  before = [t._version for t in cache]
  ast.attention_cache_write(k, v, cache, ints([[0]]), ints([3]), {"cu_seqlens": cu_of([1])})
  assert all(t._version > b for t, b in zip(cache, before))


@gpu
def test_empty_calls():
  cache = filled(2, 1, 32, 16, 16)
  none = torch.empty(0, 1, 16, device=DEV)
  ast.attention_cache_write(none, none, cache, torch.empty(0, 2, dtype=torch.int32, device=DEV), ints([]),
                            {"cu_seqlens": cu_of([])})
  ast.attention_cache_write(none, none, cache, ints([[0]]), ints([0]), {"cu_seqlens": cu_of([0])})
  assert ast.attention_cache_step(none, cache, torch.empty(0, 2, dtype=torch.int32, device=DEV), ints([])).shape == (0, 1, 16)
  empty = ast.attention_cache(0, 1, 32, 16, device=DEV)
  out = ast.attention_cache_step(torch.randn(2, 1, 16, device=DEV), empty, torch.empty(2, 0, dtype=torch.int32, device=DEV),
                                 ints([0, 0]))
  assert (out == 0).all()


@gpu
def test_compiled_matches_eager():
  cache = filled(4, 1, 32, 32, 32)
  twin = ast.AttentionCache(*(t.clone() for t in cache))
  k, v = (t.to(DEV) for t in tokens(2, 1, 32, 32, BF16))
  q = torch.randn(2, 2, 32, device=DEV).to(BF16)
  pages, starts, lengths = ints([[0], [3]]), ints([4, 0]), ints([5, 1])
  args = {"cu_seqlens": cu_of([1, 1])}
  ast.attention_cache_write(k, v, cache, pages, starts, args)
  want = ast.attention_cache_step(q, cache, pages, lengths)

  @torch.compile(fullgraph=True)
  def step(q, k, v, cache, pages, starts, lengths, cu):
    ast.attention_cache_write_compiled(k, v, cache, pages, starts, {"cu_seqlens": cu})
    return ast.attention_cache_step_compiled(q, cache, pages, lengths)

  out = step(q, k, v, tuple(twin), pages, starts, lengths, args["cu_seqlens"])
  assert torch.equal(out, want)
  for a, b in zip(cache, twin):
    assert torch.equal(a.float(), b.float())


def test_refusals():
  with FakeTensorMode():
    cache = ast.attention_cache(4, 2, 32, 64, 48, device=DEV)
    k, v = torch.empty(3, 2, 64, device=DEV), torch.empty(3, 2, 48, device=DEV)
    q = torch.empty(2, 4, 64, device=DEV)
    pages = torch.empty(2, 3, dtype=torch.int32, device=DEV)
    starts = torch.empty(2, dtype=torch.int32, device=DEV)
    args = {"cu_seqlens": torch.empty(3, dtype=torch.int32, device=DEV)}

    def write(error, match, k=k, v=v, cache=cache, pages=pages, starts=starts, args=args):
      with pytest.raises(error, match=match):
        ast.attention_cache_write(k, v, cache, pages, starts, args)

    def step(error, match, q=q, cache=cache, pages=pages, lengths=starts, **kw):
      with pytest.raises(error, match=match):
        ast.attention_cache_step(q, cache, pages, lengths, **kw)

    write(ValueError, "CUDA tensors only", k=torch.empty(3, 2, 64))
    write(TypeError, "values has dtype", v=v.half())
    write(TypeError, "unsupported dtype", k=k.double())
    write(ValueError, "head size", k=v)
    write(ValueError, "head size", v=k)
    write(ValueError, "rows", v=v[:2])
    write(ValueError, "heads", k=k[:, :1])
    write(ValueError, "heads", v=v[:, :1])
    write(TypeError, "AttentionCache", cache=cache[:3])
    write(TypeError, "float8", cache=cache._replace(keys=cache.keys.view(torch.uint8)))
    write(ValueError, "contiguous", cache=cache._replace(values=cache.values.transpose(1, 2)))
    write(ValueError, "differ", cache=cache._replace(values=cache.values[:3]))
    write(ValueError, "key_scales must be contiguous", cache=cache._replace(key_scales=cache.key_scales[:3]))
    write(TypeError, "value_scales must be float32", cache=cache._replace(value_scales=cache.value_scales.half()))
    write(ValueError, "int32", pages=pages.long())
    write(ValueError, "int32", pages=pages[0])
    write(ValueError, "starts has", starts=starts[:1])
    write(ValueError, "cu_seqlens has", args={"cu_seqlens": args["cu_seqlens"][:2]})
    write(TypeError, "int32 or int64", starts=starts.float())
    write(ValueError, "no backward", k=torch.empty(3, 2, 64, device=DEV, requires_grad=True))
    step(ValueError, "head size", q=q[..., :32])
    step(ValueError, "divide", q=q[:, :3])
    step(ValueError, "pages has 2 rows", q=q[:1])
    step(ValueError, "lengths has", lengths=starts[:1])
    step(ValueError, "scale must be", scale=0.0)
    step(ValueError, "no backward", q=torch.empty(2, 4, 64, device=DEV, requires_grad=True))
    for sizes in ((4, 2, 24, 64), (4, 2, 8192, 64), (4, 2, 32, 40), (4, 2, 32, 144), (4, 0, 32, 64)):
      with pytest.raises(ValueError):
        ast.attention_cache(*sizes, device=DEV)


def test_abi_rejects_bad_arguments_without_a_gpu():
  lib = _lib.load()
  data = torch.zeros(4096)
  at = data.data_ptr() + (-data.data_ptr()) % 256

  def step(pages=2, heads=1, page=16, dk=16, dv=16, q_heads=2, index=0, dtype=0, scale=1.0, ws=1 << 30, batch=1, off=0):
    cache = _lib.Cache(at + off, at, at, at, pages, heads, page, dk, dv)
    return lib.ascan_cache_step(ctypes.byref(_lib.Rows(at, 8, 4, q_heads)), ctypes.byref(cache), at, batch, 1, at, index, dtype, scale,
                                at, at, ws, None)

  for bad in ({"pages": -1}, {"heads": 0}, {"page": 8}, {"page": 8192}, {"dk": 8}, {"dv": 144}, {"q_heads": 0},
              {"heads": 3}, {"index": 2}, {"dtype": 5}, {"scale": -1.0}, {"batch": 65536}, {"off": 4}):
    assert step(**bad) == -1, bad
  assert step(ws=100) == -2
  assert step(batch=0) == 0


def test_custom_ops_have_fake_kernels():
  with FakeTensorMode():
    cache = ast.attention_cache(4, 2, 32, 64, 48, device=DEV)
    pages = torch.empty(2, 3, dtype=torch.int32, device=DEV)
    starts = torch.empty(2, dtype=torch.int32, device=DEV)
    out = ast.attention_cache_step_compiled(torch.empty(2, 4, 64, device=DEV), cache, pages, starts)
    assert out.shape == (2, 4, 48)
    ast.attention_cache_write_compiled(torch.empty(3, 2, 64, device=DEV), torch.empty(3, 2, 48, device=DEV), cache, pages,
                                       starts, {"cu_seqlens": torch.empty(3, dtype=torch.int32, device=DEV)})
