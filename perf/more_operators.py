"""Workloads of the softmax-attention operators: cases, inputs, plain forms and 64-bit results.

Four operators of an attention layer that stands between gated linear-attention
layers, each as a user calls it:

* ``rotate``: norms of queries and keys with a rotation by several axes (time,
  height, width) in the same pass (``qk_norm_rotate`` with ``sections``), alone
  or with its gradients;
* ``attend``: causal softmax attention over packed sequences with grouped heads
  (``attention_causal``), alone or with its gradients;
* ``write``: new keys and values into the pages of an 8-bit cache with a scale
  for each page and head (``attention_cache_write``);
* ``step``: the next token of every running request over that cache
  (``attention_cache_step``).

``run`` with ``own`` false computes the plain form in elementary torch
operations in float32; with ``own`` true it calls the package.
"""

import math
import os
import random
import sys

import torch

own = False

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
PLAIN_ROWS = 1024  # query rows of one block of the plain attention
LARGEST = 448.0  # of e4m3
SCALE_BITS = 64  # a page's scale is a power of two between 2^-64 and 2^64


def _package():
  dist = os.path.join(REPO, "associative-scan-triton_b200")
  if dist not in sys.path:
    sys.path.insert(1, dist)
  import associative_scan_triton

  return associative_scan_triton


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------


def _rotate(name, tokens, heads, key_heads, dim, sections, dtype, train, interleaved=False):
  return {"name": name, "op": "rotate", "tokens": tokens, "heads": heads, "key_heads": key_heads,
          "dim": dim, "sections": ",".join(str(x) for x in sections), "dtype": dtype,
          "train": train, "interleaved": interleaved}


def _attend(name, tokens, seqs, heads, key_heads, dim, value_dim, dtype, train, ragged):
  return {"name": name, "op": "attend", "tokens": tokens, "seqs": seqs, "heads": heads,
          "key_heads": key_heads, "dim": dim, "value_dim": value_dim, "dtype": dtype,
          "train": train, "ragged": ragged}


def _write(name, tokens, seqs, key_heads, dim, value_dim, page, dtype, continues):
  return {"name": name, "op": "write", "tokens": tokens, "seqs": seqs, "key_heads": key_heads,
          "dim": dim, "value_dim": value_dim, "page": page, "dtype": dtype,
          "continues": continues, "ragged": True}


def _step(name, batch, context, heads, key_heads, dim, value_dim, page, dtype):
  return {"name": name, "op": "step", "seqs": batch, "tokens": batch * context, "heads": heads,
          "key_heads": key_heads, "dim": dim, "value_dim": value_dim, "page": page,
          "dtype": dtype, "ragged": True}


def listed():
  return [
    # a prompt of text and video frames, 2048 channels of queries, shared key heads
    _rotate("rotate_axes_prompt", 32768, 16, 4, 128, (16, 24, 24), "bf16", False),
    # training on ragged samples of text and images, odd heads, adjacent pairs
    _rotate("rotate_axes_train", 4999, 16, 4, 80, (8, 16, 16), "f16", True, interleaved=True),
    # a short prompt; latency counts
    _attend("attend_prompt_short", 131, 1, 12, 12, 128, 128, "bf16", False, False),
    # prompts of many requests packed, keys and values shared by four heads each
    _attend("attend_prompt_packed", 16384, 16, 16, 4, 128, 128, "bf16", False, True),
    # one long document
    _attend("attend_prompt_long", 32768, 1, 16, 4, 128, 128, "bf16", False, False),
    # a training step's 8 sequences of 2048 tokens, 1536 channels
    _attend("attend_train", 8 * 2048, 8, 12, 12, 128, 128, "bf16", True, False),
    # float32 training on ragged sequences, small heads
    _attend("attend_train_f32", 3001, 5, 12, 12, 64, 64, "f32", True, True),
    # prompts' keys and values into fresh pages
    _write("write_prompt", 16384, 8, 4, 128, 128, 64, "bf16", False),
    # the new token of every request of a full batch, into pages already begun
    _write("write_batch", 256, 256, 4, 128, 128, 64, "bf16", True),
    # a single request's next token after a short conversation
    _step("step_single", 1, 500, 12, 12, 128, 128, 64, "bf16"),
    # a single request's next token after a long document
    _step("step_long", 1, 131072, 16, 4, 128, 128, 64, "bf16"),
    # the next token of a full batch of requests of different lengths
    _step("step_batch", 128, 4000, 16, 4, 128, 128, 64, "bf16"),
  ]


def _log_int(rng, low, high):
  n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
  return min(max(n, low), high)


def draw(rng):
  op = rng.choice(("rotate", "attend", "attend", "attend", "write", "step", "step"))
  dtype = rng.choice(("bf16", "bf16", "bf16", "f16", "f32"))
  heads, key_heads = rng.choice(((12, 12), (16, 4), (16, 16), (8, 1), (12, 3), (5, 5), (24, 1)))
  if op == "rotate":
    train = rng.random() < 0.5
    dim, sections = rng.choice(((128, (16, 24, 24)), (64, (8, 12, 12)), (80, (8, 16, 16)),
                                (96, (24, 24)), (128, (8, 8, 8, 8)), (72, (11, 13, 12))))
    case = _rotate("", _log_int(rng, 1, 32768), heads, key_heads, dim, sections, dtype, train,
                   rng.random() < 0.4)
  elif op == "attend":
    train = rng.random() < 0.5
    dim, value_dim = rng.choice(((64, 64), (128, 128), (128, 128), (96, 96), (128, 64), (40, 72),
                                 (80, 80)))
    largest = 4096 if dtype == "f32" else (8192 if train else 20000)
    tokens = _log_int(rng, 1, largest)
    case = _attend("", tokens, rng.randint(1, min(tokens, 16)), heads, key_heads, dim, value_dim,
                   dtype, train, rng.random() < 0.7)
  elif op == "write":
    dim, value_dim = rng.choice(((64, 64), (128, 128), (96, 96), (128, 64), (80, 48)))
    page, continues = rng.choice((16, 32, 64, 128)), rng.random() < 0.6
    tokens = _log_int(rng, 1, 16384)
    case = _write("", tokens, _log_int(rng, 1, min(tokens, 256)), key_heads, dim, value_dim, page,
                  dtype, continues)
  else:
    dim, value_dim = rng.choice(((64, 64), (128, 128), (128, 128), (96, 96), (128, 64), (80, 48)))
    batch = _log_int(rng, 1, 128)
    case = _step("", batch, _log_int(rng, 1, 400000 // batch), heads, key_heads, dim, value_dim,
                 rng.choice((16, 32, 64, 128)), dtype)
  del case["name"]
  return case


def _lengths(case):
  """The sequences' lengths: equal, or spread between a quarter and 1.75 of the mean."""
  n, tokens = case["seqs"], case["tokens"]
  if not case["ragged"] or n == 1 or tokens == n:
    return [tokens // n + (1 if i < tokens % n else 0) for i in range(n)]
  rng = random.Random(tokens * 31 + n)
  weights = [rng.uniform(0.25, 1.75) for _ in range(n)]
  ends = [int(round((tokens - n) * sum(weights[:i + 1]) / sum(weights))) for i in range(n)]
  return [b - a + 1 for a, b in zip([0] + ends[:-1], ends)]


def _starts(case):
  """Tokens that the cache holds of each request before a write."""
  if not case["continues"]:
    return [0] * case["seqs"]
  rng = random.Random(case["tokens"] * 17 + case["seqs"])
  return [rng.randint(0, 4 * case["page"]) for _ in range(case["seqs"])]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _ints(values, device):
  return torch.tensor(values, dtype=torch.int32, device=device)


def _ends(lengths):
  ends = [0]
  for m in lengths:
    ends.append(ends[-1] + m)
  return ends


def _table(rows, half, device):
  freq = torch.exp(torch.arange(half, device=device, dtype=torch.float64)
                   * (-math.log(10000.0) / max(1, half)))
  angle = torch.arange(rows, device=device, dtype=torch.float64)[:, None] * freq
  return angle.cos().float(), angle.sin().float()


def _places(tokens, axes, device):
  """Positions of text runs of 64 tokens, each followed by an image of 24 x 24."""
  at = torch.arange(tokens, device=device)
  r, base = at % 640, at // 640 * 88
  text, cell = r < 64, r - 64
  place = [torch.where(text, base + r, base + 64 + d)
           for d in (torch.zeros_like(cell), cell // 24, cell % 24, cell % 7)]
  return torch.stack(place[:axes]), (tokens // 640 + 1) * 88 + 64


def _pack(x, scale):
  """Elements in units of their page's scale, rounded to e4m3."""
  return (x / scale).to(torch.float8_e4m3fn)


def _scale_for(largest):
  """The smallest power of two that brings `largest` to at most 448."""
  m, e = torch.frexp(largest.float())  # largest = m 2^e, m in [0.5, 1); 448 = 0.875 2^9
  e = torch.where(m > 0.875, e - 8, e - 9)
  e = torch.where(largest > 0, e, torch.full_like(e, -SCALE_BITS)).clamp(-SCALE_BITS, SCALE_BITS)
  return torch.ldexp(torch.ones_like(m), e)


def _pool(pages, heads, page, dim, gen, device):
  """Pages of a cache that holds keys or values of different sizes per head and channel."""
  x = torch.randn(pages, heads, page, dim, generator=gen, device=device)
  x *= 0.25 + 2.0 * torch.rand(heads, 1, dim, generator=gen, device=device)
  scale = _scale_for(x.abs().amax((-1, -2)))
  return _pack(x, scale[..., None, None]), scale


def prepare(case, seed):
  device = torch.device("cuda")
  gen = torch.Generator(device=device).manual_seed(seed)
  dtype = TYPES[case["dtype"]]

  def normal(*shape):
    return torch.randn(shape, generator=gen, device=device)

  s = {"case": case}
  dim, key_heads, tokens = case["dim"], case["key_heads"], case["tokens"]
  if case["op"] == "rotate":
    heads = case["heads"]
    # queries and keys are views of one projection's output, as a layer has them
    both = normal(tokens, heads + key_heads, dim) * (0.5 + 1.5 * torch.rand(
      (heads + key_heads, 1), generator=gen, device=device))
    both = both.to(dtype)
    s["queries"], s["keys"] = both[:, :heads], both[:, heads:]
    s["query_weight"] = (1.0 + 0.2 * normal(dim)).to(dtype)
    s["key_weight"] = (1.0 + 0.2 * normal(dim)).to(dtype)
    s["sections"] = tuple(int(x) for x in case["sections"].split(","))
    s["positions"], rows = _places(tokens, len(s["sections"]), device)
    s["cos"], s["sin"] = _table(rows, sum(s["sections"]), device)
    if case["train"]:
      s["d_queries"] = normal(tokens, heads, dim).to(dtype)
      s["d_keys"] = normal(tokens, key_heads, dim).to(dtype)
    wrt = ("queries", "keys", "query_weight", "key_weight")
  elif case["op"] == "attend":
    heads = case["heads"]
    # scores of a few units and a direction that all keys share, as trained heads have them
    both = normal(tokens, heads + key_heads, dim)
    both[:, heads:] += 0.5 * normal(key_heads, dim)
    both = both.to(dtype)
    s["queries"], s["keys"] = both[:, :heads], both[:, heads:]
    s["values"] = normal(tokens, key_heads, case["value_dim"]).to(dtype)
    s["lengths"] = _lengths(case)
    s["cu_seqlens"] = _ints(_ends(s["lengths"]), device)
    if case["train"]:
      s["d_out"] = normal(tokens, heads, case["value_dim"]).to(dtype)
    wrt = ("queries", "keys", "values")
  else:
    page, value_dim, lengths = case["page"], case["value_dim"], _lengths(case)
    if case["op"] == "write":
      starts = _starts(case)
      # the pages that the write touches; earlier ones are not in this pool (-1)
      first = [a // page for a in starts]
      held = [[-1] * f for f in first]
      ends = [-(-(a + m) // page) for a, m in zip(starts, lengths)]
      s["keys"] = (normal(tokens, key_heads, dim)
                   * (0.25 + 2.0 * torch.rand(key_heads, dim, generator=gen, device=device))).to(dtype)
      s["values"] = normal(tokens, key_heads, value_dim).to(dtype)
      s["cu_seqlens"], s["starts"] = _ints(_ends(lengths), device), _ints(starts, device)
    else:
      first, held = [0] * len(lengths), [[] for _ in lengths]
      ends = [-(-m // page) for m in lengths]
      s["queries"] = normal(len(lengths), case["heads"], dim).to(dtype)
      s["lengths"] = _ints(lengths, device)
    pool = sum(e - f for e, f in zip(ends, first)) + 2
    order = torch.randperm(pool, generator=gen, device=device).tolist()
    for f, e, row in zip(first, ends, held):
      row += [order.pop() for _ in range(e - f)]
    width = max(ends)
    s["pages"] = _ints([row + [-1] * (width - len(row)) for row in held], device)
    s["cache"] = [None] * 4  # keys, values, their scales
    s["cache"][0], s["cache"][2] = _pool(pool, key_heads, page, dim, gen, device)
    s["cache"][1], s["cache"][3] = _pool(pool, key_heads, page, value_dim, gen, device)
    wrt = ()
  if case.get("train"):
    s["wrt"] = wrt
    for w in wrt:
      s[w] = s[w].detach().requires_grad_(True)
  return s


# ---------------------------------------------------------------------------
# plain forms: float32, elementary operations
# ---------------------------------------------------------------------------


def _plain_rotate(s):
  case, half = s["case"], sum(s["sections"])
  axis = torch.repeat_interleave(torch.arange(len(s["sections"]), device="cuda"),
                                 torch.tensor(s["sections"], device="cuda"), output_size=half)
  rows = s["positions"][axis].t()  # [tokens, half]: each pair's table row
  pair = torch.arange(half, device="cuda")
  cos, sin = s["cos"][rows, pair][:, None, :], s["sin"][rows, pair][:, None, :]

  def one(x, w):
    y = x.float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w.float()
    if case["interleaved"]:
      a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
      turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
      a, b = y[..., :half], y[..., half:2 * half]
      turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, y[..., 2 * half:]), -1).to(x.dtype)

  return one(s["queries"], s["query_weight"]), one(s["keys"], s["key_weight"])


def _plain_attend(s):
  case, parts, at = s["case"], [], 0
  share, scale = case["heads"] // case["key_heads"], case["dim"] ** -0.5
  for m in s["lengths"]:
    rows = slice(at, at + m)
    q = s["queries"][rows].float().transpose(0, 1) * scale  # [heads, m, dim]
    q = q.reshape(case["key_heads"], share, m, -1)
    k = s["keys"][rows].float().permute(1, 2, 0)[:, None]
    v = s["values"][rows].float().transpose(0, 1)[:, None]
    for i in range(0, m, PLAIN_ROWS):
      e = min(i + PLAIN_ROWS, m)
      score = q[:, :, i:e] @ k[..., :e]
      late = torch.arange(e, device="cuda") > torch.arange(i, e, device="cuda")[:, None]
      score = score.masked_fill(late, -math.inf)
      p = torch.exp(score - score.amax(-1, keepdim=True))
      o = (p @ v[:, :, :e]) / p.sum(-1, keepdim=True)
      parts.append(o.flatten(0, 1).transpose(0, 1).to(s["values"].dtype))
    at += m
  return torch.cat(parts)


def _plain_write(s):
  """Pages as rows: scale from what each holds already and what it gets, then both rounded."""
  case, page = s["case"], s["case"]["page"]
  cu, starts = s["cu_seqlens"].long(), s["starts"].long()
  at = torch.arange(case["tokens"], device=cu.device)
  seq = torch.searchsorted(cu, at, right=True) - 1
  place = at - cu[seq] + starts[seq]
  target = s["pages"].long()[seq, place // page]
  # what the request wrote to the page before keeps its place and grows with the scale
  opened = (place % page != 0) & (at == cu[seq])
  for x, held, scales in ((s["keys"], s["cache"][0], s["cache"][2]),
                          (s["values"], s["cache"][1], s["cache"][3])):
    x = x.float()
    largest = torch.zeros_like(scales).index_reduce_(0, target, x.abs().amax(-1), "amax")
    need = _scale_for(largest)
    begun = torch.zeros(scales.shape[0], device=x.device).index_add_(
      0, target, torch.where(opened, place % page, 0).float())
    need = torch.where((begun > 0)[:, None], torch.maximum(need, scales), need)
    touched = torch.zeros(scales.shape[0], dtype=torch.bool, device=x.device)
    touched[target] = True
    need = torch.where(touched[:, None], need, scales)
    old = torch.arange(page, device=x.device) < begun[:, None]
    again = held.float() * (scales / need)[..., None, None]
    pool = torch.where(old[:, None, :, None], again, held.float()).to(torch.float8_e4m3fn)
    pool.view(torch.uint8)[target, :, place % page] = _pack(x, need[target][..., None]).view(torch.uint8)
    held.copy_(pool)
    scales.copy_(need)


def _plain_step(s):
  case, page = s["case"], s["case"]["page"]
  share, scale = case["heads"] // case["key_heads"], case["dim"] ** -0.5
  q = s["queries"].float().view(case["seqs"], case["key_heads"], share, case["dim"]) * scale
  width = s["pages"].shape[1]
  lengths, parts = s["lengths"].long(), []
  group = max(1, 65536 // (width * page))  # requests at once, for the memory
  for b in range(0, case["seqs"], group):
    at = s["pages"][b:b + group].long().clamp(min=0)
    n = at.shape[0]
    k, v = (x.view(torch.uint8)[at].view(torch.float8_e4m3fn).float() * f[at][..., None, None]
            for x, f in ((s["cache"][0], s["cache"][2]), (s["cache"][1], s["cache"][3])))
    k = k.transpose(1, 2).reshape(n, case["key_heads"], width * page, -1)
    v = v.transpose(1, 2).reshape(n, case["key_heads"], width * page, -1)
    beyond = torch.arange(width * page, device=k.device) >= lengths[b:b + group, None]
    score = (q[b:b + group] @ k.transpose(-1, -2)).masked_fill(beyond[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    parts.append((p @ v) / p.sum(-1, keepdim=True))
  return torch.cat(parts).flatten(1, 2).to(s["queries"].dtype)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(s):
  case = s["case"]
  if case["op"] == "write":
    if own:
      _package().attention_cache_write(s["keys"], s["values"], tuple(s["cache"]), s["pages"],
                                       s["starts"], {"cu_seqlens": s["cu_seqlens"]})
    else:
      _plain_write(s)
    keys, values, key_scales, value_scales = s["cache"]
    # what the bytes stand for: four digits and a power of two, exact in bfloat16
    return {"keys": keys.bfloat16() * key_scales.bfloat16()[..., None, None],
            "values": values.bfloat16() * value_scales.bfloat16()[..., None, None],
            "key_scales": key_scales, "value_scales": value_scales}
  if case["op"] == "step":
    if own:
      return _package().attention_cache_step(s["queries"], tuple(s["cache"]), s["pages"],
                                             s["lengths"])
    return _plain_step(s)
  if case["op"] == "rotate":
    if own:
      q, k = _package().qk_norm_rotate(s["queries"], s["keys"], s["query_weight"],
                                       s["key_weight"], s["cos"], s["sin"],
                                       positions=s["positions"], eps=1e-6,
                                       interleaved=case["interleaved"], sections=s["sections"])
    else:
      q, k = _plain_rotate(s)
    result = {"queries": q, "keys": k}
    ends, grads = [q, k], [s.get("d_queries"), s.get("d_keys")]
  else:
    if own:
      out = _package().attention_causal(s["queries"], s["keys"], s["values"],
                                        {"cu_seqlens": s["cu_seqlens"]})
    else:
      out = _plain_attend(s)
    result = {"out": out}
    ends, grads = [out], [s.get("d_out")]
  if case["train"]:
    found = torch.autograd.grad(ends, [s[w] for w in s["wrt"]], grads)
    result.update({"grad_" + w: d for w, d in zip(s["wrt"], found)})
  return {name: x.detach() for name, x in result.items()}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
  size, key_heads, dim = SIZE[case["dtype"]], case["key_heads"], case["dim"]
  tokens = case["tokens"]
  if case["op"] == "rotate":
    sections = [int(x) for x in case["sections"].split(",")]
    n = tokens * (case["heads"] + key_heads) * dim
    rows = min(tokens, (tokens // 640 + 1) * 88 + 64)  # of the tables that are used
    # forward: x in, y out; with gradients also dy in, dx out
    return {"bytes": n * size * (4 if case["train"] else 2) + rows * sum(sections) * 8
            + tokens * len(sections) * 8 + 2 * dim * size * (2 if case["train"] else 1),
            "flops": n * (24 if case["train"] else 8)}
  value_dim = case["value_dim"]
  both = dim + value_dim
  if case["op"] == "attend":
    heads = case["heads"]
    pairs = sum(m * (m + 1) // 2 for m in _lengths(case))
    row = (heads + key_heads) * both * size  # queries, keys, values, out
    # scores and out; with gradients again the scores, and of p, v, q and k
    return {"bytes": tokens * row * (2 if case["train"] else 1),
            "flops": 2 * heads * pairs * (both + (3 * dim + 2 * value_dim if case["train"] else 0))}
  if case["op"] == "write":
    touched = sum(-(-(a + m) // case["page"]) - a // case["page"]
                  for a, m in zip(_starts(case), _lengths(case)))
    return {"bytes": tokens * key_heads * both * (size + 1) + touched * (key_heads * 8 + 4),
            "flops": 2 * tokens * key_heads * both}
  pages = sum(-(-m // case["page"]) for m in _lengths(case))
  return {"bytes": tokens * key_heads * both + pages * (8 * key_heads + 4)
          + case["seqs"] * (case["heads"] * both * size + 4),
          "flops": 2 * tokens * case["heads"] * both}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------


def _exact_rotate(s):
  """Norm, weight, and the turn as a product of complex numbers; the gradients
  by the formulas of the norm and of the inverse turn."""
  case, rotary = s["case"], 2 * sum(s["sections"])
  turns, first = [], 0
  for place, count in zip(s["positions"], s["sections"]):
    part = slice(first, first + count)
    turns.append(torch.complex(s["cos"][:, part].double(), s["sin"][:, part].double())[place])
    first += count
  turn = torch.cat(turns, -1)[:, None, :]

  def turned(y, by):
    y = y.clone()
    if case["interleaved"]:
      z = torch.view_as_complex(y[..., :rotary].unflatten(-1, (-1, 2)).contiguous()) * by
      y[..., :rotary] = torch.view_as_real(z).flatten(-2)
    else:
      z = torch.complex(y[..., :rotary // 2], y[..., rotary // 2:rotary]) * by
      y[..., :rotary] = torch.cat((z.real, z.imag), -1)
    return y

  result = {}
  for name, weight in (("queries", "query_weight"), ("keys", "key_weight")):
    x, w = s[name].detach().double(), s[weight].detach().double()
    r = 1.0 / torch.sqrt((x * x).sum(-1, keepdim=True) / case["dim"] + 1e-6)
    result[name] = turned(x * r * w, turn)
    if case["train"]:
      dz = turned(s["d_" + name].double(), turn.conj())
      mean = (dz * w * x * r).sum(-1, keepdim=True) / case["dim"]
      result["grad_" + name] = r * (dz * w - x * r * mean)
      result["grad_" + weight] = (dz * x * r).sum((0, 1))
  return result


def _exact_attend(s):
  """One head of one sequence at a time, probabilities by softmax, gradients by their formulas."""
  case = s["case"]
  share, scale = case["heads"] // case["key_heads"], 1.0 / math.sqrt(case["dim"])
  x = {n: s[n].detach() for n in ("queries", "keys", "values", "d_out") if n in s}

  def empty(name):
    return torch.zeros_like(x[name], dtype=torch.float64, memory_format=torch.contiguous_format)

  result = {"out": torch.zeros(case["tokens"], case["heads"], case["value_dim"],
                               dtype=torch.float64, device="cuda")}
  if case["train"]:
    result.update({"grad_" + n: empty(n) for n in ("queries", "keys", "values")})
  for a, m in zip(_ends(s["lengths"]), s["lengths"]):
    for h in range(case["heads"]):
      k, v = x["keys"][a:a + m, h // share].double(), x["values"][a:a + m, h // share].double()
      for i in range(0, m, 4096):
        e = min(i + 4096, m)
        rows = slice(a + i, a + e)
        q = x["queries"][rows, h].double()
        score = torch.einsum("id,jd->ij", q, k[:e]) * scale
        seen = torch.ones(e - i, e, dtype=torch.bool, device="cuda").tril(i)
        p = torch.softmax(torch.where(seen, score, float("-inf")), -1)
        o = torch.einsum("ij,jd->id", p, v[:e])
        result["out"][rows, h] = o
        if case["train"]:
          do = x["d_out"][rows, h].double()
          ds = p * (do @ v[:e].T - (do * o).sum(-1, keepdim=True)) * scale
          result["grad_queries"][rows, h] = ds @ k[:e]
          result["grad_keys"][a:a + e, h // share] += ds.T @ q
          result["grad_values"][a:a + e, h // share] += p.T @ do
  return result


def _round_e4m3(y):
  """To the nearest of e4m3, ties to even: steps of 2^(e-3) from 2^e on, of 2^-9 below 2^-6."""
  _, e = torch.frexp(y)
  step = torch.ldexp(torch.ones_like(y), (e - 1).clamp(min=-6) - 3)
  return torch.round(y / step) * step


def _exact_write(s):
  """Request by request and page by page."""
  case, page = s["case"], s["case"]["page"]
  keys, values, key_scales, value_scales = s["cache"]
  result = {}
  cu, starts, table = s["cu_seqlens"].tolist(), s["starts"].tolist(), s["pages"].tolist()
  for name, x, held, scales in (("key", s["keys"], keys, key_scales),
                                ("value", s["values"], values, value_scales)):
    pool, unit = held.double(), scales.double()
    x = x.double()
    for b, start in enumerate(starts):
      at, last = start, start + cu[b + 1] - cu[b]
      while at < last:
        end = min(last, (at // page + 1) * page)
        p, o = table[b][at // page], at % page
        new = x[cu[b] + at - start:cu[b] + end - start].transpose(0, 1)  # [heads, n, dim]
        top = new.abs().amax((1, 2))
        need = torch.exp2(torch.ceil(torch.log2(top / LARGEST)).clamp(-SCALE_BITS, SCALE_BITS))
        # log2 next to a power of two may fall on either side of it
        need = torch.where(top > LARGEST * need, 2 * need, need)
        need = torch.where((top <= LARGEST * need / 2) & (need > 2.0**-SCALE_BITS), need / 2, need)
        if o > 0:
          need = torch.maximum(need, unit[p])
          pool[p, :, :o] = _round_e4m3(pool[p, :, :o] * (unit[p] / need)[:, None, None])
        pool[p, :, o:o + end - at] = _round_e4m3(new / need[:, None, None])
        unit[p] = need
        at = end
    result[name + "s"] = pool * unit[..., None, None]
    result[name + "_scales"] = unit
  return {n: result[n] for n in ("keys", "values", "key_scales", "value_scales")}


def _exact_step(s):
  """One request at a time: its tokens gathered in order."""
  case = s["case"]
  share = case["heads"] // case["key_heads"]
  keys, values, key_scales, value_scales = s["cache"]
  out = []
  for b, m in enumerate(s["lengths"].tolist()):
    at = s["pages"][b, :-(-m // case["page"])].long()

    def tokens(x, f):
      x = x.view(torch.uint8)[at].view(torch.float8_e4m3fn).double() * f[at].double()[..., None, None]
      return x.permute(1, 0, 2, 3).flatten(1, 2)[:, :m].repeat_interleave(share, 0)

    score = torch.einsum("hd,hjd->hj", s["queries"][b].double(), tokens(keys, key_scales))
    p = torch.softmax(score / math.sqrt(case["dim"]), -1)
    out.append(torch.einsum("hj,hjd->hd", p, tokens(values, value_scales)))
  return torch.stack(out)


def exact(case, seed):
  s = prepare(case, seed)
  return {"rotate": _exact_rotate, "attend": _exact_attend, "write": _exact_write,
          "step": _exact_step}[case["op"]](s)
