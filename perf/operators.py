"""Workloads of the matrix-state operators: cases, inputs, plain forms and 64-bit results.

Three operators of a gated linear-attention layer, each as a user calls it:

* ``rotate``: RMS norms of queries and keys per head with the position
  rotation in the same pass (``qk_norm_rotate``), alone or with its gradients;
* ``scan``: the matrix-state recurrence S[t] = exp(g[t]) S[t-1] + k[t] v[t]^T,
  o[t] = scale q[t] S[t] over packed sequences (``matrix_scan_causal``), alone
  or with its gradients;
* ``step``: one token of the same recurrence for every running request, over
  a pool of states (``matrix_scan_step``).

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
PLAIN_CHUNK = 64  # tokens of one block of the plain scan


def _package():
  dist = os.path.join(REPO, "associative-scan-triton_b200")
  if dist not in sys.path:
    sys.path.insert(1, dist)
  import associative_scan_triton

  return associative_scan_triton


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------


def _rotate(name, tokens, heads, key_heads, dim, rotary, dtype, train, packed, seqs=1,
            interleaved=False):
  return {"name": name, "op": "rotate", "tokens": tokens, "seqs": seqs, "heads": heads,
          "key_heads": key_heads, "dim": dim, "rotary": rotary, "dtype": dtype, "train": train,
          "packed": packed, "interleaved": interleaved}


def _scan(name, tokens, seqs, heads, key_heads, dim, value_dim, dtype, train, carry, ragged,
          gate_dtype="f32"):
  return {"name": name, "op": "scan", "tokens": tokens, "seqs": seqs, "heads": heads,
          "key_heads": key_heads, "dim": dim, "value_dim": value_dim, "dtype": dtype,
          "train": train, "carry": carry, "ragged": ragged, "gate_dtype": gate_dtype}


def _step(name, batch, heads, key_heads, dim, value_dim, dtype):
  return {"name": name, "op": "step", "batch": batch, "heads": heads, "key_heads": key_heads,
          "dim": dim, "value_dim": value_dim, "dtype": dtype}


def listed():
  return [
    # one new token of each of 16 requests, positions far apart; latency counts
    _rotate("rotate_decode", 16, 12, 12, 128, 128, "bf16", False, "positions"),
    # a training step's 8 sequences of 2048 tokens, 1536 channels
    _rotate("rotate_train", 8 * 2048, 12, 12, 128, 128, "bf16", True, "sequences", seqs=8),
    # ragged sequences, part of an odd head rotated, adjacent pairs, few key heads
    _rotate("rotate_train_ragged", 4999, 16, 4, 80, 32, "f16", True, "sequences", seqs=5,
            interleaved=True),
    # a long prompt, 2048 channels of queries, shared key heads
    _rotate("rotate_prompt_long", 65536, 16, 4, 128, 128, "bf16", False, "sequences"),
    # a short prompt that continues a conversation's state
    _scan("scan_prompt_short", 257, 1, 12, 12, 128, 128, "bf16", False, True, False),
    # prompts of many requests packed, keys and queries shared by four value heads each
    _scan("scan_prompt_packed", 16384, 16, 16, 4, 128, 128, "bf16", False, False, True),
    # one long document
    _scan("scan_prompt_long", 65536, 1, 12, 12, 128, 128, "bf16", False, False, False),
    # a training step's 8 sequences of 2048 tokens, 1536 channels
    _scan("scan_train", 8 * 2048, 8, 12, 12, 128, 128, "bf16", True, False, False),
    # float32 training on ragged sequences, small heads
    _scan("scan_train_f32", 6001, 7, 12, 12, 64, 64, "f32", True, False, True),
    # training on pieces of long documents whose state is carried from piece to piece
    _scan("scan_train_carry", 4 * 8192, 4, 16, 4, 64, 128, "bf16", True, True, False, "bf16"),
    # a single request's next token
    _step("step_single", 1, 12, 12, 128, 128, "bf16"),
    # the next token of a full batch of requests
    _step("step_batch", 256, 12, 12, 128, 128, "bf16"),
  ]


def _log_int(rng, low, high):
  n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
  n = min(max(n, low), high)
  return n + 1 if n == 3 * 1024 else n


def draw(rng):
  op = rng.choice(("rotate", "scan", "scan", "step"))
  dtype = rng.choice(("bf16", "bf16", "bf16", "f16", "f32"))
  heads, key_heads = rng.choice(((12, 12), (16, 4), (16, 16), (8, 1), (12, 3), (5, 5)))
  if op == "rotate":
    train = rng.random() < 0.5
    dim = rng.choice((64, 128, 80, 96, 48))
    rotary = rng.choice((dim, dim // 2))
    packed = rng.choice(("positions", "sequences"))
    tokens = _log_int(rng, 1, 32768 if train else 65536)
    seqs = rng.randint(1, min(tokens, 16)) if packed == "sequences" else 1
    case = _rotate("", tokens, heads, key_heads, dim, rotary, dtype, train, packed, seqs,
                   rng.random() < 0.4)
  elif op == "scan":
    train = rng.random() < 0.5
    dim, value_dim = rng.choice(((64, 64), (128, 128), (128, 128), (64, 128), (128, 64),
                                 (96, 96), (40, 72)))
    largest = 16384 if dtype == "f32" or train else 65536
    tokens = _log_int(rng, 1, largest)
    seqs = rng.randint(1, min(tokens, 16))
    case = _scan("", tokens, seqs, heads, key_heads, dim, value_dim, dtype, train,
                 rng.random() < 0.4, rng.random() < 0.7, rng.choice(("f32", dtype)))
  else:
    dim, value_dim = rng.choice(((64, 64), (128, 128), (64, 128), (96, 96), (40, 72)))
    case = _step("", _log_int(rng, 1, 192), heads, key_heads, dim, value_dim, dtype)
  del case["name"]
  return case


def _lengths(case):
  """The sequences' lengths: equal, or spread between a quarter and 1.75 of the mean."""
  n, tokens = case["seqs"], case["tokens"]
  if not case.get("ragged", case["op"] == "rotate"):
    return [tokens // n + (1 if i < tokens % n else 0) for i in range(n)]
  rng = random.Random(tokens * 31 + n)
  weights = [rng.uniform(0.25, 1.75) for _ in range(n)]
  ends = [int(round((tokens - n) * sum(weights[:i + 1]) / sum(weights))) for i in range(n)]
  return [b - a + 1 for a, b in zip([0] + ends[:-1], ends)]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _unit(x):
  return x / x.square().mean(-1, keepdim=True).sqrt()


def _gates(shape, heads, gen, device):
  """Log gates as trained layers have them: a rate per head over two decades,
  and a step size per token and head."""
  rate = torch.exp(torch.linspace(0.0, math.log(16.0), heads, device=device))
  size = torch.rand(shape, generator=gen, device=device) * (math.log(0.1) - math.log(0.001))
  return -rate * torch.exp(size + math.log(0.001))


def _table(rows, half, device):
  freq = torch.exp(torch.arange(half, device=device, dtype=torch.float64)
                   * (-math.log(10000.0) / max(1, half)))
  angle = torch.arange(rows, device=device, dtype=torch.float64)[:, None] * freq
  return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
  device = torch.device("cuda")
  gen = torch.Generator(device=device).manual_seed(seed)
  dtype = TYPES[case["dtype"]]

  def normal(*shape):
    return torch.randn(shape, generator=gen, device=device)

  s = {"case": case}
  heads, key_heads, dim = case["heads"], case["key_heads"], case["dim"]
  if case["op"] == "rotate":
    n = case["tokens"]
    # queries and keys are views of one projection's output, as a layer has them
    both = normal(n, heads + key_heads, dim) * (0.5 + 1.5 * torch.rand(
      (heads + key_heads, 1), generator=gen, device=device))
    both = both.to(dtype)
    s["queries"], s["keys"] = both[:, :heads], both[:, heads:]
    s["query_weight"] = (1.0 + 0.2 * normal(dim)).to(dtype)
    s["key_weight"] = (1.0 + 0.2 * normal(dim)).to(dtype)
    if case["packed"] == "positions":
      s["positions"] = torch.randint(0, 65536, (n,), generator=gen, device=device)
      rows = 65536
    else:
      lengths = _lengths(case)
      s["cu_seqlens"] = torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)],
                                     dtype=torch.int32, device=device)
      rows = max(lengths)
    s["cos"], s["sin"] = _table(rows, case["rotary"] // 2, device)
    if case["train"]:
      s["d_queries"] = normal(n, heads, dim).to(dtype)
      s["d_keys"] = normal(n, key_heads, dim).to(dtype)
    wrt = ("queries", "keys", "query_weight", "key_weight")
  else:
    n = case["tokens"] if case["op"] == "scan" else case["batch"]
    s["queries"] = _unit(normal(n, key_heads, dim)).to(dtype)
    s["keys"] = _unit(normal(n, key_heads, dim)).to(dtype)
    s["values"] = normal(n, heads, case["value_dim"]).to(dtype)
    s["log_gates"] = _gates((n, heads), heads, gen, device)
    if case["op"] == "scan":
      s["log_gates"] = s["log_gates"].to(TYPES[case["gate_dtype"]])
      lengths = _lengths(case)
      s["max_len"] = max(lengths)
      s["cu_seqlens"] = torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)],
                                     dtype=torch.int32, device=device)
      if case["carry"]:
        s["initial_state"] = normal(len(lengths), heads, dim, case["value_dim"]) * 4.0
      if case["train"]:
        s["d_out"] = normal(n, heads, case["value_dim"]).to(dtype)
        if case["carry"]:
          s["d_final_state"] = normal(len(lengths), heads, dim, case["value_dim"])
    else:
      pool = n + 3
      s["state"] = normal(pool, heads, dim, case["value_dim"]) * 4.0
      s["state_out"] = torch.zeros_like(s["state"])
      s["slots"] = torch.randperm(pool, generator=gen, device=device)[:n].to(torch.int32)
    wrt = ("queries", "keys", "values", "log_gates", "initial_state")
  if case.get("train"):
    s["wrt"] = [w for w in wrt if w in s]
    for w in s["wrt"]:
      s[w] = s[w].detach().requires_grad_(True)
  return s


# ---------------------------------------------------------------------------
# plain forms: float32, elementary operations
# ---------------------------------------------------------------------------


def _plain_rotate(s):
  case = s["case"]
  if "positions" in s:
    pos = s["positions"]
  else:
    cu = s["cu_seqlens"].long()
    at = torch.arange(case["tokens"], device=cu.device)
    pos = at - cu[torch.searchsorted(cu, at, right=True) - 1]
  cos, sin = s["cos"][pos][:, None, :], s["sin"][pos][:, None, :]
  rotary, half = case["rotary"], case["rotary"] // 2

  def one(x, w):
    y = x.float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w.float()
    if case["interleaved"]:
      a, b = y[..., 0:rotary:2], y[..., 1:rotary:2]
      turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
      a, b = y[..., :half], y[..., half:rotary]
      turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, y[..., rotary:]), -1).to(x.dtype)

  return one(s["queries"], s["query_weight"]), one(s["keys"], s["key_weight"])


def _segment_sums(x):
  """[..., n] -> [..., n, n]: the sum of x over (j, i] for i >= j, else -inf."""
  n = x.shape[-1]
  below = torch.ones(n, n, dtype=torch.bool, device=x.device).tril(-1)
  sums = x[..., :, None].expand(*x.shape, n).masked_fill(~below, 0.0).cumsum(-2)
  return sums.masked_fill(~below.logical_or(torch.eye(n, dtype=torch.bool, device=x.device)),
                          -math.inf)


def _plain_scan(s):
  case, c = s["case"], PLAIN_CHUNK
  v = s["values"]
  heads, dim, scale = case["heads"], case["dim"], case["dim"] ** -0.5
  cu = s["cu_seqlens"].long()
  n, blocks = cu.numel() - 1, -(-s["max_len"] // c)
  at = cu[:-1, None] + torch.arange(blocks * c, device=v.device)
  inside = at < cu[1:, None]
  at = at.clamp(max=case["tokens"] - 1)

  def lay(x, share):  # [tokens, heads, d] -> [seqs, heads, blocks, c, d]
    x = x.float()[at].masked_fill(~inside[..., None, None], 0.0)
    x = x.repeat_interleave(share, 2) if share > 1 else x
    return x.view(n, blocks, c, heads, -1).permute(0, 3, 1, 2, 4)

  share = heads // case["key_heads"]
  q, k, v = lay(s["queries"], share), lay(s["keys"], share), lay(s["values"], 1)
  g = lay(s["log_gates"][..., None], 1)[..., 0]
  decay = torch.exp(_segment_sums(g))
  out = (q @ k.transpose(-1, -2) * decay) @ v
  added = (k * decay[..., -1, :, None]).transpose(-1, -2) @ v
  first = s.get("initial_state")
  if first is None:
    first = added.new_zeros(n, heads, dim, case["value_dim"])
  states = torch.cat((first[:, :, None], added), 2)
  across = torch.exp(_segment_sums(torch.nn.functional.pad(g.sum(-1), (1, 0))))
  states = (across @ states.flatten(-2)).view_as(states)
  out = out + (q * torch.exp(g.cumsum(-1))[..., None]) @ states[:, :, :-1]
  out = (out * scale).permute(0, 2, 3, 1, 4).reshape(n, blocks * c, heads, -1)
  return out[inside].to(s["values"].dtype), states[:, :, -1]


def _plain_step(s):
  case = s["case"]
  share = case["heads"] // case["key_heads"]
  q = s["queries"].float().repeat_interleave(share, 1)
  k = s["keys"].float().repeat_interleave(share, 1)
  slots = s["slots"].long()
  new = (s["state"][slots] * torch.exp(s["log_gates"].float())[..., None, None]
         + k[..., :, None] * s["values"].float()[..., None, :])
  out = (q[..., None] * new).sum(-2) * case["dim"] ** -0.5
  s["state_out"][slots] = new
  return out.to(s["values"].dtype)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(s):
  case = s["case"]
  if case["op"] == "step":
    if own:
      out = _package().matrix_scan_step(s["queries"], s["keys"], s["values"], s["log_gates"],
                                        s["state"], slots=s["slots"], state_out=s["state_out"])
    else:
      out = _plain_step(s)
    return {"out": out, "state": s["state_out"]}
  if case["op"] == "rotate":
    if own:
      where = ({"positions": s["positions"]} if "positions" in s
               else {"args": {"cu_seqlens": s["cu_seqlens"]}})
      q, k = _package().qk_norm_rotate(s["queries"], s["keys"], s["query_weight"],
                                       s["key_weight"], s["cos"], s["sin"], eps=1e-6,
                                       interleaved=case["interleaved"], **where)
    else:
      q, k = _plain_rotate(s)
    result = {"queries": q, "keys": k}
    ends, grads = [q, k], [s.get("d_queries"), s.get("d_keys")]
  else:
    if own:
      out, final = _package().matrix_scan_causal(
        s["queries"], s["keys"], s["values"], s["log_gates"], {"cu_seqlens": s["cu_seqlens"]},
        initial_state=s.get("initial_state"), return_final_state=True)
    else:
      out, final = _plain_scan(s)
    result = {"out": out, "final_state": final}
    ends, grads = [out], [s.get("d_out")]
    if "d_final_state" in s:
      ends, grads = [out, final], [s["d_out"], s["d_final_state"]]
  if case["train"]:
    found = torch.autograd.grad(ends, [s[w] for w in s["wrt"]], grads)
    result.update({"grad_" + w: d for w, d in zip(s["wrt"], found)})
  return {name: x.detach() for name, x in result.items()}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
  size, heads, key_heads, dim = (SIZE[case["dtype"]], case["heads"], case["key_heads"],
                                 case["dim"])
  if case["op"] == "rotate":
    n = case["tokens"] * (heads + key_heads) * dim
    table = (case["tokens"] if case["packed"] == "positions" else max(_lengths(case))) * (
      case["rotary"] * 4)
    # forward: x in, y out; with gradients also dy in, dx out
    return {"bytes": n * size * (4 if case["train"] else 2) + table
            + 2 * dim * size * (2 if case["train"] else 1),
            "flops": n * (24 if case["train"] else 8)}
  n = case["tokens"] if case["op"] == "scan" else case["batch"]
  value_dim = case["value_dim"]
  row_in = (2 * key_heads * dim + heads * value_dim) * size
  row_out = heads * value_dim * size
  matrix = heads * dim * value_dim
  if case["op"] == "step":
    # the state in and out; decay, outer product and one product with the query
    return {"bytes": n * (row_in + row_out + heads * 4 + 8 * matrix + 4), "flops": 5 * n * matrix}
  gate = heads * SIZE[case["gate_dtype"]]
  state = case["seqs"] * matrix * 4
  if not case["train"]:
    return {"bytes": n * (row_in + gate + row_out) + state * (2 if case["carry"] else 1),
            "flops": 5 * n * matrix}
  # gradients: inputs and d_out in, out and the inputs' gradients out; the states
  # once more, their adjoints, and three products with them per token
  return {"bytes": n * (2 * (row_in + gate) + 2 * row_out) + state * (4 if case["carry"] else 1),
          "flops": 17 * n * matrix}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------


def _exact_rotate(s):
  """Norm, weight, and the turn as a product of complex numbers; the gradients
  by the formulas of the norm and of the inverse turn."""
  case = s["case"]
  if "positions" in s:
    pos = s["positions"]
  else:
    pos = torch.cat([torch.arange(m, device="cuda") for m in _lengths(case)])
  turn = torch.complex(s["cos"].double(), s["sin"].double())[pos][:, None, :]
  rotary = case["rotary"]

  def turned(y, by):
    y = y.clone()
    if case["interleaved"]:
      z = torch.complex(y[..., 0:rotary:2], y[..., 1:rotary:2]) * by
      y[..., 0:rotary:2], y[..., 1:rotary:2] = z.real, z.imag
    else:
      z = torch.complex(y[..., :rotary // 2], y[..., rotary // 2:rotary]) * by
      y[..., :rotary // 2], y[..., rotary // 2:rotary] = z.real, z.imag
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


def _exact_scan(s):
  """Token by token, forwards for the states and, for the gradients, backwards
  for their adjoints."""
  case = s["case"]
  lengths = _lengths(case)
  n, heads, longest = len(lengths), case["heads"], max(lengths)
  share = heads // case["key_heads"]
  scale = 1.0 / math.sqrt(case["dim"])
  rows = torch.repeat_interleave(torch.arange(n, device="cuda"),
                                 torch.tensor(lengths, device="cuda"))
  cols = torch.cat([torch.arange(m, device="cuda") for m in lengths])

  def spread(x):  # [tokens, h, d] -> [longest, seqs, heads, d], zero past each end
    y = torch.zeros(longest, n, x.shape[1], x.shape[2], dtype=torch.float64, device="cuda")
    y[cols, rows] = x.detach().double()
    return y.repeat_interleave(heads // x.shape[1], 2)

  q, k, v = spread(s["queries"]) * scale, spread(s["keys"]), spread(s["values"])
  g = spread(s["log_gates"][..., None])[..., 0]
  a = g.exp()
  alive = torch.zeros(longest, n, 1, dtype=torch.float64, device="cuda")
  alive[cols, rows] = 1.0
  matrix = torch.zeros(n, heads, case["dim"], case["value_dim"], dtype=torch.float64,
                       device="cuda")
  if "initial_state" in s:
    matrix = matrix + s["initial_state"].detach().double()
  out = torch.empty_like(v)
  dq = torch.empty_like(q)
  do = spread(s["d_out"]) if case["train"] else None
  for t in range(longest):
    matrix.mul_(a[t, :, :, None, None]).addcmul_(k[t, :, :, :, None], v[t, :, :, None, :])
    out[t] = (matrix * q[t, :, :, :, None]).sum(-2)
    if case["train"]:
      dq[t] = (matrix * do[t, :, :, None, :]).sum(-1)
  result = {"out": out[cols, rows], "final_state": matrix}
  if not case["train"]:
    return result
  adjoint = torch.zeros_like(matrix)
  ends = torch.zeros(n, heads, dtype=torch.float64, device="cuda")
  if "d_final_state" in s:
    adjoint = adjoint + s["d_final_state"].double()
    ends = (adjoint * matrix).sum((-1, -2))
  dk, dv = torch.empty_like(k), torch.empty_like(v)
  for t in range(longest - 1, -1, -1):
    adjoint.addcmul_(q[t, :, :, :, None], do[t, :, :, None, :])
    dk[t] = (adjoint * v[t, :, :, None, :]).sum(-1)
    dv[t] = (adjoint * k[t, :, :, :, None]).sum(-2)
    adjoint.mul_(a[t, :, :, None, None])
  # a gate's gradient: every later q.dq less every later k.dk, and the end's share
  flow = (q * dq).sum(-1) - (k * dk).sum(-1)
  dg = (flow * alive).flip(0).cumsum(0).flip(0) + ends

  def summed(x):
    x = x[cols, rows]
    return x.view(x.shape[0], heads // share, share, -1).sum(2)

  result.update({"grad_queries": summed(dq * scale), "grad_keys": summed(dk),
                 "grad_values": dv[cols, rows], "grad_log_gates": dg[cols, rows]})
  if "initial_state" in s:
    result["grad_initial_state"] = adjoint
  return result


def exact(case, seed):
  s = prepare(case, seed)
  if case["op"] == "rotate":
    return _exact_rotate(s)
  if case["op"] == "scan":
    return _exact_scan(s)
  share, slots = case["heads"] // case["key_heads"], s["slots"].long()
  q = s["queries"].double().repeat_interleave(share, 1)
  k = s["keys"].double().repeat_interleave(share, 1)
  state = torch.zeros_like(s["state"], dtype=torch.float64)
  state[slots] = (s["state"].double()[slots] * s["log_gates"].double().exp()[..., None, None]
                  + torch.einsum("bhi,bhj->bhij", k, s["values"].double()))
  return {"out": torch.einsum("bhi,bhij->bhj", q, state[slots]) / math.sqrt(case["dim"]),
          "state": state}
