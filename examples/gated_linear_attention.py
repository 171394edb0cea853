"""A gated linear-attention layer: trained on packed sequences, then decoded token by token.

    python examples/gated_linear_attention.py [--steps 300] [--dim 256] [--heads 4]

One layer between an embedding and a linear head learns to remember: a
sequence opens with a marker, noise follows, and every token has to name the
marker, which only the layer's state can know.  Training runs the whole packed batch through
``qk_norm_rotate`` and ``matrix_scan_causal``; serving reads a prompt the same
way, keeps only the final state of every request, and continues with
``matrix_scan_step``.  The two must agree.  Needs a CUDA device (B200).
"""

from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "associative-scan-triton_b200"))

import associative_scan_triton as ast  # noqa: E402


def angle_tables(positions: int, half: int, device) -> tuple[torch.Tensor, torch.Tensor]:
  freq = torch.exp(torch.arange(half, device=device) * (-math.log(10000.0) / half))
  angle = torch.arange(positions, device=device)[:, None] * freq
  return angle.cos().contiguous(), angle.sin().contiguous()


class GatedLinearAttention(nn.Module):
  """Queries and keys with norm and rotation, a decay per head and token, a matrix state."""

  def __init__(self, dim: int, heads: int, positions: int, device="cuda"):
    super().__init__()
    self.heads, self.size = heads, dim // heads
    kw = {"bias": False, "device": device}
    self.qkv = nn.Linear(dim, 3 * dim, **kw)
    self.gate = nn.Linear(dim, heads, device=device)
    nn.init.constant_(self.gate.bias, 4.0)  # long memory to begin with
    self.out = nn.Linear(dim, dim, **kw)
    self.query_weight = nn.Parameter(torch.ones(self.size, device=device))
    self.key_weight = nn.Parameter(torch.ones(self.size, device=device))
    cos, sin = angle_tables(positions, self.size // 2, device)
    self.register_buffer("cos", cos)
    self.register_buffer("sin", sin)

  def _project(self, x, **where):
    # views of one projection; no copies before the kernels
    q, k, v = self.qkv(x).view(x.shape[0], 3, self.heads, self.size).unbind(1)
    q, k = ast.qk_norm_rotate(q, k, self.query_weight, self.key_weight, self.cos, self.sin, **where)
    log_gates = nn.functional.logsigmoid(self.gate(x).float())
    return q, k, v, log_gates

  def forward(self, x, args, initial_state=None):
    """x: [BL, dim] packed by args["cu_seqlens"].  Returns (y, final_state)."""
    y, state = ast.matrix_scan_causal(*self._project(x, args=args), args,
                                      initial_state=initial_state, return_final_state=True)
    return self.out(y.flatten(1)), state

  @torch.no_grad()
  def step(self, x, positions, pool, slots):
    """x: [B, dim], one new token of each request; the pool is updated in place."""
    y = ast.matrix_scan_step(*self._project(x, positions=positions), pool, slots=slots)
    return self.out(y.flatten(1))


class Model(nn.Module):
  """Float32 weights, bfloat16 products and kernels."""

  def __init__(self, vocab: int, dim: int, heads: int, positions: int):
    super().__init__()
    self.embed = nn.Embedding(vocab, dim, device="cuda")
    self.layer = GatedLinearAttention(dim, heads, positions)
    self.head = nn.Linear(dim, vocab, device="cuda")

  @torch.autocast("cuda", dtype=torch.bfloat16)
  def forward(self, tokens, args):
    x = self.embed(tokens)
    y, state = self.layer(x, args)
    return self.head(x + y), state

  @torch.no_grad()
  @torch.autocast("cuda", dtype=torch.bfloat16)
  def step(self, tokens, positions, pool, slots):
    x = self.embed(tokens)
    return self.head(x + self.layer.step(x, positions, pool, slots))


def batch(lengths: list[int], vocab: int, gen) -> tuple[torch.Tensor, torch.Tensor, dict]:
  """Packed sequences, a marker (the lower half of the vocabulary) before noise
  (the upper half): tokens, targets, args."""
  tokens, targets = [], []
  for n in lengths:
    marker = torch.randint(0, vocab // 2, (1,), generator=gen)
    tokens.append(torch.cat((marker, torch.randint(vocab // 2, vocab, (n - 1,), generator=gen))))
    targets.append(marker.expand(n))
  ends = torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32)
  return torch.cat(tokens).cuda(), torch.cat(targets).cuda(), {"cu_seqlens": ends.cuda()}


def train(model: Model, steps: int, vocab: int, gen) -> list[float]:
  optimizer = torch.optim.Adam(model.parameters(), lr=3e-3)
  losses = []
  for _ in range(steps):
    lengths = torch.randint(8, 160, (16,), generator=gen).tolist()
    tokens, targets, args = batch(lengths, vocab, gen)
    logits, _ = model(tokens, args)
    loss = nn.functional.cross_entropy(logits.float(), targets)
    optimizer.zero_grad()
    loss.backward()
    optimizer.step()
    losses.append(float(loss.detach()))
  return losses


@torch.no_grad()
def decode(model: Model, prompts: torch.Tensor, args: dict,
           new_tokens: int) -> tuple[torch.Tensor, torch.Tensor]:
  """Greedy continuation of packed prompts: tokens [requests, new_tokens] and their logits."""
  lengths = args["cu_seqlens"].diff()
  logits, state = model(prompts, args)
  # requests come and go in a server: states sit in a pool, a request has a slot
  pool = torch.zeros(len(lengths) + 2, *state.shape[1:], device="cuda")
  slots = torch.arange(len(lengths), 0, -1, dtype=torch.int32, device="cuda")
  pool[slots.long()] = state
  seen = [logits[(args["cu_seqlens"][1:] - 1).long()]]
  positions = lengths.clone()
  for _ in range(new_tokens - 1):
    seen.append(model.step(seen[-1].argmax(-1), positions, pool, slots))
    positions += 1
  seen = torch.stack(seen, 1)
  return seen.argmax(-1), seen


def main(argv: list[str] | None = None) -> int:
  ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
  ap.add_argument("--steps", type=int, default=300)
  ap.add_argument("--dim", type=int, default=256)
  ap.add_argument("--heads", type=int, default=4)
  ap.add_argument("--vocab", type=int, default=32)
  a = ap.parse_args(argv)
  torch.manual_seed(0)
  gen = torch.Generator().manual_seed(1)
  model = Model(a.vocab, a.dim, a.heads, positions=256)
  losses = train(model, a.steps, a.vocab, gen)
  print(f"loss: first {losses[0]:.3f}, last {losses[-1]:.3f}")

  prompts, targets, args = batch([40, 61, 25], a.vocab, gen)
  chosen, seen = decode(model, prompts, args, new_tokens=24)
  starts = args["cu_seqlens"].tolist()
  right = int((chosen == targets[args["cu_seqlens"][:-1].long(), None]).sum())
  print(f"continuation: {right} of {chosen.numel()} tokens name the marker")

  # the same tokens in one pass: the same logits, but for bfloat16's roundings
  whole = torch.cat([torch.cat((prompts[x:y], chosen[i, :-1])) for i, (x, y) in enumerate(zip(starts, starts[1:]))])
  grown = [y - x + chosen.shape[1] - 1 for x, y in zip(starts, starts[1:])]
  ends = torch.tensor([sum(grown[:i]) for i in range(len(grown) + 1)], dtype=torch.int32, device="cuda")
  with torch.no_grad():
    logits, _ = model(whole, {"cu_seqlens": ends})
  tail = torch.cat([torch.arange(int(e) - chosen.shape[1], int(e)) for e in ends[1:]])
  again = logits[tail.cuda()].view_as(seen).float()
  apart = float((again - seen.float()).norm() / again.norm())
  print(f"one pass and step by step: logits {100 * apart:.2f}% apart")
  ast.check_device_error()
  return 0 if apart < 0.05 and losses[-1] < losses[0] else 1


if __name__ == "__main__":
  sys.exit(main())
