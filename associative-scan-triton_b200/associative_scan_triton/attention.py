"""Softmax attention for the layers that stand between gated linear-attention layers.

* :func:`attention_causal`: causal softmax attention over packed sequences with
  grouped heads, with gradients for every input.
* :func:`attention_cache_write`: new keys and values into the pages of a cache
  in 8 bits with a scale for each page and head.
* :func:`attention_cache_step`: the attention of one new token of many requests
  over that cache.

Tensors are as in matrix_scan.py: ``[BL, heads, dim]``, all sequences packed
along the first axis, unit stride along the last, token and head strides free;
float32, float16 and bfloat16.  Every call runs on torch's current stream and
takes its workspace from torch's allocator.  No forward-mode derivatives.

Precision: scores, softmax statistics and sums are float32.  float32 inputs
are computed in float32, float16 and bfloat16 ones (head sizes a multiple of 8)
on tensor cores: probabilities and, for gradients, their derivatives are
rounded to the inputs' type as operands of the second products, which adds as
much to a result as its own rounding does.
"""

from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch

from . import _lib
from ._lib import DTYPE_CODES, INDEX_CODES
from .matrix_scan import (_NS, _check_index, _check_rows, _like, _none, _on, _ptr, _refuse_tangents,
                          _rows, _stream)

MAX_DIM = 128  # of a head
MAX_TOKENS = 0x3FFFFFFF
MAX_PAGE = 4096
CACHE_DTYPE = torch.float8_e4m3fn


def _check_scale(scale, dim: int) -> float:
  scale = float(dim) ** -0.5 if scale is None else float(scale)
  if not 0.0 < scale < float("inf"):
    raise ValueError(f"scale must be positive and finite, got {scale}")
  return scale


# ---------------------------------------------------------------------------
# causal attention over packed sequences
# ---------------------------------------------------------------------------


def _check_attention(queries, keys, values, cu_seqlens):
  try:  # the usual call in one expression; whatever fails it is looked at below
    (n, h, dk), (nk, hk, dkk), (nv, hv, dv) = queries.shape, keys.shape, values.shape
    device, dtype = queries.device, queries.dtype
    if (queries.is_cuda and keys.device == device and values.device == device
        and cu_seqlens.device == device and dtype in DTYPE_CODES and keys.dtype == dtype
        and values.dtype == dtype and cu_seqlens.dtype in INDEX_CODES and nk == n and nv == n
        and dkk == dk and 1 < dk <= MAX_DIM and 1 < dv <= MAX_DIM and 0 < h <= 65535 and hk > 0
        and hv == hk and h % hk == 0 and n <= MAX_TOKENS and cu_seqlens.dim() == 1
        and 0 < cu_seqlens.shape[0] <= MAX_TOKENS and cu_seqlens.is_contiguous()
        and queries.stride(2) == 1 and keys.stride(2) == 1 and values.stride(2) == 1):
      return _lib._enable_error_flag()
  except (AttributeError, TypeError, ValueError):
    pass
  _check_rows("queries", queries, None, None)
  device, tokens, dim = queries.device, queries.shape[0], queries.shape[2]
  _check_rows("keys", keys, device, queries.dtype, tokens, dim)
  _check_rows("values", values, device, queries.dtype, tokens)
  if max(dim, values.shape[2]) > MAX_DIM:
    raise ValueError(f"head sizes up to {MAX_DIM} are supported, got {dim} and {values.shape[2]}")
  if values.shape[1] != keys.shape[1] or queries.shape[1] % keys.shape[1]:
    raise ValueError(f"keys and values need the same number of heads, a divisor of the queries' "
                     f"{queries.shape[1]}, got {keys.shape[1]} and {values.shape[1]}")
  _check_index("cu_seqlens", cu_seqlens, device)
  if cu_seqlens.numel() < 1:
    raise ValueError("cu_seqlens must have at least one entry")
  if max(tokens, cu_seqlens.numel()) > MAX_TOKENS:
    raise ValueError(f"at most {MAX_TOKENS} tokens and sequences are supported")
  _lib._enable_error_flag()


def _wide(t: torch.Tensor) -> torch.Tensor:
  """16-bit rows in the layout that the tensor-core kernels load: a view that
  starts or steps off 16 bytes, or repeats itself, is copied once."""
  if t.dtype == torch.float32 or t.shape[2] % 8:
    return t
  st, sh, _ = t.stride()
  if (t.data_ptr() % 16 == 0 and st % 8 == 0 and st >= t.shape[2] and st < 1 << 38
      and (t.shape[1] == 1 or (sh % 8 == 0 and sh >= t.shape[2] and sh < 1 << 38))):
    return t
  return t.clone(memory_format=torch.contiguous_format)


def _attention_forward(queries, keys, values, cu_seqlens, scale, train):
  """(out, rest, lse); the last two None unless ``train``."""
  _refuse_tangents(NotImplementedError, "attention_causal", queries, keys, values)
  _check_attention(queries, keys, values, cu_seqlens)
  device, (tokens, heads, dim), value_dim = queries.device, queries.shape, values.shape[2]
  num_seq = cu_seqlens.numel() - 1
  inputs = [_wide(t) for t in (queries, keys, values)]  # the copies, if any, live until the launch
  out = torch.empty((tokens, heads, value_dim), dtype=values.dtype, device=device)
  rest = torch.empty_like(out) if train and out.dtype != torch.float32 else None
  lse = torch.empty((heads, tokens), dtype=torch.float32, device=device) if train else None
  if tokens == 0 or num_seq == 0:
    out.zero_()
    return out, rest, lse
  with _on(device):
    rc = _lib.load().ascan_attention_forward(
      *_rows(*inputs), cu_seqlens.data_ptr(),
      INDEX_CODES[cu_seqlens.dtype], num_seq, tokens, dim, value_dim, DTYPE_CODES[queries.dtype],
      scale, out.data_ptr(), _ptr(rest), _ptr(lse), _stream(device))
  _lib._finish(rc, "ascan_attention_forward", device)
  return out, rest, lse


def _attention_backward(queries, keys, values, cu_seqlens, out, rest, lse, scale, d_out):
  device, (tokens, heads, dim), value_dim = queries.device, queries.shape, values.shape[2]
  num_seq = cu_seqlens.numel() - 1
  d_queries, d_keys, d_values = _like(queries), _like(keys), _like(values)
  if tokens == 0 or num_seq == 0:
    return d_queries.zero_(), d_keys.zero_(), d_values.zero_()
  if d_out.stride(2) != 1 and value_dim > 1:
    d_out = d_out.contiguous()
  lib = _lib.load()
  with _on(device):
    ws = torch.empty(lib.ascan_attention_workspace(tokens, heads), dtype=torch.uint8, device=device)
    inputs = [_wide(t) for t in (queries, keys, values, d_out)]
    rc = lib.ascan_attention_backward(
      *_rows(*inputs), out.data_ptr(), _ptr(rest), lse.data_ptr(), cu_seqlens.data_ptr(),
      INDEX_CODES[cu_seqlens.dtype], num_seq, tokens, dim, value_dim, DTYPE_CODES[queries.dtype],
      scale, d_queries.data_ptr(), d_keys.data_ptr(), d_values.data_ptr(), ws.data_ptr(),
      ws.numel(), _stream(device))
  _lib._finish(rc, "ascan_attention_backward", device)
  return d_queries, d_keys, d_values


class AttentionCausal(torch.autograd.Function):
  """attention_causal with its gradients."""

  @staticmethod
  def forward(ctx, queries, keys, values, cu_seqlens, scale):
    out, rest, lse = _attention_forward(queries, keys, values, cu_seqlens, scale, True)
    ctx.save_for_backward(queries, keys, values, cu_seqlens, out, rest, lse)
    ctx.scale = scale
    ctx.set_materialize_grads(False)
    return out

  @staticmethod
  @torch.autograd.function.once_differentiable
  def backward(ctx, d_out):
    if d_out is None:
      return (None,) * 5
    return (*_attention_backward(*ctx.saved_tensors, ctx.scale, d_out), None, None)


def attention_causal(
  queries: torch.Tensor,
  keys: torch.Tensor,
  values: torch.Tensor,
  args: dict,
  scale: float | None = None,
) -> torch.Tensor:
  """Causal softmax attention over packed sequences.

  ``out[i] = sum_j p[i, j] values[j]`` over the tokens ``j <= i`` of i's
  sequence, with ``p`` the softmax over them of ``scale queries[i].keys[j]``.

  Args:
    queries: [BL, H, Dk]; keys: [BL, Hk, Dk]; values: [BL, Hk, Dv]; Hk divides
      H and query head h reads head h // (H // Hk); Dk, Dv <= 128.
    args: {"cu_seqlens": [N+1] int tensor}; other entries are not used.
    scale: factor of the scores, positive; Dk**-0.5 by default.
  A key or value that is not finite reaches its own row and later ones only.
  Shared heads get the summed gradient.  Tokens of no sequence give zero rows.
  Returns:
    out [BL, H, Dv].
  """
  scale = _check_scale(scale, queries.shape[-1])
  cu_seqlens = args["cu_seqlens"]
  if torch.is_grad_enabled() and (queries.requires_grad or keys.requires_grad
                                  or values.requires_grad):
    return AttentionCausal.apply(queries, keys, values, cu_seqlens, scale)
  return _attention_forward(queries, keys, values, cu_seqlens, scale, False)[0]


# ---------------------------------------------------------------------------
# the cache
# ---------------------------------------------------------------------------


class AttentionCache(NamedTuple):
  """Pages of keys and values in 8 bits; a page's values are ``scale * element``.

  keys: [pages, heads, page, Dk] float8_e4m3fn; values: [pages, heads, page, Dv];
  key_scales, value_scales: [pages, heads] float32.
  """

  keys: torch.Tensor
  values: torch.Tensor
  key_scales: torch.Tensor
  value_scales: torch.Tensor


def attention_cache(pages: int, heads: int, page: int, key_dim: int, value_dim: int | None = None,
                    device="cuda") -> AttentionCache:
  """An empty cache of ``pages`` pages of ``page`` tokens (a multiple of 16)."""
  value_dim = key_dim if value_dim is None else value_dim
  cache = AttentionCache(
    torch.zeros(pages, heads, page, key_dim, dtype=torch.uint8, device=device).view(CACHE_DTYPE),
    torch.zeros(pages, heads, page, value_dim, dtype=torch.uint8, device=device).view(CACHE_DTYPE),
    torch.ones(pages, heads, device=device), torch.ones(pages, heads, device=device))
  _check_cache_sizes(cache.keys, cache.values)
  return cache


def _check_cache_sizes(keys, values) -> None:
  page, key_dim, value_dim = keys.shape[2], keys.shape[3], values.shape[3]
  if page < 16 or page > MAX_PAGE or page % 16:
    raise ValueError(f"a page holds a multiple of 16 tokens, at most {MAX_PAGE}, got {page}")
  for dim in (key_dim, value_dim):
    if dim < 16 or dim > MAX_DIM or dim % 16:
      raise ValueError(f"head sizes must be multiples of 16 up to {MAX_DIM}, got {key_dim} and "
                       f"{value_dim}")
  if keys.shape[1] < 1 or keys.shape[1] > 65535:
    raise ValueError(f"a cache has between 1 and 65535 heads, got {keys.shape[1]}")


def _usual_cache(cache, device, heads: int, key_dim: int):
  """Value size of a cache that passes _check_cache, in one expression; None sends the caller there."""
  keys, values, key_scales, value_scales = cache
  (pages, h, page, dk), (pv, hv, page_v, dv) = keys.shape, values.shape
  return dv if (
    keys.device == device and values.device == device and key_scales.device == device
    and value_scales.device == device and keys.dtype == CACHE_DTYPE and values.dtype == CACHE_DTYPE
    and key_scales.dtype == torch.float32 and value_scales.dtype == torch.float32 and pv == pages
    and hv == h and page_v == page and h > 0 and heads % h == 0 and dk == key_dim and not dk % 16
    and not dv % 16 and not page % 16 and 0 < dk <= MAX_DIM and 0 < dv <= MAX_DIM
    and 0 < page <= MAX_PAGE and h <= 65535 and key_scales.shape == (pages, h)
    and value_scales.shape == (pages, h) and keys.is_contiguous() and values.is_contiguous()
    and key_scales.is_contiguous() and value_scales.is_contiguous()) else None


def _check_cache(cache, device):
  """The cache's four tensors."""
  try:
    keys, values, key_scales, value_scales = cache
  except (TypeError, ValueError):
    raise TypeError("cache must be an AttentionCache: keys, values, key_scales, value_scales") from None
  for name, t in (("cache keys", keys), ("cache values", values)):
    _lib._require_cuda(name, t, device)
    if t.dtype != CACHE_DTYPE:
      raise TypeError(f"{name} must be {CACHE_DTYPE}, got {t.dtype}")
    if t.dim() != 4 or not t.is_contiguous():
      raise ValueError(f"{name} must be contiguous [pages, heads, page, dim], got shape "
                       f"{tuple(t.shape)}")
  if values.shape[:3] != keys.shape[:3]:
    raise ValueError(f"cache keys and values differ in pages, heads or page size: "
                     f"{tuple(keys.shape)}, {tuple(values.shape)}")
  _check_cache_sizes(keys, values)
  for name, t in (("key_scales", key_scales), ("value_scales", value_scales)):
    _lib._require_cuda(name, t, device)
    if t.dtype != torch.float32:
      raise TypeError(f"{name} must be float32, got {t.dtype}")
    if t.shape != keys.shape[:2] or not t.is_contiguous():
      raise ValueError(f"{name} must be contiguous [pages, heads], got {tuple(t.shape)}")
  return keys, values, key_scales, value_scales


def _native_cache(tensors):
  keys, values, key_scales, value_scales = tensors
  if keys.data_ptr() % 16 or values.data_ptr() % 16:
    raise ValueError("cache keys and values must start at 16 bytes")
  return ctypes.byref(_lib.Cache(
    keys.data_ptr(), values.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(),
    *keys.shape, values.shape[3]))


def _check_pages(pages, device) -> tuple[int, int]:
  _lib._require_cuda("pages", pages, device)
  if pages.dtype != torch.int32 or pages.dim() != 2 or not pages.is_contiguous():
    raise ValueError(f"pages must be a contiguous int32 tensor [requests, pages of each], got "
                     f"{pages.dtype} {tuple(pages.shape)}")
  if pages.shape[0] > 65535:
    raise ValueError(f"at most 65535 requests per call, got {pages.shape[0]}")
  return pages.shape[0], pages.shape[1]


def _refuse_gradients(name: str, *tensors: torch.Tensor) -> None:
  if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors):
    raise ValueError(f"{name} has no backward; use attention_causal, or torch.no_grad()")


def _check_write(keys, values, cache, pages, starts, cu_seqlens):
  """Tokens, requests and pages in a row."""
  try:  # the usual call in a few expressions; whatever fails them is looked at below
    (tokens, heads, dim), (batch, width), device = keys.shape, pages.shape, keys.device
    value_dim = _usual_cache(cache, device, heads, dim)
    if (value_dim and keys.is_cuda and keys.dtype in DTYPE_CODES and values.device == device
        and values.dtype == keys.dtype and values.shape == (tokens, heads, value_dim)
        and heads == cache[0].shape[1] and keys.stride(2) == 1 and values.stride(2) == 1
        and pages.device == device and starts.device == device and cu_seqlens.device == device
        and pages.dtype == torch.int32 and starts.dtype in INDEX_CODES
        and cu_seqlens.dtype in INDEX_CODES and batch <= 65535 and tokens <= MAX_TOKENS
        and starts.shape == (batch,) and cu_seqlens.shape == (batch + 1,) and pages.is_contiguous()
        and starts.is_contiguous() and cu_seqlens.is_contiguous()):
      return tokens, batch, width
  except (AttributeError, TypeError, ValueError):
    pass
  _check_rows("keys", keys, None, None)
  device, tokens = keys.device, keys.shape[0]
  tensors = _check_cache(cache, device)
  _check_rows("keys", keys, device, None, None, tensors[0].shape[3])
  _check_rows("values", values, device, keys.dtype, tokens, tensors[1].shape[3])
  for name, t in (("keys", keys), ("values", values)):
    if t.shape[1] != tensors[0].shape[1]:
      raise ValueError(f"{name} has {t.shape[1]} heads, the cache {tensors[0].shape[1]}")
  batch, width = _check_pages(pages, device)
  _check_index("starts", starts, device, batch)
  _check_index("cu_seqlens", cu_seqlens, device, batch + 1)
  if tokens > MAX_TOKENS:
    raise ValueError(f"at most {MAX_TOKENS} tokens are supported")
  return tokens, batch, width


def attention_cache_write(
  keys: torch.Tensor,
  values: torch.Tensor,
  cache: AttentionCache,
  pages: torch.Tensor,
  starts: torch.Tensor,
  args: dict,
) -> None:
  """New tokens of B requests into their pages of the cache, in place.

  Args:
    keys: [BL, heads, Dk]; values: [BL, heads, Dv]; the requests' new tokens,
      packed; heads and sizes are the cache's.
    cache: AttentionCache, or its four tensors.
    pages: [B, width] int32; position t of request b is row ``t % page`` of page
      ``pages[b, t // page]``.  A call may write no page
      for two requests, or for two places of one.
    starts: [B] int32 or int64, tokens that the cache holds of each request: the
      position of its first new one.  Negative: no request, nothing is written.
    args: {"cu_seqlens": [B+1] int tensor}, where each request's tokens lie.
  A page's scale for a head is the smallest power of two, 2**-64 to 2**64, that
  every finite value written to it fits in; a page that is written from its
  first row on starts anew, and one that was begun is brought to a larger
  scale when a new token needs it.  Values are rounded to nearest; what is not
  finite becomes NaN.  A page outside the pool is skipped, with ScanError as
  for every device-side check.  The write counts as one of torch's in-place
  operations.  No gradients.
  """
  _refuse_gradients("attention_cache_write", keys, values)
  _refuse_tangents(ValueError, "attention_cache_write", keys, values)
  cu_seqlens = args["cu_seqlens"]
  tokens, batch, width = _check_write(keys, values, cache, pages, starts, cu_seqlens)
  device, tensors = keys.device, tuple(cache)
  _lib._enable_error_flag()
  if tokens == 0 or batch == 0:
    return
  with _on(device):
    rc = _lib.load().ascan_cache_write(
      *_rows(keys, values), _native_cache(tensors), pages.data_ptr(), batch, width,
      starts.data_ptr(), INDEX_CODES[starts.dtype], cu_seqlens.data_ptr(),
      INDEX_CODES[cu_seqlens.dtype], tokens, DTYPE_CODES[keys.dtype], _stream(device))
  # the write goes past torch: whoever saved the cache for a backward must see it
  for t in tensors:
    torch.autograd.graph.increment_version(t)
  _lib._finish(rc, "ascan_cache_write", device)


@functools.lru_cache(maxsize=256)
def _step_workspace(batch: int, value_dim: int) -> int:
  return _lib.load().ascan_cache_step_workspace(batch, value_dim)


def _check_step(queries, cache, pages, lengths):
  """Requests, heads, head size, value size and pages in a row."""
  try:  # the usual call in a few expressions; whatever fails them is looked at below
    (batch, heads, dim), (rows, width), device = queries.shape, pages.shape, queries.device
    value_dim = _usual_cache(cache, device, heads, dim)
    if (value_dim and queries.is_cuda and queries.dtype in DTYPE_CODES and 0 < heads <= 65535
        and queries.stride(2) == 1 and pages.device == device and lengths.device == device
        and pages.dtype == torch.int32 and lengths.dtype in INDEX_CODES and rows == batch <= 65535
        and lengths.shape == (batch,) and pages.is_contiguous() and lengths.is_contiguous()):
      return batch, heads, dim, value_dim, width
  except (AttributeError, TypeError, ValueError):
    pass
  _check_rows("queries", queries, None, None)
  device, (batch, heads, dim) = queries.device, queries.shape
  tensors = _check_cache(cache, device)
  (_, cache_heads, _, key_dim), value_dim = tensors[0].shape, tensors[1].shape[3]
  if dim != key_dim:
    raise ValueError(f"queries have head size {dim}, the cache {key_dim}")
  if heads % cache_heads:
    raise ValueError(f"the cache's {cache_heads} heads do not divide the queries' {heads}")
  rows, width = _check_pages(pages, device)
  if rows != batch:
    raise ValueError(f"pages has {rows} rows, expected {batch}")
  _check_index("lengths", lengths, device, batch)
  return batch, heads, dim, value_dim, width


def attention_cache_step(
  queries: torch.Tensor,
  cache: AttentionCache,
  pages: torch.Tensor,
  lengths: torch.Tensor,
  scale: float | None = None,
) -> torch.Tensor:
  """One token of attention_causal for each of B requests, over their cache.

  Args:
    queries: [B, H, Dk]; the cache's heads divide H, and query head h reads
      head h // (H // heads).
    cache, pages: as for attention_cache_write; pages may be shared.
    lengths: [B] int32 or int64, tokens of each request to attend to, the new
      one among them (write it first).  0 or less gives a zero row.
    scale: factor of the scores, positive; Dk**-0.5 by default.
  A page outside the pool, or tokens beyond the row of pages, are left out, with
  ScanError as for every device-side check.
  Returns:
    out [B, H, Dv] in the queries' type.  No gradients.
  """
  _refuse_gradients("attention_cache_step", queries)
  _refuse_tangents(ValueError, "attention_cache_step", queries)
  batch, heads, dim, value_dim, width = _check_step(queries, cache, pages, lengths)
  device, tensors = queries.device, tuple(cache)
  scale = _check_scale(scale, dim)
  _lib._enable_error_flag()
  out = torch.empty((batch, heads, value_dim), dtype=queries.dtype, device=device)
  if batch == 0:
    return out
  lib = _lib.load()
  with _on(device):
    ws = torch.empty(_step_workspace(batch, value_dim), dtype=torch.uint8, device=device)
    rc = lib.ascan_cache_step(
      *_rows(queries), _native_cache(tensors), pages.data_ptr(), batch, width, lengths.data_ptr(),
      INDEX_CODES[lengths.dtype], DTYPE_CODES[queries.dtype], scale, out.data_ptr(), ws.data_ptr(),
      ws.numel(), _stream(device))
  _lib._finish(rc, "ascan_cache_step", device)
  return out


# ---------------------------------------------------------------------------
# torch.compile-safe variants: custom ops with fake kernels and gradients
# ---------------------------------------------------------------------------


@torch.library.custom_op(f"{_NS}::attention_fwd", mutates_args=())
def attention_fwd_op(queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor,
                     cu_seqlens: torch.Tensor, scale: float
                     ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
  """attention_causal; returns (out, what its rounding left over or empty, log2 sums)."""
  out, rest, lse = _attention_forward(queries, keys, values, cu_seqlens, scale, True)
  return out, _none(rest, queries), lse


@attention_fwd_op.register_fake
def _attention_fwd_fake(queries, keys, values, cu_seqlens, scale):
  shape = (queries.shape[0], queries.shape[1], values.shape[2])
  rest = (values.new_empty(0, dtype=torch.float32) if values.dtype == torch.float32
          else values.new_empty(shape))
  return (values.new_empty(shape), rest,
          values.new_empty((queries.shape[1], queries.shape[0]), dtype=torch.float32))


@torch.library.custom_op(f"{_NS}::attention_bwd", mutates_args=())
def attention_bwd_op(queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor,
                     cu_seqlens: torch.Tensor, out: torch.Tensor, rest: torch.Tensor,
                     lse: torch.Tensor, scale: float, d_out: torch.Tensor
                     ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
  """Gradients of queries, keys and values."""
  return _attention_backward(queries, keys, values, cu_seqlens, out,
                             None if queries.dtype == torch.float32 else rest, lse, scale, d_out)


@attention_bwd_op.register_fake
def _attention_bwd_fake(queries, keys, values, cu_seqlens, out, rest, lse, scale, d_out):
  return tuple(t.new_empty(t.shape) for t in (queries, keys, values))


def _attention_setup(ctx, inputs, output) -> None:
  *tensors, ctx.scale = inputs
  ctx.save_for_backward(*tensors, *output)
  ctx.set_materialize_grads(False)


def _attention_op_backward(ctx, d_out, d_rest, d_lse):
  if d_out is None:
    return (None,) * 5
  return (*attention_bwd_op(*ctx.saved_tensors, ctx.scale, d_out), None, None)


attention_fwd_op.register_autograd(_attention_op_backward, setup_context=_attention_setup)


def attention_causal_compiled(queries, keys, values, args, scale=None):
  """attention_causal that torch.compile can trace (same arguments and results)."""
  return attention_fwd_op(queries, keys, values, args["cu_seqlens"],
                          _check_scale(scale, queries.shape[-1]))[0]


@torch.library.custom_op(f"{_NS}::attention_cache_write",
                         mutates_args=("key_cache", "value_cache", "key_scales", "value_scales"))
def attention_cache_write_op(keys: torch.Tensor, values: torch.Tensor, key_cache: torch.Tensor,
                             value_cache: torch.Tensor, key_scales: torch.Tensor,
                             value_scales: torch.Tensor, pages: torch.Tensor, starts: torch.Tensor,
                             cu_seqlens: torch.Tensor) -> None:
  """attention_cache_write."""
  attention_cache_write(keys, values, (key_cache, value_cache, key_scales, value_scales), pages,
                        starts, {"cu_seqlens": cu_seqlens})


@attention_cache_write_op.register_fake
def _attention_cache_write_fake(keys, values, key_cache, value_cache, key_scales, value_scales,
                                pages, starts, cu_seqlens):
  return None


def attention_cache_write_compiled(keys, values, cache, pages, starts, args):
  """attention_cache_write that torch.compile can trace (same arguments and results)."""
  attention_cache_write_op(keys, values, *cache, pages, starts, args["cu_seqlens"])


@torch.library.custom_op(f"{_NS}::attention_cache_step", mutates_args=())
def attention_cache_step_op(queries: torch.Tensor, key_cache: torch.Tensor,
                            value_cache: torch.Tensor, key_scales: torch.Tensor,
                            value_scales: torch.Tensor, pages: torch.Tensor, lengths: torch.Tensor,
                            scale: float) -> torch.Tensor:
  """attention_cache_step."""
  return attention_cache_step(queries, (key_cache, value_cache, key_scales, value_scales), pages,
                              lengths, scale)


@attention_cache_step_op.register_fake
def _attention_cache_step_fake(queries, key_cache, value_cache, key_scales, value_scales, pages,
                               lengths, scale):
  return queries.new_empty((queries.shape[0], queries.shape[1], value_cache.shape[3]))


def attention_cache_step_compiled(queries, cache, pages, lengths, scale=None):
  """attention_cache_step that torch.compile can trace (same arguments and results)."""
  return attention_cache_step_op(queries, *cache, pages, lengths,
                                 _check_scale(scale, queries.shape[-1]))
