"""The operators of a gated linear-attention layer.

* :func:`matrix_scan_causal`: the recurrence with a matrix state per head,
  ``S[t] = exp(g[t]) S[t-1] + k[t] v[t]^T``, ``o[t] = scale q[t] S[t]``, over
  packed sequences, with gradients for every input.
* :func:`matrix_scan_step`: its form for one new token of many requests, over
  a pool of states.
* :func:`qk_norm_rotate`: RMS norm of every query and key head, weight and
  rotation by position in one pass, with gradients.

Tokens are rows here: a tensor is ``[BL, heads, dim]`` (all sequences packed
along the first axis, ``args["cu_seqlens"]`` as for the other scans), its last
dimension has unit stride, and token and head strides are free, so views of a
packed projection need no copy.  float32, float16 and bfloat16; states, sums
and norms are float32.  Every call runs on torch's current stream and takes
its workspace from torch's allocator.  No forward-mode derivatives.

Precision: float32 and float16 inputs are computed in float32.  bfloat16
inputs (head sizes a multiple of 8, 16-byte aligned rows) run on tensor cores:
what is computed on the way to a product keeps 16 bits, so that a bfloat16
result carries its own rounding only; what enters a state keeps 24 where a
float32 result depends on it, and final states and initial states' gradients
are as good as float32 arithmetic's.  Float32 gate gradients are within
1e-5 of their norm (3e-6 at the median).
"""

from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import DTYPE_CODES, INDEX_CODES

MAX_DIM = 128  # of a matrix state's sides

MAX_AXES = 4  # of positions

_ROWS = {n: ctypes.c_int64 * (4 * n) for n in (1, 2, 3, 4)}


def _rows(*tensors: torch.Tensor):
  """``ascan_rows`` of [tokens, heads, dim] or [tokens, heads] tensors, one pointer each.

  One array holds them all (pointer, two strides, heads: four words), which
  costs a call less than a structure for each.
  """
  words = []
  for t in tensors:
    st = t.stride()
    words += (t.data_ptr(), st[0], st[1], t.shape[1])
  block = _ROWS[len(tensors)](*words)
  return [ctypes.byref(block, 32 * i) for i in range(len(tensors))]


def _like(t: torch.Tensor) -> torch.Tensor:
  """Uninitialised, contiguous, of the same shape, type and device."""
  return torch.empty_like(t, memory_format=torch.contiguous_format)


@functools.lru_cache(maxsize=256)
def _scan_workspace(*sizes: int) -> int:
  return _lib.load().ascan_matrix_scan_workspace_of(*sizes)


@functools.lru_cache(maxsize=256)
def _rotate_workspace(*sizes: int) -> int:
  return _lib.load().ascan_qk_norm_rotate_workspace(*sizes)


def _stream(device: torch.device) -> int:
  return torch._C._cuda_getCurrentRawStream(device.index)


def _ptr(t: torch.Tensor | None):
  return None if t is None else t.data_ptr()


def _check_rows(name: str, t: torch.Tensor, device, dtype, tokens=None, dim=None, dims=3) -> None:
  _lib._require_cuda(name, t, device)
  if t.dim() != dims:
    raise ValueError(f"{name} must have {dims} dimensions, got shape {tuple(t.shape)}")
  if dtype is not None and t.dtype != dtype:
    raise TypeError(f"{name} has dtype {t.dtype}, expected {dtype}")
  if t.dtype not in DTYPE_CODES:
    raise TypeError(f"unsupported dtype {t.dtype}; use float32, float16 or bfloat16")
  if tokens is not None and t.shape[0] != tokens:
    raise ValueError(f"{name} has {t.shape[0]} rows, expected {tokens}")
  if t.shape[1] < 1 or t.shape[1] > 65535:
    raise ValueError(f"{name} must have between 1 and 65535 heads, got {t.shape[1]}")
  if dims == 3:
    if dim is not None and t.shape[2] != dim:
      raise ValueError(f"{name} has head size {t.shape[2]}, expected {dim}")
    if t.shape[2] < 1:
      raise ValueError(f"{name} has an empty head")
    if t.shape[2] > 1 and t.stride(2) != 1:
      raise ValueError(f"{name} must have unit stride along its last dimension")


def _check_index(name: str, t: torch.Tensor, device, entries=None) -> None:
  _lib._require_cuda(name, t, device)
  if t.dtype not in INDEX_CODES:
    raise TypeError(f"{name} must be int32 or int64, got {t.dtype}")
  if t.dim() != 1 or not t.is_contiguous():
    raise ValueError(f"{name} must be contiguous with one dimension")
  if entries is not None and t.numel() != entries:
    raise ValueError(f"{name} has {t.numel()} entries, expected {entries}")


def _check_state(name: str, t: torch.Tensor, device, shape) -> None:
  _lib._require_cuda(name, t, device)
  if t.dtype != torch.float32:
    raise TypeError(f"{name} must be float32, got {t.dtype}")
  if tuple(t.shape) != tuple(shape):
    raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
  if not t.is_contiguous():
    raise ValueError(f"{name} must be contiguous")


def _check_operands(queries, keys, values, log_gates, max_dim):
  """Checks the four inputs; returns (device, tokens, heads, key_dim, value_dim)."""
  try:  # the usual call in one expression; whatever fails it is looked at below
    (n, hq, dk), (nk, hk, dkk), (nv, hv, dv), (ng, hg) = (queries.shape, keys.shape, values.shape,
                                                         log_gates.shape)
    device, dtype, gate_dtype = queries.device, queries.dtype, log_gates.dtype
    heads = max(hq, hk, hv, hg)
    if (queries.is_cuda and keys.device == device and values.device == device
        and log_gates.device == device and dtype in DTYPE_CODES and keys.dtype == dtype
        and values.dtype == dtype and (gate_dtype == torch.float32 or gate_dtype == dtype)
        and nk == n and nv == n and ng == n and dkk == dk and dk > 1 and dv > 1
        and (max_dim is None or (dk <= max_dim and dv <= max_dim)) and heads <= 65535
        and hq > 0 and hk > 0 and hv > 0 and hg > 0
        and not (heads % hq or heads % hk or heads % hv or heads % hg)
        and queries.stride(2) == 1 and keys.stride(2) == 1 and values.stride(2) == 1):
      return device, n, heads, dk, dv
  except (AttributeError, TypeError, ValueError):
    pass
  _check_rows("queries", queries, None, None)
  device, tokens, key_dim = queries.device, queries.shape[0], queries.shape[2]
  _check_rows("keys", keys, device, queries.dtype, tokens, key_dim)
  _check_rows("values", values, device, queries.dtype, tokens)
  _check_rows("log_gates", log_gates, device, None, tokens, dims=2)
  if log_gates.dtype not in (torch.float32, queries.dtype):
    raise TypeError(f"log_gates must be float32 or {queries.dtype}, got {log_gates.dtype}")
  value_dim = values.shape[2]
  if max_dim is not None and max(key_dim, value_dim) > max_dim:
    raise ValueError(f"head sizes up to {max_dim} are supported, got {key_dim} and {value_dim}")
  shapes = {"queries": queries, "keys": keys, "values": values, "log_gates": log_gates}
  heads = max(t.shape[1] for t in shapes.values())
  for name, t in shapes.items():
    if heads % t.shape[1]:
      raise ValueError(f"{name} has {t.shape[1]} heads, which do not divide {heads}")
  return device, tokens, heads, key_dim, value_dim


def _refuse_tangents(error: type, name: str, *tensors: torch.Tensor | None) -> None:
  """Forward-mode derivatives: the native call would drop the tangents without a word."""
  if forward_ad._current_level >= 0:
    for t in tensors:
      if t is not None and forward_ad.unpack_dual(t).tangent is not None:
        raise error(f"{name} has no derivatives in forward mode, and an input has a tangent")


class _on:
  """Makes ``device`` current for a launch; free when it is already."""

  __slots__ = ("guard",)

  def __init__(self, device):
    self.guard = None if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)

  def __enter__(self):
    if self.guard is not None:
      self.guard.__enter__()

  def __exit__(self, *exc):
    if self.guard is not None:
      self.guard.__exit__(*exc)


# ---------------------------------------------------------------------------
# the recurrence over packed sequences
# ---------------------------------------------------------------------------


def _scan_forward(queries, keys, values, log_gates, cu_seqlens, scale, initial_state, want_final):
  _refuse_tangents(NotImplementedError, "matrix_scan_causal", queries, keys, values, log_gates, initial_state)
  device, tokens, heads, key_dim, value_dim = _check_operands(queries, keys, values, log_gates,
                                                              MAX_DIM)
  _check_index("cu_seqlens", cu_seqlens, device)
  num_seq = cu_seqlens.numel() - 1
  if num_seq < 0:
    raise ValueError("cu_seqlens must have at least one entry")
  state_shape = (num_seq, heads, key_dim, value_dim)
  if initial_state is not None:
    _check_state("initial_state", initial_state, device, state_shape)
  _lib._enable_error_flag()
  if tokens == 0 or num_seq == 0:
    out = values.new_zeros(tokens, heads, value_dim)
    final = None
    if want_final:
      final = (initial_state.clone() if initial_state is not None
               else torch.zeros(state_shape, dtype=torch.float32, device=device))
    return out, final
  out = torch.empty((tokens, heads, value_dim), dtype=values.dtype, device=device)
  final = torch.empty(state_shape, dtype=torch.float32, device=device) if want_final else None
  lib = _lib.load()
  with _on(device):
    ws = torch.empty(
      _scan_workspace(tokens, num_seq, heads, queries.shape[1], keys.shape[1], values.shape[1],
                      log_gates.shape[1], key_dim, value_dim, DTYPE_CODES[queries.dtype],
                      DTYPE_CODES[log_gates.dtype], 0),
      dtype=torch.uint8, device=device)
    rc = lib.ascan_matrix_scan_forward(
      *_rows(queries, keys, values, log_gates), DTYPE_CODES[log_gates.dtype],
      cu_seqlens.data_ptr(), INDEX_CODES[cu_seqlens.dtype], num_seq, tokens, heads, key_dim,
      value_dim, DTYPE_CODES[queries.dtype], scale, _ptr(initial_state), out.data_ptr(),
      _ptr(final), ws.data_ptr(), ws.numel(), _stream(device))
  _lib._finish(rc, "ascan_matrix_scan_forward", device)
  return out, final


def _scan_backward(queries, keys, values, log_gates, cu_seqlens, scale, initial_state, final_state,
                   d_out, d_final):
  device, tokens, heads, key_dim, value_dim = _check_operands(queries, keys, values, log_gates,
                                                              MAX_DIM)
  num_seq = cu_seqlens.numel() - 1
  d_queries, d_keys, d_values, d_gates = (_like(queries), _like(keys), _like(values),
                                          _like(log_gates))
  d_initial = torch.empty_like(initial_state) if initial_state is not None else None
  if tokens == 0 or num_seq == 0:
    for t in (d_queries, d_keys, d_values, d_gates):
      t.zero_()
    if d_initial is not None:
      d_initial.zero_() if d_final is None else d_initial.copy_(d_final)
    return d_queries, d_keys, d_values, d_gates, d_initial
  if d_out is None:
    d_out = torch.zeros((tokens, heads, value_dim), dtype=values.dtype, device=device)
  elif d_out.stride(2) != 1 and value_dim > 1:
    d_out = d_out.contiguous()
  if d_final is not None:
    d_final = d_final.contiguous()
  lib = _lib.load()
  with _on(device):
    ws = torch.empty(
      _scan_workspace(tokens, num_seq, heads, queries.shape[1], keys.shape[1], values.shape[1],
                      log_gates.shape[1], key_dim, value_dim, DTYPE_CODES[queries.dtype],
                      DTYPE_CODES[log_gates.dtype], 1),
      dtype=torch.uint8, device=device)
    rc = lib.ascan_matrix_scan_backward(
      *_rows(queries, keys, values, log_gates), DTYPE_CODES[log_gates.dtype],
      *_rows(d_out, d_out)[:1], _ptr(initial_state), _ptr(final_state), _ptr(d_final), cu_seqlens.data_ptr(),
      INDEX_CODES[cu_seqlens.dtype], num_seq, tokens, heads, key_dim, value_dim,
      DTYPE_CODES[queries.dtype], scale, d_queries.data_ptr(), d_keys.data_ptr(),
      d_values.data_ptr(), d_gates.data_ptr(), _ptr(d_initial), ws.data_ptr(), ws.numel(),
      _stream(device))
  _lib._finish(rc, "ascan_matrix_scan_backward", device)
  return d_queries, d_keys, d_values, d_gates, d_initial


class MatrixScanCausal(torch.autograd.Function):
  """matrix_scan_causal with its gradients."""

  @staticmethod
  def forward(ctx, queries, keys, values, log_gates, cu_seqlens, scale, initial_state, want_final):
    out, final = _scan_forward(queries, keys, values, log_gates, cu_seqlens, scale, initial_state,
                               want_final)
    ctx.save_for_backward(queries, keys, values, log_gates, cu_seqlens, initial_state, final)
    ctx.scale = scale
    ctx.set_materialize_grads(False)
    return out, final

  @staticmethod
  @torch.autograd.function.once_differentiable
  def backward(ctx, d_out, d_final):
    if d_out is None and d_final is None:
      return (None,) * 8
    queries, keys, values, log_gates, cu_seqlens, initial_state, final = ctx.saved_tensors
    d_queries, d_keys, d_values, d_gates, d_initial = _scan_backward(
      queries, keys, values, log_gates, cu_seqlens, ctx.scale, initial_state, final, d_out, d_final)
    return d_queries, d_keys, d_values, d_gates, None, None, d_initial, None


def matrix_scan_causal(
  queries: torch.Tensor,
  keys: torch.Tensor,
  values: torch.Tensor,
  log_gates: torch.Tensor,
  args: dict,
  scale: float | None = None,
  initial_state: torch.Tensor | None = None,
  return_final_state: bool = False,
):
  """Causal scan with a matrix state per head, over packed sequences.

  ``S[t] = exp(log_gates[t]) S[t-1] + keys[t] values[t]^T`` and
  ``out[t] = scale * queries[t] S[t]``, started anew (or from
  ``initial_state``) at every sequence.

  Args:
    queries, keys: [BL, heads, Dk]; values: [BL, heads, Dv]; Dk, Dv <= 128.
    log_gates: [BL, heads], float32 or the tokens' type; -inf drops the state.
    args: {"cu_seqlens": [N+1] int tensor}; other entries are not used.
    scale: factor of the outputs, Dk**-0.5 by default.
    initial_state: [N, H, Dk, Dv] float32 before each sequence; zero if None.
    return_final_state: also return the float32 state after each sequence.
  Errors (the module's docstring has the reasons): one rounding of 16-bit
  results; about 1e-6 of the norm of float32 ones, 1e-5 of that of float32
  log_gates' gradients.
  Head counts may differ: H is the largest, the others divide it, and head h
  reads head h // (H // heads) of each input; shared heads get the summed
  gradient.  Tokens of no sequence give zero rows.
  Returns:
    out [BL, H, Dv], or (out, final_state).
  """
  scale = float(queries.shape[-1]) ** -0.5 if scale is None else float(scale)
  cu_seqlens = args["cu_seqlens"]
  if torch.is_grad_enabled() and (queries.requires_grad or keys.requires_grad
                                  or values.requires_grad or log_gates.requires_grad
                                  or (initial_state is not None and initial_state.requires_grad)):
    out, final = MatrixScanCausal.apply(queries, keys, values, log_gates, cu_seqlens, scale,
                                        initial_state, bool(return_final_state))
  else:
    out, final = _scan_forward(queries, keys, values, log_gates, cu_seqlens, scale, initial_state,
                               bool(return_final_state))
  return (out, final) if return_final_state else out


# ---------------------------------------------------------------------------
# one token
# ---------------------------------------------------------------------------


def _state_ptr(state: torch.Tensor, any_other: torch.Tensor) -> int:
  """A pool of no states has no address, and none of it is read: every slot lies outside."""
  return state.data_ptr() or any_other.data_ptr()


def matrix_scan_step(
  queries: torch.Tensor,
  keys: torch.Tensor,
  values: torch.Tensor,
  log_gates: torch.Tensor,
  state: torch.Tensor,
  slots: torch.Tensor | None = None,
  scale: float | None = None,
  state_out: torch.Tensor | None = None,
) -> torch.Tensor:
  """One step of matrix_scan_causal for each of B requests.

  Args:
    queries, keys: [B, heads, Dk]; values: [B, heads, Dv]; log_gates: [B, heads].
    state: [S, H, Dk, Dv] float32, a pool of states; updated in place unless
      ``state_out`` (same shape) receives the new states instead.  The write
      counts as one of torch's in-place operations: a backward that saved the
      tensor raises.
    slots: [B] int32, each request's state in the pool (no two alike); row b
      itself if None.  A negative slot marks a row without a request: its
      output is zero and no state is touched.
  Returns:
    out [B, H, Dv].  No gradients: call it under ``torch.no_grad()`` when an
    input requires them.
  """
  device, batch, heads, key_dim, value_dim = _check_operands(queries, keys, values, log_gates, None)
  if torch.is_grad_enabled() and (queries.requires_grad or keys.requires_grad
                                  or values.requires_grad or log_gates.requires_grad
                                  or state.requires_grad):
    raise ValueError("matrix_scan_step has no backward; use matrix_scan_causal, or torch.no_grad()")
  _refuse_tangents(ValueError, "matrix_scan_step", queries, keys, values, log_gates, state, state_out)
  if batch > 65535:
    raise ValueError(f"at most 65535 requests per call, got {batch}")
  _check_state("state", state, device, (*state.shape[:1], heads, key_dim, value_dim))
  if state_out is None:
    state_out = state
  elif state_out is not state:
    _check_state("state_out", state_out, device, state.shape)
    if (state_out.data_ptr() != state.data_ptr()
        and abs(state_out.data_ptr() - state.data_ptr()) < 4 * state.numel()):
      raise ValueError("state_out overlaps state; pass the same tensor or a separate one")
  if slots is not None:
    _lib._require_cuda("slots", slots, device)
    if slots.dtype != torch.int32 or slots.shape != (batch,) or not slots.is_contiguous():
      raise ValueError(f"slots must be a contiguous int32 tensor of {batch} entries")
  elif batch > state.shape[0]:
    raise ValueError(f"{batch} requests need {batch} states, the pool has {state.shape[0]}")
  _lib._enable_error_flag()
  out = torch.empty((batch, heads, value_dim), dtype=values.dtype, device=device)
  if batch == 0:
    return out
  scale = float(key_dim) ** -0.5 if scale is None else float(scale)
  with _on(device):
    rc = _lib.load().ascan_matrix_scan_step(
      *_rows(queries, keys, values, log_gates), DTYPE_CODES[log_gates.dtype],
      _ptr(slots), batch, state.shape[0], heads, key_dim, value_dim, DTYPE_CODES[queries.dtype],
      scale, _state_ptr(state, out), _state_ptr(state_out, out), out.data_ptr(), _stream(device))
  # the write goes past torch: a scan that saved this state must refuse its backward
  torch.autograd.graph.increment_version(state_out)
  _lib._finish(rc, "ascan_matrix_scan_step", device)
  return out


# ---------------------------------------------------------------------------
# norm and rotation of queries and keys
# ---------------------------------------------------------------------------


def _rotate_common(queries, keys, query_weight, key_weight, cos, sin, positions, cu_seqlens, eps,
                   interleaved, sections):
  """The leading arguments that the two native calls share, by name of their place."""
  index = positions if positions is not None else cu_seqlens
  return (*_rows(queries, keys), query_weight.data_ptr(), key_weight.data_ptr(),
          DTYPE_CODES[query_weight.dtype], cos.data_ptr(), sin.data_ptr(), cos.shape[0],
          cos.shape[1], int(interleaved), _ptr(positions),
          None if positions is not None else cu_seqlens.data_ptr(), INDEX_CODES[index.dtype],
          0 if positions is not None else cu_seqlens.numel() - 1, queries.shape[0],
          queries.shape[2], DTYPE_CODES[queries.dtype], eps, 1 if sections is None else len(sections),
          None if sections is None else (ctypes.c_int32 * len(sections))(*sections))


def _check_sections(sections, positions, half: int, tokens: int) -> None:
  if positions is None:
    raise ValueError("sections need positions, one row of them for each")
  if not 1 <= len(sections) <= MAX_AXES:
    raise ValueError(f"between 1 and {MAX_AXES} sections are supported, got {len(sections)}")
  if min(sections) < 0 or sum(sections) != half:
    raise ValueError(f"sections {tuple(sections)} do not add up to the tables' {half} columns")
  if positions.dim() != 2 or positions.shape != (len(sections), tokens) or not positions.is_contiguous():
    raise ValueError(f"positions must be contiguous [{len(sections)}, {tokens}], a row for each "
                     f"section, got {tuple(positions.shape)}")


def _check_rotate(queries, keys, query_weight, key_weight, cos, sin, positions, cu_seqlens,
                  sections=None):
  if sections is not None:  # then the rest is as with the first axis alone
    for name, t in (("queries", queries), ("cos", cos), ("positions", positions)):
      if t is not None:
        _lib._require_cuda(name, t, None)
    if cos.dim() == 2 and queries.dim() == 3:  # else refused below
      _check_sections(sections, positions, cos.shape[1], queries.shape[0])
      positions = positions[0]
  try:  # the usual call in one expression; whatever fails it is looked at below
    (n, hq, d), (nk, hk, dk), (rows, half) = queries.shape, keys.shape, cos.shape
    device, dtype, wtype = queries.device, queries.dtype, query_weight.dtype
    index = positions if cu_seqlens is None else cu_seqlens
    if (queries.is_cuda and keys.device == device and query_weight.device == device
        and key_weight.device == device and cos.device == device and sin.device == device
        and index.device == device and (positions is None) != (cu_seqlens is None)
        and dtype in DTYPE_CODES and keys.dtype == dtype and key_weight.dtype == wtype
        and (wtype == torch.float32 or wtype == dtype) and cos.dtype == torch.float32
        and sin.dtype == torch.float32 and index.dtype in INDEX_CODES and nk == n and dk == d
        and d > 1 and 0 < hq <= 65535 and 0 < hk <= 65535 and 2 * half <= d
        and query_weight.shape == (d,) and key_weight.shape == (d,) and sin.shape == (rows, half)
        and index.dim() == 1 and (index.shape[0] == n if cu_seqlens is None else index.shape[0] > 0)
        and queries.stride(2) == 1 and keys.stride(2) == 1 and index.is_contiguous()
        and query_weight.is_contiguous() and key_weight.is_contiguous() and cos.is_contiguous()
        and sin.is_contiguous()):
      return _lib._enable_error_flag()
  except (AttributeError, TypeError, ValueError):
    pass
  _check_rows("queries", queries, None, None)
  device, tokens, dim = queries.device, queries.shape[0], queries.shape[2]
  _check_rows("keys", keys, device, queries.dtype, tokens, dim)
  for name, w in (("query_weight", query_weight), ("key_weight", key_weight)):
    _lib._require_cuda(name, w, device)
    if w.dtype not in (torch.float32, queries.dtype) or w.dtype != query_weight.dtype:
      raise TypeError(f"both weights must be float32 or both {queries.dtype}, got {w.dtype}")
    if w.shape != (dim,) or not w.is_contiguous():
      raise ValueError(f"{name} must be contiguous with {dim} entries, got {tuple(w.shape)}")
  for name, t in (("cos", cos), ("sin", sin)):
    _lib._require_cuda(name, t, device)
    if t.dtype != torch.float32:
      raise TypeError(f"{name} must be float32, got {t.dtype}")
    if t.dim() != 2 or not t.is_contiguous() or t.shape != cos.shape or 2 * t.shape[1] > dim:
      raise ValueError(f"{name} must be contiguous [positions, half] with half <= {dim // 2}, "
                       f"both tables alike, got {tuple(t.shape)}")
  if (positions is None) == (cu_seqlens is None):
    raise ValueError("give either positions or args with cu_seqlens")
  if positions is not None:
    _check_index("positions", positions, device, tokens)
  else:
    _check_index("cu_seqlens", cu_seqlens, device)
    if cu_seqlens.numel() < 1:
      raise ValueError("cu_seqlens must have at least one entry")
  _lib._enable_error_flag()


def _rotate_forward(queries, keys, query_weight, key_weight, cos, sin, positions, cu_seqlens, eps,
                    interleaved, sections=None):
  _refuse_tangents(NotImplementedError, "qk_norm_rotate", queries, keys, query_weight, key_weight, cos, sin)
  _check_rotate(queries, keys, query_weight, key_weight, cos, sin, positions, cu_seqlens, sections)
  device = queries.device
  out_q, out_k = _like(queries), _like(keys)
  if queries.shape[0] == 0:
    return out_q, out_k
  with _on(device):
    rc = _lib.load().ascan_qk_norm_rotate_axes(
      *_rotate_common(queries, keys, query_weight, key_weight, cos, sin, positions, cu_seqlens,
                      eps, interleaved, sections),
      out_q.data_ptr(), out_k.data_ptr(), _stream(device))
  _lib._finish(rc, "ascan_qk_norm_rotate", device)
  return out_q, out_k


def _rotate_backward(queries, keys, query_weight, key_weight, cos, sin, positions, cu_seqlens, eps,
                     interleaved, d_out_q, d_out_k, sections=None):
  device, tokens = queries.device, queries.shape[0]
  d_q, d_k = _like(queries), _like(keys)
  d_qw, d_kw = torch.empty_like(query_weight), torch.empty_like(key_weight)
  if tokens == 0:
    return d_q, d_k, d_qw.zero_(), d_kw.zero_()
  grads = []
  for d, out in ((d_out_q, d_q), (d_out_k, d_k)):
    if d is None:
      d = torch.zeros_like(out)
    grads.append(d if d.stride(2) == 1 or d.shape[2] == 1 else d.contiguous())
  lib = _lib.load()
  with _on(device):
    ws = torch.empty(
      _rotate_workspace(tokens, queries.shape[1], keys.shape[1],
                                         queries.shape[2]), dtype=torch.uint8, device=device)
    rc = lib.ascan_qk_norm_rotate_axes_backward(
      *_rotate_common(queries, keys, query_weight, key_weight, cos, sin, positions, cu_seqlens,
                      eps, interleaved, sections),
      *_rows(grads[0], grads[1]), d_q.data_ptr(), d_k.data_ptr(), d_qw.data_ptr(),
      d_kw.data_ptr(), ws.data_ptr(), ws.numel(), _stream(device))
  _lib._finish(rc, "ascan_qk_norm_rotate_backward", device)
  return d_q, d_k, d_qw, d_kw


class QkNormRotate(torch.autograd.Function):
  """qk_norm_rotate with its gradients."""

  @staticmethod
  def forward(ctx, queries, keys, query_weight, key_weight, cos, sin, positions, cu_seqlens, eps,
              interleaved, sections=None):
    # with the tables and positions: changed in place before the backward, it must raise
    ctx.save_for_backward(queries, keys, query_weight, key_weight, cos, sin, positions, cu_seqlens)
    ctx.eps, ctx.interleaved, ctx.sections = eps, interleaved, sections
    ctx.set_materialize_grads(False)
    return _rotate_forward(queries, keys, query_weight, key_weight, cos, sin, positions, cu_seqlens,
                           eps, interleaved, sections)

  @staticmethod
  @torch.autograd.function.once_differentiable
  def backward(ctx, d_q, d_k):
    if d_q is None and d_k is None:
      return (None,) * 11
    return (*_rotate_backward(*ctx.saved_tensors, ctx.eps, ctx.interleaved, d_q, d_k, ctx.sections),
            *(None,) * 7)


def qk_norm_rotate(
  queries: torch.Tensor,
  keys: torch.Tensor,
  query_weight: torch.Tensor,
  key_weight: torch.Tensor,
  cos: torch.Tensor,
  sin: torch.Tensor,
  args: dict | None = None,
  positions: torch.Tensor | None = None,
  eps: float = 1e-6,
  interleaved: bool = False,
  sections: tuple[int, ...] | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
  """RMS norm per head, weight and rotation of queries and keys, in one pass.

  ``n = x * rsqrt(mean(x^2) + eps) * weight``; then the first ``2 * half``
  elements of each head turn by the token's angles, in pairs ``(i, i + half)``
  or, when ``interleaved``, ``(2i, 2i + 1)``:
  ``(n[i] cos - n[j] sin, n[j] cos + n[i] sin)``.

  Args:
    queries: [BL, Hq, D]; keys: [BL, Hk, D].
    query_weight, key_weight: [D], float32 or the tokens' type.
    cos, sin: [positions, half] float32, half <= D / 2; constants, without
      gradients.
    args: {"cu_seqlens": ...}: a token's position is its place in its
      sequence, and tokens of no sequence give zero rows; or
    positions: [BL] int32 or int64, every token's row of the tables (outside
      them: a zero row, and ScanError as for every device-side check).
    sections: with positions [axes, BL] (axes <= 4, as of time, height and
      width): how many of the half pairs turn by each axis, the first ones by
      the first.  A pair keeps its column of the tables; a token with any
      position outside them gives a zero row.
  Returns:
    queries and keys, contiguous, in their type.
  """
  cu_seqlens = None if args is None else args["cu_seqlens"]
  sections = None if sections is None else tuple(int(n) for n in sections)
  if torch.is_grad_enabled() and (cos.requires_grad or sin.requires_grad):
    raise ValueError("cos and sin get no gradient; detach them")
  if torch.is_grad_enabled() and (queries.requires_grad or keys.requires_grad
                                  or query_weight.requires_grad or key_weight.requires_grad):
    return QkNormRotate.apply(queries, keys, query_weight, key_weight, cos, sin, positions,
                              cu_seqlens, float(eps), bool(interleaved), sections)
  return _rotate_forward(queries, keys, query_weight, key_weight, cos, sin, positions, cu_seqlens,
                         float(eps), bool(interleaved), sections)


# ---------------------------------------------------------------------------
# torch.compile-safe variants: custom ops with fake kernels and gradients
# ---------------------------------------------------------------------------

_NS = "associative_scan_triton"


def _none(t: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
  """An op returns tensors only: what is not asked for comes out empty."""
  return t if t is not None else like.new_empty(0, dtype=torch.float32)


@torch.library.custom_op(f"{_NS}::matrix_scan_fwd", mutates_args=())
def matrix_scan_fwd_op(queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor,
                       log_gates: torch.Tensor, cu_seqlens: torch.Tensor, scale: float,
                       initial_state: torch.Tensor | None) -> tuple[torch.Tensor, torch.Tensor]:
  """matrix_scan_causal; returns (out, final_state)."""
  return _scan_forward(queries, keys, values, log_gates, cu_seqlens, scale, initial_state, True)


@matrix_scan_fwd_op.register_fake
def _matrix_scan_fwd_fake(queries, keys, values, log_gates, cu_seqlens, scale, initial_state):
  heads = max(t.shape[1] for t in (queries, keys, values, log_gates))
  return (values.new_empty(values.shape[0], heads, values.shape[2]),
          values.new_empty((cu_seqlens.shape[0] - 1, heads, queries.shape[2], values.shape[2]),
                           dtype=torch.float32))


@torch.library.custom_op(f"{_NS}::matrix_scan_bwd", mutates_args=())
def matrix_scan_bwd_op(
  queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, log_gates: torch.Tensor,
  cu_seqlens: torch.Tensor, scale: float, initial_state: torch.Tensor | None,
  final_state: torch.Tensor, d_out: torch.Tensor | None, d_final: torch.Tensor | None
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
  """Gradients of queries, keys, values, log_gates and (empty without one) initial_state."""
  *grads, d_initial = _scan_backward(queries, keys, values, log_gates, cu_seqlens, scale,
                                     initial_state, final_state, d_out, d_final)
  return (*grads, _none(d_initial, queries))


@matrix_scan_bwd_op.register_fake
def _matrix_scan_bwd_fake(queries, keys, values, log_gates, cu_seqlens, scale, initial_state,
                          final_state, d_out, d_final):
  grads = tuple(t.new_empty(t.shape) for t in (queries, keys, values, log_gates))
  d_initial = queries.new_empty(0 if initial_state is None else initial_state.shape,
                                dtype=torch.float32)
  return (*grads, d_initial)


def _matrix_scan_setup(ctx, inputs, output) -> None:
  queries, keys, values, log_gates, cu_seqlens, scale, initial_state = inputs
  ctx.save_for_backward(queries, keys, values, log_gates, cu_seqlens, initial_state, output[1])
  ctx.scale = scale
  ctx.set_materialize_grads(False)


def _matrix_scan_backward(ctx, d_out, d_final):
  queries, keys, values, log_gates, cu_seqlens, initial_state, final = ctx.saved_tensors
  if d_out is None and d_final is None:
    return (None,) * 7
  *grads, d_initial = matrix_scan_bwd_op(queries, keys, values, log_gates, cu_seqlens, ctx.scale,
                                         initial_state, final, d_out, d_final)
  return (*grads, None, None, d_initial if initial_state is not None else None)


matrix_scan_fwd_op.register_autograd(_matrix_scan_backward, setup_context=_matrix_scan_setup)


def matrix_scan_causal_compiled(queries, keys, values, log_gates, args, scale=None,
                                initial_state=None, return_final_state=False):
  """matrix_scan_causal that torch.compile can trace (same arguments and results)."""
  scale = float(queries.shape[-1]) ** -0.5 if scale is None else float(scale)
  out, final = matrix_scan_fwd_op(queries, keys, values, log_gates, args["cu_seqlens"], scale,
                                  initial_state)
  return (out, final) if return_final_state else out


@torch.library.custom_op(f"{_NS}::matrix_scan_step", mutates_args=("state",))
def matrix_scan_step_op(queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor,
                        log_gates: torch.Tensor, state: torch.Tensor, slots: torch.Tensor | None,
                        scale: float) -> torch.Tensor:
  """matrix_scan_step in place."""
  return matrix_scan_step(queries, keys, values, log_gates, state, slots=slots, scale=scale)


@matrix_scan_step_op.register_fake
def _matrix_scan_step_fake(queries, keys, values, log_gates, state, slots, scale):
  return values.new_empty(values.shape[0], state.shape[1], values.shape[2])


def matrix_scan_step_compiled(queries, keys, values, log_gates, state, slots=None, scale=None):
  """matrix_scan_step, in place, that torch.compile can trace."""
  scale = float(queries.shape[-1]) ** -0.5 if scale is None else float(scale)
  return matrix_scan_step_op(queries, keys, values, log_gates, state, slots, scale)


@torch.library.custom_op(f"{_NS}::qk_norm_rotate_fwd", mutates_args=())
def qk_norm_rotate_fwd_op(queries: torch.Tensor, keys: torch.Tensor, query_weight: torch.Tensor,
                          key_weight: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                          positions: torch.Tensor | None, cu_seqlens: torch.Tensor | None,
                          eps: float, interleaved: bool, sections: list[int] | None = None
                          ) -> tuple[torch.Tensor, torch.Tensor]:
  """qk_norm_rotate."""
  return _rotate_forward(queries, keys, query_weight, key_weight, cos, sin, positions, cu_seqlens,
                         eps, interleaved, sections)


@qk_norm_rotate_fwd_op.register_fake
def _qk_norm_rotate_fwd_fake(queries, keys, query_weight, key_weight, cos, sin, positions,
                             cu_seqlens, eps, interleaved, sections=None):
  return queries.new_empty(queries.shape), keys.new_empty(keys.shape)


@torch.library.custom_op(f"{_NS}::qk_norm_rotate_bwd", mutates_args=())
def qk_norm_rotate_bwd_op(
  queries: torch.Tensor, keys: torch.Tensor, query_weight: torch.Tensor, key_weight: torch.Tensor,
  cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor | None,
  cu_seqlens: torch.Tensor | None, eps: float, interleaved: bool, d_queries: torch.Tensor | None,
  d_keys: torch.Tensor | None, sections: list[int] | None = None
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
  """Gradients of queries, keys and the two weights."""
  return _rotate_backward(queries, keys, query_weight, key_weight, cos, sin, positions, cu_seqlens,
                          eps, interleaved, d_queries, d_keys, sections)


@qk_norm_rotate_bwd_op.register_fake
def _qk_norm_rotate_bwd_fake(queries, keys, query_weight, key_weight, cos, sin, positions,
                             cu_seqlens, eps, interleaved, d_queries, d_keys, sections=None):
  return tuple(t.new_empty(t.shape) for t in (queries, keys, query_weight, key_weight))


def _qk_norm_rotate_setup(ctx, inputs, output) -> None:
  *tensors, ctx.eps, ctx.interleaved, ctx.sections = inputs
  ctx.save_for_backward(*tensors)
  ctx.set_materialize_grads(False)


def _qk_norm_rotate_backward(ctx, d_queries, d_keys):
  if d_queries is None and d_keys is None:
    return (None,) * 11
  return (*qk_norm_rotate_bwd_op(*ctx.saved_tensors, ctx.eps, ctx.interleaved, d_queries, d_keys,
                                 ctx.sections), *(None,) * 7)


qk_norm_rotate_fwd_op.register_autograd(_qk_norm_rotate_backward,
                                        setup_context=_qk_norm_rotate_setup)


def qk_norm_rotate_compiled(queries, keys, query_weight, key_weight, cos, sin, args=None,
                            positions=None, eps=1e-6, interleaved=False, sections=None):
  """qk_norm_rotate that torch.compile can trace (same arguments and results)."""
  if torch.is_grad_enabled() and (cos.requires_grad or sin.requires_grad):
    raise ValueError("cos and sin get no gradient; detach them")
  return qk_norm_rotate_fwd_op(queries, keys, query_weight, key_weight, cos, sin, positions,
                               None if args is None else args["cu_seqlens"], float(eps),
                               bool(interleaved),
                               None if sections is None else [int(n) for n in sections])
