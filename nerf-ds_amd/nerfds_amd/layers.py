"""Differentiable layers on the GPU for networks a caller puts next to the rendered rays (a colour-correction or uncertainty head on the outputs of
``autograd.DifferentiableRenderer``, say): ``dense`` - the reference's ``nn.Dense`` + activation (hypernerf/modules.py:61-82) with a residual in the
same kernel - and ``layer_norm``.  Parameters keep the Flax layout and names: ``kernel`` [in, out], ``bias`` [out], ``scale`` [d].

Both run on torch's current stream of the tensors' device, take float32, float16 or bfloat16 (one type per call), any leading axes, and views with unit
stride along the last axis as they are (others are copied).  Gradients by ``torch.autograd`` (first order); ``dense_backward`` and
``layer_norm_backward`` are the same gradients as plain calls without an autograd graph, for loops captured into a HIP graph.  Non-finite inputs are not
an error.  No CPU path."""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _native as N


def _check_operands(what: str, x: torch.Tensor, **others) -> None:
  if not isinstance(x, torch.Tensor) or x.dim() < 1:
    raise ValueError(f'{what}: x must be a tensor with at least one axis')
  if not x.is_cuda:
    raise RuntimeError(f'{what} runs on the GPU: x must be a CUDA tensor (there is no CPU path)')
  N.dtype_code(x.dtype)
  for name, t in others.items():
    if t is None:
      continue
    if not isinstance(t, torch.Tensor) or t.device != x.device or t.dtype != x.dtype:
      raise ValueError(f'{what}: {name} must be a {x.dtype} tensor on {x.device}, got '
                       + (f'{t.dtype} on {t.device}' if isinstance(t, torch.Tensor) else type(t).__name__))


def _rows(t: torch.Tensor, cols: int, one_row: bool = False) -> Tuple[torch.Tensor, int]:
  """``t`` as [rows, cols] with unit stride along the columns, and its row stride (``one_row``: 0, one row for all, is allowed)."""
  if t.is_contiguous():
    return t, cols
  t = t.reshape(-1, cols)
  ld = t.stride(0) if t.shape[0] > 1 else cols
  if (cols > 1 and t.stride(1) != 1) or (ld < cols and not (one_row and ld == 0)):
    t, ld = t.contiguous(), cols
  return t, ld


def _ptr(t: Optional[torch.Tensor]):
  return t.data_ptr() if t is not None else None


# the handle of torch's current stream of a device, without building a Stream object around it (the launch of a small layer costs less than that)
_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(what: str, fn, x: torch.Tensor, args) -> None:
  index = x.device.index
  rc = fn(index, C.byref(args), _raw_stream(index))
  if rc != 0:
    raise RuntimeError(f'{what} failed ({rc}): {N.last_error(None)}')


def _call_with_workspace(what: str, query, fn, x: torch.Tensor, args) -> None:
  index = x.device.index
  nbytes = query(index, C.byref(args))
  if nbytes < 0:
    raise RuntimeError(f'{what}: workspace query failed ({nbytes}): {N.last_error(None)}')
  if nbytes:
    ws = x.new_empty(nbytes, dtype=torch.uint8)
    args.workspace, args.workspace_bytes = ws.data_ptr(), nbytes
  _call(what, fn, x, args)


# ---- dense ------------------------------------------------------------------------------------------------------------------------------------
def _check_dense(what, x, kernel, bias, residual, activation):
  _check_operands(what, x, kernel=kernel, bias=bias, residual=residual)
  if activation not in N.ACTIVATIONS:
    raise ValueError(f'{what}: unknown activation {activation!r} (one of {", ".join(N.ACTIVATIONS)})')
  if kernel.dim() != 2 or kernel.shape[0] != x.shape[-1] or kernel.shape[0] < 1 or kernel.shape[1] < 1:
    raise ValueError(f'{what}: kernel {tuple(kernel.shape)} does not fit x {tuple(x.shape)}: [in, out] with in = x.shape[-1] >= 1 and out >= 1')
  n = kernel.shape[1]
  if bias is not None and bias.shape != (n,):
    raise ValueError(f'{what}: bias {tuple(bias.shape)} for {n} outputs')
  if residual is not None and residual.shape != (*x.shape[:-1], n):
    raise ValueError(f'{what}: residual {tuple(residual.shape)}, the output is {(*x.shape[:-1], n)}')


def _dense_forward(x, kernel, bias, residual, activation, keep):
  """(y, what the backward needs of the pre-activation or None)."""
  lib = N.load()
  k, n = kernel.shape
  x2, ldx = _rows(x, k)
  w, ldk = _rows(kernel, n)
  r, ldr = _rows(residual, n, one_row=True) if residual is not None else (None, 0)
  if bias is not None:
    bias = bias.contiguous()
  m, dt, act = x.numel() // k, N.dtype_code(x.dtype), N.ACTIVATIONS[activation]
  y = x.new_empty((*x.shape[:-1], n))
  save = None
  if keep and act:
    save = x.new_empty((m, (n + 7) // 8), dtype=torch.uint8) if activation == 'relu' else x.new_empty((m, n))
  args = N.DenseForwardArgs(dt, act, m, k, n, x2.data_ptr(), ldx, w.data_ptr(), ldk, _ptr(bias), _ptr(r), ldr, y.data_ptr(), n, _ptr(save), None, 0)
  if 8 < m < 32768:      # (outside: never a workspace)
    _call_with_workspace('nerfds_dense_forward', lib.nerfds_dense_forward_workspace, lib.nerfds_dense_forward, x, args)
  else:
    _call('nerfds_dense_forward', lib.nerfds_dense_forward, x, args)
  return y, save


def dense_backward(dy: torch.Tensor, x: torch.Tensor, kernel: torch.Tensor, saved: Optional[torch.Tensor], activation: str = 'none', *, need_dx: bool = True,
                   need_dkernel: bool = True, need_dbias: bool = True):
  """(dx, dkernel, dbias) of ``dense`` for the cotangent ``dy``, None where not needed; the residual's gradient is ``dy`` itself.  ``saved`` comes from
  ``dense_forward``."""
  _check_dense('dense_backward', x, kernel, None, None, activation)
  _check_operands('dense_backward', x, dy=dy)
  k, n = kernel.shape
  if tuple(dy.shape) != (*x.shape[:-1], n):
    raise ValueError(f'dense_backward: dy {tuple(dy.shape)}, the output is {(*x.shape[:-1], n)}')
  m = x.numel() // k
  if activation != 'none':
    want = (torch.uint8, (m, (n + 7) // 8)) if activation == 'relu' else (x.dtype, (m, n))
    if saved is None or saved.dtype != want[0] or tuple(saved.shape) != want[1] or saved.device != x.device or not saved.is_contiguous():
      raise ValueError(f'dense_backward: {activation} needs what dense_forward saved: a contiguous {want[0]} tensor of shape {want[1]} on {x.device}')
  return _dense_backward(dy, x, kernel, saved if activation != 'none' else None, activation, need_dx, need_dkernel, need_dbias)


def _dense_backward(dy, x, kernel, saved, activation, need_dx, need_dkernel, need_dbias):
  lib = N.load()
  k, n = kernel.shape
  x2, ldx = _rows(x, k)
  w, ldk = _rows(kernel, n)
  g, ldg = _rows(dy, n)
  dx = x.new_empty(x.shape) if need_dx else None
  dkernel = x.new_empty((k, n)) if need_dkernel else None
  dbias = x.new_empty(n) if need_dbias else None
  _call_with_workspace('nerfds_dense_backward', lib.nerfds_dense_backward_workspace, lib.nerfds_dense_backward, x,
                       N.DenseBackwardArgs(N.dtype_code(x.dtype), N.ACTIVATIONS[activation], x.numel() // k, k, n, x2.data_ptr(), ldx, w.data_ptr(), ldk, g.data_ptr(), ldg,
                                           _ptr(saved), _ptr(dx), k, _ptr(dkernel), _ptr(dbias), None, 0))
  return dx, dkernel, dbias


def dense_forward(x: torch.Tensor, kernel: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = 'none',
                  residual: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
  """``dense`` without an autograd graph, and what ``dense_backward`` needs of it (None for no activation)."""
  _check_dense('dense_forward', x, kernel, bias, residual, activation)
  with torch.no_grad():
    return _dense_forward(x, kernel, bias, residual, activation, True)


class _Dense(torch.autograd.Function):

  @staticmethod
  def forward(ctx, x, kernel, bias, residual, activation):
    y, saved = _dense_forward(x, kernel, bias, residual, activation, any(ctx.needs_input_grad[:3]))
    ctx.activation = activation
    ctx.save_for_backward(x, kernel, saved)
    return y

  @staticmethod
  def backward(ctx, dy):
    return _dense_gradients_once(ctx, dy) if torch.is_grad_enabled() else _Dense.gradients(ctx, dy)

  @staticmethod
  def gradients(ctx, dy):
    x, kernel, saved = ctx.saved_tensors
    need = ctx.needs_input_grad
    dx = dkernel = dbias = None
    if any(need[:3]):
      dx, dkernel, dbias = _dense_backward(dy, x, kernel, saved, ctx.activation, need[0], need[1], need[2])
    return dx, dkernel, dbias, dy if need[3] else None, None


# with create_graph=True the gradients come out marked as not differentiable again (the mark costs more than the launch, so it is left out otherwise)
_dense_gradients_once = once_differentiable(_Dense.gradients)


def dense(x: torch.Tensor, kernel: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = 'none', residual: Optional[torch.Tensor] = None) -> torch.Tensor:
  """act(x @ kernel + bias) + residual for x [..., in], kernel [in, out]; ``activation``: none, relu, sigmoid, softplus, silu or gelu (erf form)."""
  _check_dense('dense', x, kernel, bias, residual, activation)
  if torch.is_grad_enabled() and (x.requires_grad or kernel.requires_grad or (bias is not None and bias.requires_grad)
                                  or (residual is not None and residual.requires_grad)):
    return _Dense.apply(x, kernel, bias, residual, activation)
  return _dense_forward(x, kernel, bias, residual, activation, False)[0]


# ---- layer norm ---------------------------------------------------------------------------------------------------------------------------------
def _check_norm(what, x, scale, bias, epsilon):
  _check_operands(what, x, scale=scale, bias=bias)
  d = x.shape[-1]
  if d < 1:
    raise ValueError(f'{what}: x {tuple(x.shape)} has no elements along its last axis')
  for name, t in (('scale', scale), ('bias', bias)):
    if t is not None and t.shape != (d,):
      raise ValueError(f'{what}: {name} {tuple(t.shape)} for rows of {d}')
  if not 0.0 <= epsilon < float('inf'):
    raise ValueError(f'{what}: epsilon must be finite and >= 0, got {epsilon}')


def _norm_forward(x, scale, bias, epsilon, keep):
  lib = N.load()
  d = x.shape[-1]
  x2, ldx = _rows(x, d)
  m = x.numel() // d
  scale = scale.contiguous() if scale is not None else None
  bias = bias.contiguous() if bias is not None else None
  y = x.new_empty(x.shape)
  stats = x.new_empty((m, 2), dtype=torch.float32) if keep else None
  _call('nerfds_layer_norm_forward', lib.nerfds_layer_norm_forward, x, N.LayerNormForwardArgs(N.dtype_code(x.dtype), d, m, epsilon, x2.data_ptr(), ldx, _ptr(scale), _ptr(bias),
                                                                                        y.data_ptr(), d, _ptr(stats)))
  return y, stats


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, scale: Optional[torch.Tensor], stats: torch.Tensor, *, need_dx: bool = True, need_dscale: bool = True,
                        need_dbias: bool = True):
  """(dx, dscale, dbias) of ``layer_norm`` for the cotangent ``dy``, None where not needed; ``stats`` comes from ``layer_norm_forward``."""
  _check_norm('layer_norm_backward', x, scale, None, 0.0)
  _check_operands('layer_norm_backward', x, dy=dy)
  if dy.shape != x.shape:
    raise ValueError(f'layer_norm_backward: dy {tuple(dy.shape)} for x {tuple(x.shape)}')
  m = x.numel() // x.shape[-1]
  if stats is None or tuple(stats.shape) != (m, 2) or stats.dtype != torch.float32 or stats.device != x.device or not stats.is_contiguous():
    raise ValueError(f'layer_norm_backward: stats must be the contiguous float32 [{m}, 2] tensor of layer_norm_forward')
  return _norm_backward(dy, x, scale, stats, need_dx, need_dscale, need_dbias)


def _norm_backward(dy, x, scale, stats, need_dx, need_dscale, need_dbias):
  lib = N.load()
  d = x.shape[-1]
  x2, ldx = _rows(x, d)
  g, ldg = _rows(dy, d)
  scale = scale.contiguous() if scale is not None else None
  dx = x.new_empty(x.shape) if need_dx else None
  dscale = x.new_empty(d) if need_dscale else None
  dbias = x.new_empty(d) if need_dbias else None
  _call_with_workspace('nerfds_layer_norm_backward', lib.nerfds_layer_norm_backward_workspace, lib.nerfds_layer_norm_backward, x,
                       N.LayerNormBackwardArgs(N.dtype_code(x.dtype), d, x.numel() // d, x2.data_ptr(), ldx, _ptr(scale), g.data_ptr(), ldg, stats.data_ptr(), _ptr(dx), d,
                                               _ptr(dscale), _ptr(dbias), None, 0))
  return dx, dscale, dbias


def layer_norm_forward(x: torch.Tensor, scale: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, epsilon: float = 1e-6):
  """``layer_norm`` without an autograd graph, and the statistics [rows, 2] (mean, 1 / sqrt(var + epsilon)) that ``layer_norm_backward`` needs."""
  _check_norm('layer_norm_forward', x, scale, bias, epsilon)
  with torch.no_grad():
    return _norm_forward(x, scale, bias, epsilon, True)


class _LayerNorm(torch.autograd.Function):

  @staticmethod
  def forward(ctx, x, scale, bias, epsilon):
    y, stats = _norm_forward(x, scale, bias, epsilon, True)
    ctx.save_for_backward(x, scale, stats)
    return y

  @staticmethod
  def backward(ctx, dy):
    return _norm_gradients_once(ctx, dy) if torch.is_grad_enabled() else _LayerNorm.gradients(ctx, dy)

  @staticmethod
  def gradients(ctx, dy):
    x, scale, stats = ctx.saved_tensors
    need = ctx.needs_input_grad
    return (*_norm_backward(dy, x, scale, stats, need[0], need[1], need[2]), None)


_norm_gradients_once = once_differentiable(_LayerNorm.gradients)


def layer_norm(x: torch.Tensor, scale: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, epsilon: float = 1e-6) -> torch.Tensor:
  """(x - mean) / sqrt(var + epsilon) * scale + bias over the last axis of x (flax ``nn.LayerNorm``'s names and default epsilon; var is the mean of the
  squared deviations, computed in two passes)."""
  _check_norm('layer_norm', x, scale, bias, epsilon)
  if torch.is_grad_enabled() and (x.requires_grad or (scale is not None and scale.requires_grad) or (bias is not None and bias.requires_grad)):
    return _LayerNorm.apply(x, scale, bias, epsilon)
  return _norm_forward(x, scale, bias, epsilon, False)[0]
