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
  t = t.reshape(-1, cols)
  ld = t.stride(0) if t.shape[0] > 1 else cols
  if (cols > 1 and t.stride(1) != 1) or (ld < cols and not (one_row and ld == 0)):
    t, ld = t.contiguous(), cols
  return t, ld


def _ptr(t: Optional[torch.Tensor]):
  return t.data_ptr() if t is not None else None


def _call(what: str, fn, x: torch.Tensor, args) -> None:
  rc = fn(x.device.index, C.byref(args), torch.cuda.current_stream(x.device).cuda_stream)
  if rc != 0:
    raise RuntimeError(f'{what} failed ({rc}): {N.last_error(None)}')


def _workspace(nbytes: int, x: torch.Tensor) -> Optional[torch.Tensor]:
  if nbytes < 0:
    raise RuntimeError(f'workspace query failed ({nbytes}): {N.last_error(None)}')
  return torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None


# ---- dense ------------------------------------------------------------------------------------------------------------------------------------
def _check_dense(what, x, kernel, bias, residual, activation):
  _check_operands(what, x, kernel=kernel, bias=bias, residual=residual)
  if activation not in N.ACTIVATIONS:
    raise ValueError(f'{what}: unknown activation {activation!r} (one of {", ".join(N.ACTIVATIONS)})')
  if kernel.dim() != 2 or kernel.shape[0] != x.shape[-1] or kernel.shape[0] < 1 or kernel.shape[1] < 1:
    raise ValueError(f'{what}: kernel {tuple(kernel.shape)} does not fit x {tuple(x.shape)}: [in, out] with in = x.shape[-1] >= 1 and out >= 1')
  n = kernel.shape[1]
  if bias is not None and tuple(bias.shape) != (n,):
    raise ValueError(f'{what}: bias {tuple(bias.shape)} for {n} outputs')
  if residual is not None and tuple(residual.shape) != (*x.shape[:-1], n):
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
  m, dt, act = x2.shape[0], N.dtype_code(x.dtype), N.ACTIVATIONS[activation]
  y = torch.empty((*x.shape[:-1], n), dtype=x.dtype, device=x.device)
  save = None
  if keep and act:
    save = torch.empty((m, (n + 7) // 8), dtype=torch.uint8, device=x.device) if activation == 'relu' else torch.empty((m, n), dtype=x.dtype, device=x.device)
  _call('nerfds_dense_forward', lib.nerfds_dense_forward, x, N.DenseForwardArgs(dt, act, m, k, n, x2.data_ptr(), ldx, w.data_ptr(), ldk, _ptr(bias), _ptr(r), ldr,
                                                                              y.data_ptr(), n, _ptr(save)))
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
  x2, ldx = _rows(x, k)
  m = x2.shape[0]
  if activation != 'none':
    want = (torch.uint8, (m, (n + 7) // 8)) if activation == 'relu' else (x.dtype, (m, n))
    if saved is None or saved.dtype != want[0] or tuple(saved.shape) != want[1] or saved.device != x.device or not saved.is_contiguous():
      raise ValueError(f'dense_backward: {activation} needs what dense_forward saved: a contiguous {want[0]} tensor of shape {want[1]} on {x.device}')
  lib = N.load()
  w, ldk = _rows(kernel, n)
  g, ldg = _rows(dy, n)
  dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_dx else None
  dkernel = torch.empty((k, n), dtype=x.dtype, device=x.device) if need_dkernel else None
  dbias = torch.empty(n, dtype=x.dtype, device=x.device) if need_dbias else None
  args = N.DenseBackwardArgs(N.dtype_code(x.dtype), N.ACTIVATIONS[activation], m, k, n, x2.data_ptr(), ldx, w.data_ptr(), ldk, g.data_ptr(), ldg,
                             _ptr(saved) if activation != 'none' else None, _ptr(dx), k, _ptr(dkernel), _ptr(dbias), None, 0)
  ws = _workspace(lib.nerfds_dense_backward_workspace(x.device.index, C.byref(args)), x)
  args.workspace, args.workspace_bytes = _ptr(ws), ws.numel() if ws is not None else 0
  _call('nerfds_dense_backward', lib.nerfds_dense_backward, x, args)
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
  @once_differentiable
  def backward(ctx, dy):
    x, kernel, saved = ctx.saved_tensors
    need = ctx.needs_input_grad
    dx = dkernel = dbias = None
    if any(need[:3]):
      dx, dkernel, dbias = dense_backward(dy, x, kernel, saved, ctx.activation, need_dx=need[0], need_dkernel=need[1], need_dbias=need[2])
    return dx, dkernel, dbias, dy if need[3] else None, None


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
    if t is not None and tuple(t.shape) != (d,):
      raise ValueError(f'{what}: {name} {tuple(t.shape)} for rows of {d}')
  if not 0.0 <= epsilon < float('inf'):
    raise ValueError(f'{what}: epsilon must be finite and >= 0, got {epsilon}')


def _norm_forward(x, scale, bias, epsilon, keep):
  lib = N.load()
  d = x.shape[-1]
  x2, ldx = _rows(x, d)
  m = x2.shape[0]
  scale, bias = (t.contiguous() if t is not None else None for t in (scale, bias))
  y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
  stats = torch.empty((m, 2), dtype=torch.float32, device=x.device) if keep else None
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
  d = x.shape[-1]
  x2, ldx = _rows(x, d)
  m = x2.shape[0]
  if stats is None or tuple(stats.shape) != (m, 2) or stats.dtype != torch.float32 or stats.device != x.device or not stats.is_contiguous():
    raise ValueError(f'layer_norm_backward: stats must be the contiguous float32 [{m}, 2] tensor of layer_norm_forward')
  lib = N.load()
  g, ldg = _rows(dy, d)
  scale = scale.contiguous() if scale is not None else None
  dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_dx else None
  dscale = torch.empty(d, dtype=x.dtype, device=x.device) if need_dscale else None
  dbias = torch.empty(d, dtype=x.dtype, device=x.device) if need_dbias else None
  args = N.LayerNormBackwardArgs(N.dtype_code(x.dtype), d, m, x2.data_ptr(), ldx, _ptr(scale), g.data_ptr(), ldg, stats.data_ptr(), _ptr(dx), d, _ptr(dscale), _ptr(dbias), None, 0)
  ws = _workspace(lib.nerfds_layer_norm_backward_workspace(x.device.index, C.byref(args)), x)
  args.workspace, args.workspace_bytes = _ptr(ws), ws.numel() if ws is not None else 0
  _call('nerfds_layer_norm_backward', lib.nerfds_layer_norm_backward, x, args)
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
  @once_differentiable
  def backward(ctx, dy):
    x, scale, stats = ctx.saved_tensors
    need = ctx.needs_input_grad
    return (*layer_norm_backward(dy, x, scale, stats, need_dx=need[0], need_dscale=need[1], need_dbias=need[2]), None)


def layer_norm(x: torch.Tensor, scale: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, epsilon: float = 1e-6) -> torch.Tensor:
  """(x - mean) / sqrt(var + epsilon) * scale + bias over the last axis of x (flax ``nn.LayerNorm``'s names and default epsilon; var is the mean of the
  squared deviations, computed in two passes)."""
  _check_norm('layer_norm', x, scale, bias, epsilon)
  if torch.is_grad_enabled() and (x.requires_grad or (scale is not None and scale.requires_grad) or (bias is not None and bias.requires_grad)):
    return _LayerNorm.apply(x, scale, bias, epsilon)
  return _norm_forward(x, scale, bias, epsilon, False)[0]
