"""Orthogonalised updates on the GPU: ``orthogonalize`` brings the singular values of every update matrix to about 1 (include/nerfds.h
nerfds_orthogonalize), all matrices of a call together whatever their shapes.  ``training.Trainer(..., optimizer='muon')`` runs it on the radiance
field's own hidden kernels; this is the same operator for a caller's matrices.  No CPU path."""
from __future__ import annotations

import ctypes as C
from typing import Sequence, Union

import torch

from . import _native as N
from .layers import _raw_stream


def orthogonalize(updates: Union[torch.Tensor, Sequence[torch.Tensor]], steps: int = 5) -> Union[torch.Tensor, list]:
  """The orthogonal factor of each [rows, cols] matrix, to the accuracy of ``steps`` quintic Newton-Schulz steps (singular values that were above about
  1e-3 of the Frobenius norm end between 0.68 and 1.21).  One element type and device per call; new contiguous tensors come back, in the order given.
  A zero matrix gives zero; a matrix with a non-finite element gives NaN.  Not differentiable: an optimizer's step runs outside the graph."""
  single = isinstance(updates, torch.Tensor)
  mats = [updates] if single else list(updates)
  if not 1 <= int(steps) <= 16:
    raise ValueError(f'orthogonalize: steps = {steps} (1 .. 16)')
  if not mats:
    return []
  first = mats[0]
  for u in mats:
    if not isinstance(u, torch.Tensor) or u.dim() != 2:
      raise ValueError('orthogonalize: every update must be a 2-d tensor')
    if not u.is_cuda:
      raise RuntimeError('orthogonalize runs on the GPU: the updates must be CUDA tensors (there is no CPU path)')
    if u.dtype != first.dtype or u.device != first.device:
      raise ValueError(f'orthogonalize: one element type and device per call, got {u.dtype} on {u.device} next to {first.dtype} on {first.device}')
  dt = N.dtype_code(first.dtype)
  lib = N.load()
  with torch.no_grad():
    out = [u.new_empty(u.shape) for u in mats]
    keep, entries = [], []
    for u, o in zip(mats, out):
      rows, cols = u.shape
      if rows == 0 or cols == 0:
        continue
      ld = u.stride(0) if rows > 1 else cols
      if (cols > 1 and u.stride(1) != 1) or ld < cols:
        u, ld = u.contiguous(), cols
        keep.append(u)
      entries.append((u.data_ptr(), ld, o.data_ptr(), cols, rows, cols))
    if entries:
      arr = (N.Matrix * len(entries))(*entries)
      nbytes = lib.nerfds_orthogonalize_workspace(arr, len(entries))
      if nbytes < 0:
        raise ValueError(f'orthogonalize: {N.last_error(None)}')
      ws = first.new_empty(nbytes, dtype=torch.uint8)
      rc = lib.nerfds_orthogonalize(first.device.index, dt, arr, len(entries), int(steps), ws.data_ptr(), nbytes, _raw_stream(first.device.index))
      if rc != 0:
        raise RuntimeError(f'nerfds_orthogonalize failed ({rc}): {N.last_error(None)}')
  return out[0] if single else out
