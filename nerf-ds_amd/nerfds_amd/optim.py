"""Orthogonalised updates on the GPU: ``orthogonalize`` brings the singular values of every update matrix to about 1 (include/nerfds.h
nerfds_orthogonalize), all matrices of a call together whatever their shapes.  ``training.Trainer(..., optimizer='muon')`` runs it on the radiance
field's own hidden kernels; this is the same operator for a caller's matrices.  No CPU path."""
from __future__ import annotations

import struct
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
  if not isinstance(first, torch.Tensor):
    raise ValueError('orthogonalize: every update must be a 2-d tensor')
  dtype, index = first.dtype, first.get_device()
  out, keep, fields = [], [], []
  with torch.no_grad():
    for u in mats:
      if not isinstance(u, torch.Tensor) or u.dim() != 2:
        raise ValueError('orthogonalize: every update must be a 2-d tensor')
      if not u.is_cuda:
        raise RuntimeError('orthogonalize runs on the GPU: the updates must be CUDA tensors (there is no CPU path)')
      if u.dtype != dtype or u.get_device() != index:
        raise ValueError(f'orthogonalize: one element type and device per call, got {u.dtype} on {u.device} next to {dtype} on {first.device}')
      rows, cols = u.shape
      o = u.new_empty((rows, cols))
      out.append(o)
      if rows == 0 or cols == 0:
        continue
      ld, one = u.stride()
      if rows == 1:
        ld = cols
      if (cols > 1 and one != 1) or ld < cols:
        u, ld = u.contiguous(), cols
        keep.append(u)
      fields += (u.data_ptr(), ld, o.data_ptr(), cols, rows, cols)
    code = N.dtype_code(dtype)
    count = len(fields) // 6
    if count:
      lib = N.load()
      mats_c = (N.Matrix * count).from_buffer_copy(struct.pack('PqPqii' * count, *fields))
      nbytes = lib.nerfds_orthogonalize_workspace(mats_c, count)
      if nbytes < 0:
        raise ValueError(f'orthogonalize: {N.last_error(None)}')
      ws = first.new_empty(max(nbytes, 1), dtype=torch.uint8)
      rc = lib.nerfds_orthogonalize(index, code, mats_c, count, int(steps), ws.data_ptr(), nbytes, _raw_stream(index))
      if rc != 0:
        raise RuntimeError(f'nerfds_orthogonalize failed ({rc}): {N.last_error(None)}')
  return out[0] if single else out
