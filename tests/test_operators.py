"""The stand-alone operators (nerfds_amd.layers, nerfds_amd.optim) against their definitions in 64 bits, and their refusals.

Tolerances count roundings: u = half a step of the element type for each rounding to it, and 2^-24 for each float32 operation of the longest chain an element
passes through, times the sum of magnitudes it is taken of."""
import ctypes as C
import math

import pytest
import torch

from nerfds_amd import _native as N
from nerfds_amd import layers, optim

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
E24 = 2.0 ** -24
SMOOTH = ('sigmoid', 'softplus', 'silu', 'gelu')


def half_step(t):
  return torch.finfo(t).eps / 2


def tiny(t):      # half the spacing of the subnormals: what a rounding may lose where values underflow
  return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def make(*shape, t=F32, seed=0, scale=1.0, shift=0.0, grid=None):
  g = torch.Generator().manual_seed(seed)
  v = torch.randn(shape, generator=g, dtype=torch.float64) * scale + shift
  if grid is not None:
    v = (v.clamp(-2, 2) / grid).round() * grid
  return v.to(t)


def dev(*ts):
  return [None if v is None else v.cuda() for v in ts]


def act64(z, act):
  """(act(z), act'(z), a bound of |act''|)."""
  s = torch.sigmoid(z)
  if act == 'none':
    return z, torch.ones_like(z), 0.0
  if act == 'relu':
    return z.clamp_min(0), (z > 0).double(), 0.0
  if act == 'sigmoid':
    return s, s * (1 - s), 0.1
  if act == 'softplus':
    return torch.logaddexp(z, torch.zeros_like(z)), s, 0.25
  if act == 'silu':
    return z * s, s * (1 + z * (1 - s)), 0.5
  cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
  return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), 0.8


def dense64(x, w, b, r, act, dy=None):
  """{name: (value, bound of the error)} of the dense layer for inputs of x's type."""
  t = x.dtype
  u = half_step(t)
  x, w = x.double(), w.double()
  k, n, m = x.shape[1], w.shape[1], x.shape[0]
  z, mag = x @ w, x.abs() @ w.abs()
  if b is not None:
    z, mag = z + b.double(), mag + b.double().abs()
  ez = (k + 8) * E24 * mag                     # float32 accumulation (and, for float32 operands, the dropped products)
  y, slope, curve = act64(z, act)
  ey = 1.2 * ez + 16 * E24 * (y.abs() + mag * 0)      # slopes are at most 1.13; the activation's own few float32 roundings
  if r is not None:
    y = y + r.double()
    ey = ey + 2 * E24 * (y.abs() + r.double().abs())
  out = {'y': (y, ey + u * y.abs() + tiny(t) + E24 * 1e-6)}
  if dy is None:
    return out
  dy = dy.double()
  dz = dy * slope
  edz = torch.zeros_like(dz)
  if act in SMOOTH:      # z is kept in the tensors' type, dz rounded to it
    edz = dy.abs() * (curve * (ez + u * z.abs()) + 16 * E24) + u * dz.abs() + tiny(t)
  def product(a, e, b2, length):
    return a @ b2, e @ b2.abs() + (length + 8) * E24 * (a.abs() @ b2.abs())
  for name, (v, e) in {'dx': product(dz, edz, w.t(), n), 'dkernel': tuple(q.t() for q in product(dz.t(), edz.t(), x, m))}.items():
    out[name] = (v, e + u * v.abs() + tiny(t))
  v = dz.sum(0)
  out['db'] = (v, edz.sum(0) + (m + 8) * E24 * dz.abs().sum(0) + u * v.abs() + tiny(t))
  return out


def close(got, want, what=''):
  v, e = want
  got = got.detach().to(v.device).double().reshape(v.shape)
  bad = (got - v).abs() > e
  assert torch.isfinite(got).all() and not bad.any(), (what, int(bad.sum()), float(((got - v).abs() / e.clamp_min(1e-300)).max()))


SHAPES = [(1, 1, 1), (1, 256, 256), (3, 7, 5), (2, 64, 3), (5, 513, 40), (8, 1030, 77), (9, 520, 96), (17, 130, 9), (130, 33, 131), (257, 560, 128), (64, 64, 64), (129, 128, 300), (1025, 45, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize('t', [F32, F16, BF16], ids=['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('i', range(len(SHAPES)), ids=['x'.join(map(str, s)) for s in SHAPES])
def test_dense_and_its_gradients(i, t):
  m, k, n = SHAPES[i]
  for j, act in enumerate(N.ACTIVATIONS):
    bias, residual = (i + j) % 3 != 0, (i + j) % 2 == 0
    # relu: values on a grid whose products and sums float32 holds exactly, so that no rounding moves a pre-activation across 0 (many ARE 0)
    grid = 0.25 if act == 'relu' else None
    x, w = make(m, k, t=t, seed=1, grid=grid), make(k, n, t=t, seed=2, scale=1.0 if grid else k ** -0.5, grid=grid)
    b = make(n, t=t, seed=3, grid=grid) if bias else None
    r = make(m, n, t=t, seed=4) if residual else None
    dy = make(m, n, t=t, seed=5)
    want = dense64(x, w, b, r, act, dy)
    leaves = [v.requires_grad_(True) if v is not None else None for v in dev(x, w, b, r)]
    y = layers.dense(leaves[0], leaves[1], leaves[2], activation=act, residual=leaves[3])
    close(y, want['y'], act)
    close(layers.dense(*dev(x, w, b), activation=act, residual=dev(r)[0]), want['y'], act)
    y.backward(dy.cuda())
    for name, v in zip(('dx', 'dkernel', 'db'), leaves):
      if v is not None:
        close(v.grad, want[name], (act, name))
    if r is not None:
      assert torch.equal(leaves[3].grad.cpu(), dy)


# many rows past a small kernel (aligned and not), large tiles (aligned: with and without relu bits, ragged at every end), small tiles (odd sizes), few rows with splits
MANY = [(20011, 172, 131, 'relu'), (16400, 308, 256, 'relu'), (17003, 560, 128, 'silu'), (16385, 64, 64, 'none'), (16390, 33, 70, 'softplus'), (16384, 256, 256, 'gelu'),
        (4099, 520, 1031, 'gelu'), (4100, 520, 1056, 'relu'), (2057, 1048, 1032, 'sigmoid'), (4200, 264, 520, 'none'), (300, 1500, 70, 'none'), (2100, 1000, 96, 'relu')]


@pytest.mark.gpu
@pytest.mark.parametrize('t', [F32, F16, BF16], ids=['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('i', range(len(MANY)), ids=['%dx%dx%d-%s' % s for s in MANY])
def test_dense_at_sizes_with_many_tiles_and_splits(i, t):
  m, k, n, act = MANY[i]
  grid = 0.25 if act == 'relu' else None
  x, w, dy = make(m, k, t=t, seed=6, grid=grid), make(k, n, t=t, seed=7, scale=1.0 if grid else k ** -0.5, grid=grid), make(m, n, t=t, seed=8)
  b = make(n, t=t, seed=9, grid=grid) if i % 4 else None
  r = make(m, n, t=t, seed=10) if i % 2 else None
  x, w, dy, b, r = dev(x, w, dy, b, r)      # (64-bit products of this size are the GPU's work; elementwise bounds as everywhere)
  want = dense64(x, w, b, r, act, dy)
  y, saved = layers.dense_forward(x, w, b, act, r)
  close(y, want['y'])
  for name, g in zip(('dx', 'dkernel', 'db'), layers.dense_backward(dy, x, w, saved, act)):
    close(g, want[name], name)
  if m % 3 == 0:      # the same through a view of padded rows
    wide = torch.zeros((m, k + 8), dtype=t, device='cuda')
    wide[:, :k] = x
    assert torch.equal(layers.dense_forward(wide[:, :k], w, b, act, r)[0], y)


# both gradients in one pass: each width class, a last stage of a few rows or of one, several rounds of the ring of stages, one workgroup
BOTH = [(32768, 256, 256, 'relu'), (150001, 256, 256, 'relu'), (140003, 160, 136, 'gelu'), (140033, 256, 96, 'relu'), (90001, 200, 64, 'none'), (90007, 64, 256, 'relu'), (33000, 128, 200, 'silu'),
        (100001, 96, 128, 'relu'), (70000, 128, 8, 'none'),
        (1, 256, 256, 'relu'), (63, 256, 256, 'none'), (65, 128, 160, 'relu'), (500, 8, 32, 'relu'),
        (100003, 256, 64, 'softplus'), (50001, 64, 64, 'sigmoid'), (40000, 256, 256, 'silu'), (70001, 104, 256, 'gelu')]


@pytest.mark.gpu
@pytest.mark.parametrize('t', [F16, BF16], ids=['f16', 'bf16'])
@pytest.mark.parametrize('i', range(len(BOTH)), ids=['%dx%dx%d-%s' % s for s in BOTH])
def test_dense_gradients_of_narrow_layers(i, t):
  _gradients_together_and_apart(*BOTH[i], t)


# tiles that fill the card in each direction, relu with its bits tested in the tiles and before them
WIDE = [(16645, 264, 1032, 'gelu'), (16645, 1040, 64, 'relu'), (16645, 520, 1056, 'relu'), (33000, 520, 512, 'relu'), (33001, 512, 544, 'relu'), (16645, 72, 1024, 'none'), (777, 1048, 1032, 'relu')]


@pytest.mark.gpu
@pytest.mark.parametrize('t', [F16, BF16], ids=['f16', 'bf16'])
@pytest.mark.parametrize('i', range(len(WIDE)), ids=['%dx%dx%d-%s' % s for s in WIDE])
def test_dense_wide_layers_over_many_rows(i, t):
  _gradients_together_and_apart(*WIDE[i], t)


# few rows: the contraction of y (k) and of dx (n) split, each alone and both, ragged pieces
FEW = [(9, 4096, 64, 'relu'), (12, 591, 2854, 'softplus'), (33, 2048, 300, 'none'), (64, 1000, 1000, 'gelu'), (130, 700, 40, 'silu'), (513, 3000, 20, 'relu'), (700, 24, 1999, 'sigmoid'), (10, 512, 513, 'relu')]


@pytest.mark.gpu
@pytest.mark.parametrize('t', [F32, F16, BF16], ids=['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('i', range(len(FEW)), ids=['%dx%dx%d-%s' % s for s in FEW])
def test_dense_few_rows_over_long_contractions(i, t):
  m, k, n, act = FEW[i]
  grid = 0.25 if act == 'relu' else None
  x, w, dy, b, r = dev(make(m, k, t=t, seed=6, grid=grid), make(k, n, t=t, seed=7, scale=1.0 if grid else k ** -0.5, grid=grid), make(m, n, t=t, seed=8),
                       make(n, t=t, seed=9, grid=grid) if i % 3 else None, make(m, n, t=t, seed=10) if i % 2 else None)
  want = dense64(x, w, b, r, act, dy)
  y, saved = layers.dense_forward(x, w, b, act, r)
  close(y, want['y'])
  assert torch.equal(layers.dense_forward(x, w, b, act, r)[0], y)
  for name, g in zip(('dx', 'dkernel', 'db'), layers.dense_backward(dy, x, w, saved, act)):
    close(g, want[name], name)
  close(layers.dense_backward(dy, x, w, saved, act, need_dkernel=False, need_dbias=False)[0], want['dx'])
  # without a workspace, rows of y and the residual with a stride of their own; and what is no workspace
  lib, code, wide = N.load(), N.dtype_code(t), torch.full((m, n + 3), -7.0, dtype=t, device='cuda')
  a = N.DenseForwardArgs(code, N.ACTIVATIONS[act], m, k, n, x.data_ptr(), k, w.data_ptr(), n, b.data_ptr() if b is not None else None, r.data_ptr() if r is not None else None, n,
                         wide.data_ptr(), n + 3, None)
  st, index = torch.cuda.current_stream().cuda_stream, torch.cuda.current_device()
  assert lib.nerfds_dense_forward(index, C.byref(a), st) == 0
  close(wide[:, :n], want['y'])
  nbytes = lib.nerfds_dense_forward_workspace(index, C.byref(a))
  if nbytes > 0:
    ws = torch.empty(nbytes + 256, dtype=torch.uint8, device='cuda')
    wide.fill_(-7.0)
    a.workspace, a.workspace_bytes = ws.data_ptr(), nbytes
    assert lib.nerfds_dense_forward(index, C.byref(a), st) == 0
    assert torch.equal(wide[:, :n], y) and bool((wide[:, n:] == -7.0).all())
    for p, size in ((ws.data_ptr(), nbytes - 1), (ws.data_ptr() + 16, nbytes)):
      a.workspace, a.workspace_bytes = p, size
      assert lib.nerfds_dense_forward(index, C.byref(a), st) == -22


@pytest.mark.gpu
@pytest.mark.parametrize('t', [F16, BF16], ids=['f16', 'bf16'])
@pytest.mark.parametrize('act', ['sigmoid', 'softplus', 'silu', 'gelu'])
def test_dense_small_gradients_lose_only_their_own_rounding(act, t):
  for m, k, n in ((2, 438, 13), (17, 2, 32), (1, 40, 8), (200, 300, 256), (16500, 16, 3), (5, 7, 9001), (3001, 64, 16), (130, 200, 128), (1000, 24, 200), (32768, 8, 8), (77, 128, 64)):
    # pre-activations that float32 sums exactly and the tensors' type holds, so that the saved ones are exact
    x, w, b, dy = dev(make(m, k, t=t, seed=1, grid=1.0), make(k, n, t=t, seed=2, scale=0.5, grid=0.25), make(n, t=t, seed=3, grid=0.25), make(m, n, t=t, seed=4))
    z = x.double() @ w.double() + b.double()
    assert torch.equal(z.to(t).double(), z)
    slope = act64(z, act)[1]
    dz = dy.double() * slope
    u = half_step(t)
    # dz is not rounded: two parts keep u^2 of it (tiny: of a second part that underflows); beside that the slope's few float32 roundings, relative to 1
    edz = 16 * E24 * dy.double().abs() + (u * u + 4 * E24) * dz.abs() + tiny(t)
    _, saved = layers.dense_forward(x, w, b, act)
    dx, dk, db = layers.dense_backward(dy, x, w, saved, act)
    for got, v, e, length in ((dx, dz @ w.double().t(), edz @ w.double().abs().t(), n), (dk, x.double().t() @ dz, x.double().abs().t() @ edz, m), (db, dz.sum(0), edz.sum(0), m)):
      total = dz.abs() @ w.double().abs().t() if got is dx else x.double().abs().t() @ dz.abs() if got is dk else dz.abs().sum(0)
      close(got, (v, e + (length + 8) * E24 * total + u * v.abs() + tiny(t)), (m, k, n))


def _gradients_together_and_apart(m, k, n, act, t):
  grid = 0.25 if act == 'relu' else None
  x, w, dy = dev(make(m, k, t=t, seed=6, grid=grid), make(k, n, t=t, seed=7, scale=1.0 if grid else k ** -0.5, grid=grid), make(m, n, t=t, seed=8))
  want = dense64(x, w, None, None, act, dy)
  y, saved = layers.dense_forward(x, w, None, act)
  close(y, want['y'])
  first = layers.dense_backward(dy, x, w, saved, act)
  for name, g in zip(('dx', 'dkernel', 'db'), first):
    close(g, want[name], name)
  again = layers.dense_backward(dy, x, w, saved, act, need_dbias=False)
  assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1]) and again[2] is None
  close(layers.dense_backward(dy, x, w, saved, act, need_dkernel=False)[0], want['dx'], 'dx')      # apart, by other kernels
  close(layers.dense_backward(dy, x, w, saved, act, need_dx=False)[1], want['dkernel'], 'dkernel')


@pytest.mark.gpu
@pytest.mark.parametrize('t', [F32, F16], ids=['f32', 'f16'])
def test_dense_takes_views_expanded_residuals_and_leading_axes(t):
  m, k, n = 35, 37, 41
  big, wbig, gbig = make(m, 3 * k + 1, t=t, seed=1).cuda(), make(k, 2 * n + 3, t=t, seed=2).cuda(), make(n, m, t=t, seed=3).cuda()
  x, w, dy = big[:, k + 1:2 * k + 1], wbig[:, 1:n + 1], gbig.t()      # odd offsets, padded rows, a transposed cotangent
  r = make(n, t=t, seed=4).cuda().expand(m, n)                        # one row for all
  want = dense64(x.cpu(), w.cpu(), None, r.cpu(), 'silu', dy.cpu())
  y, saved = layers.dense_forward(x, w, None, 'silu', r)
  close(y, want['y'])
  for name, g in zip(('dx', 'dkernel', 'db'), layers.dense_backward(dy, x, w, saved, 'silu')):
    close(g, want[name], name)
  close(layers.dense(x.reshape(5, 7, k), w.t().contiguous().t(), None, 'silu', r.reshape(5, 7, n)), want['y'])
  shared = make(n, t=t, seed=4).cuda().requires_grad_(True)           # the gradient of a broadcast input is summed over the rows
  layers.dense(x, w, None, 'silu', shared.expand(m, n)).backward(dy)
  v = dy.cpu().double().sum(0)
  close(shared.grad, (v, (half_step(t) + m * E24) * dy.cpu().double().abs().sum(0)))


@pytest.mark.gpu
def test_dense_computes_what_is_asked_for_and_handles_no_rows():
  x, w, b, dy = dev(make(70, 40, seed=1), make(40, 50, seed=2), make(50, seed=3), make(70, 50, seed=4))
  y, saved = layers.dense_forward(x, w, b, 'softplus')
  full = layers.dense_backward(dy, x, w, saved, 'softplus')
  for need in range(8):
    flags = [bool(need >> i & 1) for i in range(3)]
    got = layers.dense_backward(dy, x, w, saved, 'softplus', need_dx=flags[0], need_dkernel=flags[1], need_dbias=flags[2])
    for f, g, ref in zip(flags, got, full):
      assert (g is None) != f and (g is None or torch.equal(g, ref))
  for act in ('none', 'relu', 'gelu'):
    e = x[:0].clone().requires_grad_(True)
    wl, bl = w.clone().requires_grad_(True), b.clone().requires_grad_(True)
    out = layers.dense(e, wl, bl, activation=act)
    assert out.shape == (0, 50)
    out.sum().backward()
    assert e.grad.shape == (0, 40) and not wl.grad.any() and not bl.grad.any()


@pytest.mark.gpu
def test_dense_gradient_against_differences():
  x, w, b, dy = make(9, 12, seed=1), make(12, 10, seed=2, scale=0.3), make(10, seed=3), make(9, 10, seed=4)
  for act in ('sigmoid', 'softplus', 'silu', 'gelu'):
    leaves = [v.requires_grad_(True) for v in dev(x, w, b)]
    layers.dense(*leaves, activation=act).backward(dy.cuda())
    for i, v in enumerate((x, w, b)):
      d = make(*v.shape, seed=7 + i).double()
      h = 1e-5
      at = lambda q: float((act64((x.double() + (q * d if i == 0 else 0)) @ (w.double() + (q * d if i == 1 else 0)) + b.double() + (q * d if i == 2 else 0), act)[0] * dy.double()).sum())
      slope = (at(h) - at(-h)) / (2 * h)
      got = float((leaves[i].grad.cpu().double() * d).sum())
      assert abs(got - slope) < 1e-4 * (1 + abs(slope)), (act, i, got, slope)      # h^2 of the difference (~1e-9) and float32 over some 100 terms


@pytest.mark.gpu
def test_dense_non_finite_inputs_stay_in_their_rows():
  for t in (F32, F16, BF16):
    x, w = make(140, 50, t=t, seed=1), make(50, 20, t=t, seed=2)
    x[3, 49], x[130, 0] = float('nan'), float('inf')
    y = layers.dense(*dev(x, w), activation='relu').cpu()
    rows = ~torch.isfinite(y).all(1)
    assert not torch.isfinite(y[3]).any() and rows[3] and rows[130] and int(rows.sum()) == 2


@pytest.mark.gpu
def test_dense_offsets_beyond_32_bits():
  m, k, n = (1 << 32) // 64 + 77, 64, 8      # more than 2^32 elements of x
  w = make(k, n, t=BF16, seed=1).cuda()
  x = torch.zeros((m, k), dtype=BF16, device='cuda')
  x[-130:] = make(130, k, t=BF16, seed=2).cuda()
  want = dense64(x[-130:].cpu(), w.cpu(), None, None, 'none', torch.ones(130, n, dtype=BF16))
  y = layers.dense(x, w)
  close(y[-130:], want['y'])
  assert not y[:1000].any()
  dx, dkernel, _ = layers.dense_backward(torch.ones_like(y), x, w, None, need_dbias=False)
  close(dx[-130:], want['dx'])
  close(dkernel, want['dkernel'])


# ---- layer norm ---------------------------------------------------------------------------------------------------------------------------------
def norm64(x, scale, bias, eps, dy):
  t = x.dtype
  u = half_step(t)
  x, d = x.double(), x.shape[1]
  one = torch.ones(d, dtype=torch.float64)
  w = one if scale is None else scale.double()
  b = 0 * one if bias is None else bias.double()
  chain = 64                                        # a lane adds at most 34 elements, then 8 partial sums
  mu = x.mean(1, keepdim=True)
  emu = (chain + 2) * E24 * x.abs().mean(1, keepdim=True)
  c = x - mu
  rstd = 1 / (c.square().mean(1, keepdim=True) + eps).sqrt()
  rel = (chain + 8) * E24 + emu * emu * rstd * rstd + 2 * E24 * c.abs().max(1, keepdim=True).values * rstd     # of rstd: the sum, emu enters squared
  xh = c * rstd
  ex = rstd * (emu + E24 * (x.abs() + mu.abs())) + xh.abs() * (rel + 2 * E24)
  y = xh * w + b
  out = {'y': (y, ex * w.abs() + 4 * E24 * (y.abs() + b.abs()) + u * y.abs() + tiny(t) + 1e-300)}
  dy = dy.double()
  h = dy * w
  m1, m2 = h.mean(1, keepdim=True), (h * xh).mean(1, keepdim=True)
  e1 = (chain + 2) * E24 * h.abs().mean(1, keepdim=True)
  e2 = (chain + 4) * E24 * (h * xh).abs().mean(1, keepdim=True) + (h.abs() * ex).mean(1, keepdim=True)
  dx = rstd * (h - m1 - xh * m2)
  edx = rstd * (e1 + ex * m2.abs() + xh.abs() * e2 + 4 * E24 * (h.abs() + m1.abs() + (xh * m2).abs())) + dx.abs() * (rel + 2 * E24)
  out['dx'] = (dx, edx + u * dx.abs() + tiny(t) + 1e-300)
  rows = min(x.shape[0], 512) + 64                   # rows a lane adds, then the partial sums
  v = (dy * xh).sum(0)
  out['dscale'] = (v, (dy.abs() * ex).sum(0) + rows * E24 * (dy * xh).abs().sum(0) + u * v.abs() + tiny(t) + 1e-300)
  v = dy.sum(0)
  out['dbias'] = (v, rows * E24 * dy.abs().sum(0) + u * v.abs() + tiny(t) + 1e-300)
  return out


NORM_SHAPES = [(1, 1), (5, 1), (3, 2), (1, 256), (33, 8), (7, 33), (70, 64), (31, 65), (9, 129), (300, 256), (6, 511), (5, 513), (13, 1023), (4, 1025), (3, 2049), (3, 4100),
               (2, 8192), (2, 8200), (3000, 24)]


@pytest.mark.gpu
@pytest.mark.parametrize('t', [F32, F16, BF16], ids=['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('i', range(len(NORM_SHAPES)), ids=['x'.join(map(str, s)) for s in NORM_SHAPES])
def test_layer_norm_and_its_gradients(i, t):
  m, d = NORM_SHAPES[i]
  x, dy = make(m, d, t=t, seed=1, scale=1.5, shift=0.5), make(m, d, t=t, seed=2)
  scale = make(d, t=t, seed=3, scale=0.2, shift=1.0) if i % 3 else None
  bias = make(d, t=t, seed=4) if i % 2 else None
  want = norm64(x, scale, bias, 1e-6, dy)
  leaves = [v.requires_grad_(True) if v is not None else None for v in dev(x, scale, bias)]
  y = layers.layer_norm(*leaves)
  close(y, want['y'])
  close(layers.layer_norm(*dev(x, scale, bias)), want['y'])
  y.backward(dy.cuda())
  for name, v in zip(('dx', 'dscale', 'dbias'), leaves):
    if v is not None:
      close(v.grad, want[name], name)


@pytest.mark.gpu
def test_layer_norm_far_mean_constant_rows_views_and_no_rows():
  x = make(40, 300, seed=1, scale=1e-2, shift=100.0)      # a difference of squares would keep no digit of this variance
  x[7] = 0.1                                               # a constant row: bias comes out
  dy = make(40, 300, seed=2)
  want = norm64(x, None, None, 1e-6, dy)
  y, stats = layers.layer_norm_forward(x.cuda())
  close(y, want['y'])
  close(layers.layer_norm_backward(*dev(dy, x), None, stats, need_dscale=False, need_dbias=False)[0], want['dx'])
  big = make(20, 101, seed=3).cuda()
  v = big[:, 1:98]
  want = norm64(v.cpu(), None, None, 0.1, v.cpu())
  y, stats = layers.layer_norm_forward(v, epsilon=0.1)
  close(y, want['y'])
  close(layers.layer_norm_backward(v, v, None, stats)[0], want['dx'])
  close(layers.layer_norm(v.reshape(4, 5, 97), epsilon=0.1), want['y'])
  s = torch.ones(97, device='cuda').requires_grad_(True)
  e = v[:0].clone().requires_grad_(True)
  layers.layer_norm(e, s).sum().backward()
  assert e.grad.shape == (0, 97) and not s.grad.any()


@pytest.mark.gpu
def test_layer_norm_gradient_against_differences_and_what_is_asked_for():
  x, s, b, dy = make(6, 20, seed=1), make(20, seed=2, shift=1.0), make(20, seed=3), make(6, 20, seed=4)
  leaves = [v.requires_grad_(True) for v in dev(x, s, b)]
  layers.layer_norm(*leaves).backward(dy.cuda())

  def f(xx, ss, bb):
    return float((norm64_value(xx, ss, bb) * dy.double()).sum())
  def norm64_value(xx, ss, bb):
    c = xx - xx.mean(1, keepdim=True)
    return c / (c.square().mean(1, keepdim=True) + 1e-6).sqrt() * ss + bb
  for i, v in enumerate((x, s, b)):
    d = make(*v.shape, seed=7 + i).double()
    args = [q.double() for q in (x, s, b)]
    hi, lo = list(args), list(args)
    hi[i], lo[i] = args[i] + 1e-5 * d, args[i] - 1e-5 * d
    slope = (f(*hi) - f(*lo)) / 2e-5
    got = float((leaves[i].grad.cpu().double() * d).sum())
    assert abs(got - slope) < 1e-4 * (1 + abs(slope)), (i, got, slope)
  _, stats = layers.layer_norm_forward(*dev(x, s, b))
  full = layers.layer_norm_backward(*dev(dy, x, s), stats)
  for need in range(8):
    flags = [bool(need >> i & 1) for i in range(3)]
    got = layers.layer_norm_backward(*dev(dy, x, s), stats, need_dx=flags[0], need_dscale=flags[1], need_dbias=flags[2])
    for fl, g, ref in zip(flags, got, full):
      assert (g is None) != fl and (g is None or torch.equal(g, ref))


# ---- orthogonalised updates ------------------------------------------------------------------------------------------------------------------------
def ortho64(u, steps=5):
  x = u.double()
  n = x.norm()
  x = x / n if n > 1e-30 else x * 0
  tall = x.shape[0] > x.shape[1]
  x = x.t() if tall else x
  for _ in range(steps):
    a = x @ x.t()
    x = 3.4445 * x + (-4.7750 * a + 2.0315 * a @ a) @ x
  return x.t() if tall else x


# Relative error of the result (2-norm over all elements): a singular value and its error grow by the same factor while the value is small, so relative
# errors add up over the 3 products of each of the steps, each 2^-22 (two f16 planes a side) times |a| + |b| + |c| = 10
def ortho_bound(t, steps=5):
  return steps * 3 * 10 * 2.0 ** -22 + (half_step(t) if t != F32 else 0.0)


ORTHO_SHAPES = [(1, 1), (1, 7), (9, 1), (3, 5), (64, 64), (63, 65), (65, 64), (128, 45), (256, 256), (130, 517), (560, 128), (20, 3001)]


@pytest.mark.gpu
@pytest.mark.parametrize('t', [F32, F16, BF16], ids=['f32', 'f16', 'bf16'])
def test_orthogonalize_alone_and_in_one_call(t):
  mats = [make(r, c, t=t, seed=10 + i, scale=0.01) for i, (r, c) in enumerate(ORTHO_SHAPES)]
  mats[4] = (make(64, 6, seed=1) @ make(6, 64, seed=2)).to(t)             # low rank: most singular values are roundings
  got = optim.orthogonalize(dev(*mats))
  for u, o in zip(mats, got):
    want = ortho64(u)
    err = float((o.cpu().double() - want).norm() / want.norm())
    assert o.dtype == t and o.shape == u.shape and err < ortho_bound(t), (tuple(u.shape), err)
    assert torch.equal(optim.orthogonalize(u.cuda()), o), tuple(u.shape)        # the same bits alone and among others
  s = torch.linalg.svdvals(got[8].double().cpu())
  assert float(s.max()) < 1.21 and float(s[:200].min()) > 0.6


@pytest.mark.gpu
def test_orthogonalize_extreme_values_zero_and_non_finite_matrices():
  u = make(70, 90, seed=1)
  want = ortho64(u)
  one = torch.zeros(70, 90)
  one[3, 80] = -1e-20
  bad = u.clone()
  bad[0, 0] = float('inf')
  got = optim.orthogonalize(dev(u * 1e30, u * 1e-25, torch.zeros(70, 90), bad, one, u))
  for o in (got[0], got[1], got[5]):
    assert float((o.cpu().double() - want).norm() / want.norm()) < ortho_bound(F32) + 2 * E24
  assert not got[2].any() and torch.isnan(got[3]).all()
  assert float((got[4].cpu().double() - ortho64(one)).abs().max()) < 1e-4
  for steps in (1, 2, 7, 16):
    want = ortho64(u, steps)
    assert float((optim.orthogonalize(u.cuda(), steps=steps).cpu().double() - want).norm() / want.norm()) < ortho_bound(F32, steps) * 4


@pytest.mark.gpu
def test_orthogonalize_many_matrices_views_and_empty_ones():
  big = make(300, 400, seed=1).cuda()
  mats = [big[i:i + 5 + i % 30, 3 * i:3 * i + 40 - i % 17] for i in range(70)] + [big.t()[:50, :60], big[:0], big[:, :0]]     # two launches' worth
  got = optim.orthogonalize(mats)
  for u, o in zip(mats, got):
    assert o.shape == u.shape and o.is_contiguous()
    if u.numel():
      want = ortho64(u.cpu())
      assert float((o.cpu().double() - want).norm() / want.norm()) < ortho_bound(F32), tuple(u.shape)
  assert optim.orthogonalize([]) == []


# ---- streams, graphs, repetition -------------------------------------------------------------------------------------------------------------------
def _block(p, dy):
  """A pre-norm residual block, its gradients and their orthogonalisation, as a user's step runs them - without autograd, so it can be captured."""
  h, stats = layers.layer_norm_forward(p['x'], p['s'], p['b'])
  a, saved = layers.dense_forward(h, p['w1'], p['b1'], 'gelu')
  y, _ = layers.dense_forward(a, p['w2'], None, 'none', residual=p['x'])
  da, dw2, _ = layers.dense_backward(dy, a, p['w2'], None, need_dbias=False)
  dh, dw1, db1 = layers.dense_backward(da, h, p['w1'], saved, 'gelu')
  dx, ds, db = layers.layer_norm_backward(dh, p['x'], p['s'], stats)
  o1, o2 = optim.orthogonalize([dw1, dw2])
  return y, dx + dy, ds, db, dw1, db1, dw2, o1, o2


def _block_state(seed, t=F32, m=200, d=96, hidden=160):
  p = dict(x=make(m, d, t=t, seed=seed), s=make(d, t=t, seed=seed + 1, shift=1.0), b=make(d, t=t, seed=seed + 2), w1=make(d, hidden, t=t, seed=seed + 3, scale=0.1),
           b1=make(hidden, t=t, seed=seed + 4), w2=make(hidden, d, t=t, seed=seed + 5, scale=0.1))
  return {k: v.cuda() for k, v in p.items()}, make(m, d, t=t, seed=seed + 6).cuda()


@pytest.mark.gpu
def test_block_against_autograd_in_64_bits_and_repeats_bit_for_bit():
  p, dy = _block_state(1)
  q = {k: v.cpu().double().requires_grad_(True) for k, v in p.items()}
  c = q['x'] - q['x'].mean(1, keepdim=True)
  h = c / (c.square().mean(1, keepdim=True) + 1e-6).sqrt() * q['s'] + q['b']
  y = q['x'] + torch.nn.functional.gelu(h @ q['w1'] + q['b1']) @ q['w2']
  y.backward(dy.cpu().double())
  got = _block(p, dy)
  want = [y] + [q[k].grad for k in ('x', 's', 'b', 'w1', 'b1', 'w2')] + [ortho64(q[k].grad) for k in ('w1', 'w2')]
  for i, (g, v) in enumerate(zip(got, want)):      # five float32 stages, the longest sum 200 terms: 5 x 200 x 2^-24 of the norm at the most
    assert float((g.cpu().double() - v).norm() / v.norm()) < 1000 * E24, i
  leaves = {k: v.clone().requires_grad_(True) for k, v in p.items()}
  a = layers.dense(layers.layer_norm(leaves['x'], leaves['s'], leaves['b']), leaves['w1'], leaves['b1'], activation='gelu')
  layers.dense(a, leaves['w2'], residual=leaves['x']).backward(dy)
  for k, v in zip(('s', 'b', 'w1', 'b1', 'w2'), got[2:7]):
    assert torch.equal(leaves[k].grad, v), k
  for _ in range(3):
    for a, b in zip(_block(p, dy), got):
      assert torch.equal(a, b)


@pytest.mark.gpu
def test_two_captured_graphs_replay_with_eager_work_between():
  states = [_block_state(1), _block_state(20)]
  eager = [[v.clone() for v in _block(*s)] for s in states]
  graphs = []
  side = torch.cuda.Stream()
  for s in states:
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
      _block(*s)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
      out = _block(*s)
    graphs.append((g, out))
  for turn in range(3):
    for (g, out), want in zip(graphs, eager):
      for o in out:
        o.zero_()
      g.replay()
      fresh = _block(*states[turn % 2])
      torch.cuda.synchronize()
      for a, b in zip(out, want):
        assert torch.equal(a, b)
      for a, b in zip(fresh, eager[turn % 2]):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_other_streams_and_the_current_device():
  states = [_block_state(40 + i) for i in range(3)]
  want = [_block(*s) for s in states]
  torch.cuda.synchronize()
  streams = [torch.cuda.Stream() for _ in states]
  got = []
  for st, s in zip(streams, states):
    with torch.cuda.stream(st):
      got.append(_block(*s))
  torch.cuda.synchronize()
  for a, b in zip(got, want):
    for x, y in zip(a, b):
      assert torch.equal(x, y)
  assert torch.cuda.current_device() == 0
  if torch.cuda.device_count() > 1:
    x = make(5, 6, seed=1)
    assert torch.equal(layers.layer_norm(x.to('cuda:1')).cpu(), layers.layer_norm(x.cuda()).cpu()) and torch.cuda.current_device() == 0


# ---- refusals (no GPU needed: every check comes before the device) -------------------------------------------------------------------------------------
def test_python_refusals():
  x = torch.zeros(4, 8)
  for f in (lambda: layers.dense(x, torch.zeros(8, 3)), lambda: layers.layer_norm(x), lambda: optim.orthogonalize(x), lambda: optim.orthogonalize([x])):
    with pytest.raises(RuntimeError, match='no CPU path'):
      f()
  with pytest.raises(ValueError, match='steps'):
    optim.orthogonalize(x, steps=0)
  with pytest.raises(ValueError, match='2-d'):
    optim.orthogonalize([torch.zeros(3)])
  with pytest.raises(ValueError, match='at least one axis'):
    layers.dense(torch.tensor(1.0), torch.zeros(1, 1))


@pytest.mark.gpu
def test_python_refusals_on_the_gpu():
  x, w = torch.zeros(4, 8, device='cuda'), torch.zeros(8, 3, device='cuda')
  cases = [(lambda: layers.dense(x, w.half()), 'kernel must be'), (lambda: layers.dense(x, w.cpu()), 'kernel must be'), (lambda: layers.dense(x, w[:7]), 'does not fit'),
           (lambda: layers.dense(x, w[:, :0]), 'does not fit'), (lambda: layers.dense(x.double(), w.double()), 'element type'), (lambda: layers.dense(x, w, activation='tanh'), 'activation'),
           (lambda: layers.dense(x, w, torch.zeros(4, device='cuda')), 'bias'), (lambda: layers.dense(x, w, residual=x), 'residual'),
           (lambda: layers.dense_backward(x[:, :3], x, w, None, 'relu'), 'saved'), (lambda: layers.dense_backward(x, x, w, None), 'dy'),
           (lambda: layers.layer_norm(x, w[:, 0][:3]), 'scale'), (lambda: layers.layer_norm(x, epsilon=-1.0), 'epsilon'), (lambda: layers.layer_norm(x[:, :0]), 'last axis'),
           (lambda: layers.layer_norm(x, epsilon=float('nan')), 'epsilon'), (lambda: layers.layer_norm_backward(x, x, None, torch.zeros(4, 2)), 'stats'),
           (lambda: optim.orthogonalize([x, x.half()]), 'one element type'), (lambda: optim.orthogonalize(torch.zeros(1, 40000, device='cuda')), '40000')]
  for f, text in cases:
    with pytest.raises(ValueError, match=text):
      f()
  x.requires_grad_(True)
  for y in (layers.dense(x, w), layers.layer_norm(x, w[:, 0].contiguous())):      # first order only, and said so
    (g,) = torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
    with pytest.raises(RuntimeError):
      g.sum().backward()


def test_c_refusals():
  lib = N.load()
  EINVAL, EDEVICE = -22, -5
  buf = (C.c_float * 1024)()
  p = (C.addressof(buf) + 255) // 256 * 256      # never reached: every call below is refused on the host

  def fwd(**kw):
    a = N.DenseForwardArgs(0, 0, 4, 4, 4, p, 4, p, 4, None, None, 0, p, 4, None)
    for k, v in kw.items():
      setattr(a, k, v)
    return lib.nerfds_dense_forward(0, C.byref(a), None)

  def bwd(**kw):
    a = N.DenseBackwardArgs(0, 0, 4, 4, 4, p, 4, p, 4, p, 4, None, p, 4, p, p, p, 1 << 20)
    for k, v in kw.items():
      setattr(a, k, v)
    return lib.nerfds_dense_backward(0, C.byref(a), None)

  def nfwd(**kw):
    a = N.LayerNormForwardArgs(0, 4, 4, 1e-6, p, 4, None, None, p, 4, None)
    for k, v in kw.items():
      setattr(a, k, v)
    return lib.nerfds_layer_norm_forward(0, C.byref(a), None)

  def nbwd(**kw):
    a = N.LayerNormBackwardArgs(0, 4, 4, p, 4, None, p, 4, p, p, 4, p, p, p, 1 << 20)
    for k, v in kw.items():
      setattr(a, k, v)
    return lib.nerfds_layer_norm_backward(0, C.byref(a), None)

  bad = [dict(dtype=3), dict(dtype=-1), dict(m=-1), dict(m=1 << 41), dict(x=None), dict(x=p + 1), dict(ldx=3)]
  for kw in bad + [dict(activation=6), dict(k=0), dict(n=0), dict(kernel=None), dict(ldk=3), dict(y=None), dict(ldy=2), dict(bias=p + 2), dict(residual=p, ldr=3),
                   dict(m=1 << 40, n=1 << 20), dict(activation=2, save=p + 2)]:
    assert fwd(**kw) == EINVAL, kw
    assert b'nerfds_dense_forward' in lib.nerfds_last_error(None)
  for kw in bad + [dict(activation=-1), dict(n=0), dict(dy=None), dict(lddy=3), dict(lddx=1), dict(activation=1), dict(dkernel=p + 1)]:
    assert bwd(**kw) == EINVAL, kw
  for kw in bad + [dict(d=0), dict(epsilon=-1.0), dict(epsilon=float('inf')), dict(epsilon=float('nan')), dict(y=None), dict(ldy=1), dict(scale=p + 3)]:
    assert nfwd(**kw) == EINVAL, kw
  for kw in bad + [dict(d=-4), dict(dy=None), dict(stats=None), dict(lddx=1), dict(dbias=p + 1)]:
    assert nbwd(**kw) == EINVAL, kw
  for f in (lib.nerfds_dense_forward, lib.nerfds_dense_backward, lib.nerfds_layer_norm_forward, lib.nerfds_layer_norm_backward):
    assert f(0, None, None) == EINVAL
  assert fwd(m=0, x=None) == 0 and nfwd(m=0, y=None) == 0

  def ortho(dtype=0, count=1, steps=5, ws=p, nbytes=1 << 20, **kw):
    mat = N.Matrix(p, 100, p, 100, 100, 100)      # (large enough to need a workspace)
    for k, v in kw.items():
      setattr(mat, k, v)
    return lib.nerfds_orthogonalize(0, dtype, C.byref(mat), count, steps, ws, nbytes, None)
  for kw in (dict(dtype=9), dict(count=-1), dict(steps=0), dict(steps=17), dict(ws=None), dict(ws=p + 8), dict(nbytes=16), dict(rows=0), dict(cols=-1), dict(rows=40000), dict(u=None),
             dict(ldu=99), dict(ldo=99), dict(o=p + 1)):
    assert ortho(**kw) == EINVAL, kw
  assert ortho(count=0) == 0 and lib.nerfds_orthogonalize(0, 0, None, 1, 5, p, 1 << 20, None) == EINVAL
  assert lib.nerfds_dense_save_bytes(1, 1, 5, 9) == 10 and lib.nerfds_dense_save_bytes(0, 5, 5, 9) == 180 and lib.nerfds_dense_save_bytes(2, 0, 5, 9) == 0
  assert lib.nerfds_dense_save_bytes(2, 7, 5, 9) == EINVAL
  a = N.DenseForwardArgs(0, 0, 4, 4, 4, p, 4, p, 4, None, None, 0, p, 4, None)
  assert lib.nerfds_dense_forward(1000, C.byref(a), None) == EDEVICE and lib.nerfds_dense_forward(-1, C.byref(a), None) == EDEVICE


def test_c_refuses_more_tiles_than_a_launch_holds():
  lib = N.load()
  p = 1 << 20      # never reached: refused on the host, on a machine with a GPU too
  for m, k, n in ((1 << 33, 4, 128), (1 << 33, 128, 4), (1 << 31, 1, 1), (4, 1 << 21, 1 << 19)):
    f = N.DenseForwardArgs(0, 0, m, k, n, p, k, p, n, None, None, 0, p, n, None)
    b = N.DenseBackwardArgs(0, 0, m, k, n, p, k, p, n, p, n, None, p, k, p, p, p, 1 << 20)
    assert lib.nerfds_dense_forward(0, C.byref(f), None) == -22 and lib.nerfds_dense_backward(0, C.byref(b), None) == -22
    assert b'tiles' in lib.nerfds_last_error(None)


@pytest.mark.gpu
@pytest.mark.parametrize('t', [F32, F16, BF16], ids=['f32', 'f16', 'bf16'])
def test_c_results_in_place(t):
  lib, code, dev_ = N.load(), N.dtype_code(t), torch.cuda.current_device()
  st = torch.cuda.current_stream().cuda_stream
  for m, k, n, act in ((1, 256, 256, 'relu'), (7, 33, 65, 'gelu'), (300, 64, 100, 'silu'), (20003, 64, 200, 'relu'), (4100, 520, 1056, 'relu')):
    x, w, b, r = dev(make(m, k, t=t, seed=1), make(k, n, t=t, seed=2, scale=k ** -0.5), make(n, t=t, seed=3), make(m, n, t=t, seed=4))
    want, saved = layers.dense_forward(x, w, b, act, r)
    save = torch.empty_like(saved)
    a = N.DenseForwardArgs(code, N.ACTIVATIONS[act], m, k, n, x.data_ptr(), k, w.data_ptr(), n, b.data_ptr(), r.data_ptr(), n, r.data_ptr(), n, save.data_ptr())
    assert lib.nerfds_dense_forward(dev_, C.byref(a), st) == 0
    assert torch.equal(r, want) and torch.equal(save, saved), (m, k, n)      # y == residual
  for m, d in ((5, 100), (33, 300), (9, 3000), (3, 9001)):
    x, s = dev(make(m, d, t=t, seed=5), make(d, t=t, seed=6))
    want = layers.layer_norm_forward(x, s)[0]
    a = N.LayerNormForwardArgs(code, d, m, 1e-6, x.data_ptr(), d, s.data_ptr(), None, x.data_ptr(), d, None)
    assert lib.nerfds_layer_norm_forward(dev_, C.byref(a), st) == 0
    assert torch.equal(x, want), (m, d)
  for shapes in ([(64, 64)], [(40, 130), (130, 40)], [(300, 200), (64, 64)], [(2000, 2047), (1100, 1000)]):
    us = dev(*(make(r, c, t=t, seed=7 + i) for i, (r, c) in enumerate(shapes)))
    want = optim.orthogonalize(us)
    mats = (N.Matrix * len(us))(*(N.Matrix(u.data_ptr(), u.shape[1], u.data_ptr(), u.shape[1], *u.shape) for u in us))
    nbytes = lib.nerfds_orthogonalize_workspace(mats, len(us))
    ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device='cuda')
    assert lib.nerfds_orthogonalize(dev_, code, mats, len(us), 5, ws.data_ptr(), nbytes, st) == 0
    assert all(torch.equal(u, o) for u, o in zip(us, want)), shapes


def test_struct_sizes_of_the_operators():
  lib = N.load()
  for which, st in ((9, N.DenseForwardArgs), (10, N.DenseBackwardArgs), (11, N.LayerNormForwardArgs), (12, N.LayerNormBackwardArgs), (13, N.Matrix)):
    assert lib.nerfds_struct_size(which) == C.sizeof(st)


# ---- the trainer's orthogonalised update -----------------------------------------------------------------------------------------------------------
def _trainer(**kw):
  from nerfds_amd import init_params, nerf_ds_config
  from nerfds_amd.training import Trainer
  cfg = nerf_ds_config(num_warp_embeds=4, num_coarse_samples=8, num_fine_samples=8)
  return Trainer(cfg, init_params(cfg, 0, warp_head_scale=5e-2, small_head_scale=0.3, bias_scale=0.1), max_rays=64, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize('nesterov', [True, False])
def test_trainer_with_orthogonalised_kernels(nesterov):
  beta, wd, lr = 0.9, 0.1, 1e-2
  muon = _trainer(optimizer='muon', optimizer_options=dict(momentum=beta, nesterov=nesterov, weight_decay=wd))
  adam = _trainer()
  names = muon.orthogonalized_leaves
  assert len(names) == 40 and 'nerf_mlps_fine/bottleneck/kernel' in names and adam.orthogonalized_leaves == []
  assert all('/hidden_' in n or 'bottleneck' in n for n in names) and not any('logit' in n or 'bias' in n or 'embed' in n for n in names)
  leaves = {name: (off, rows, cols) for name, off, rows, cols in muon.leaves}
  m = {n: 0.0 for n in names}
  w = {n: muon.params_tensor()[leaves[n][0]:leaves[n][0] + leaves[n][1] * leaves[n][2]].cpu().double().reshape(leaves[n][1:]) for n in names}
  for step in range(3):
    g = make(muon.num_params, seed=step, scale=1e-3).cuda()
    for tr in (muon, adam):
      tr.grads_tensor().copy_(g)
      torch.cuda.synchronize()
      tr.apply_gradients(lr)
    got, ref, first = (x.cpu() for x in (muon.params_tensor(), adam.params_tensor(), g))
    ema = torch.as_tensor(muon._download(2))
    rest = torch.ones(muon.num_params, dtype=torch.bool)
    for n in names:
      off, rows, cols = leaves[n]
      gi = first[off:off + rows * cols].double().reshape(rows, cols)
      m[n] = beta * m[n] + gi
      o = ortho64((gi + beta * m[n] if nesterov else m[n]))
      w[n] = w[n] * (1 - lr * wd) - lr * 0.2 * math.sqrt(max(rows, cols)) * o
      err = got[off:off + rows * cols].double().reshape(rows, cols) - w[n]
      assert float(err.norm()) < float((step + 1) * (4 * E24 * w[n].norm() + lr * 0.2 * math.sqrt(max(rows, cols)) * (ortho_bound(F32) + 8 * E24) * o.norm())), n
      assert float((ema[off:off + rows * cols].double().reshape(rows, cols) - m[n]).abs().max()) <= 4 * E24 * float(m[n].abs().max())
      rest[off:off + rows * cols] = False
    # the other leaves: Adam's formula in another kernel, whose multiply-adds may be fused elsewhere: per step the moments differ by 2 roundings each, quotient,
    # root and product by 4 more, the update (at most 0.1 / sqrt(0.001) = 3.2 lr, the first step's bias correction aside, which makes it lr) by 8 x 2^-24 of itself, the parameter by one
    assert float((got[rest] - ref[rest]).abs().max()) <= (step + 1) * E24 * (8 * 3.2 * lr + float(ref[rest].abs().max()))
  assert muon.optimizer_step == 3 and not muon.nonfinite()
  before, moments = muon._download(0), muon._download(2)
  g[5] = float('inf')
  muon.grads_tensor().copy_(g)
  torch.cuda.synchronize()
  muon.apply_gradients(lr)
  assert muon.nonfinite() and muon.optimizer_step == 3 and (muon._download(0) == before).all() and (muon._download(2) == moments).all()
  muon.set_optimizer('adam')
  assert muon.optimizer_step == 0 and not muon._download(2).any() and muon.orthogonalized_leaves == []


@pytest.mark.gpu
def test_trainer_steps_and_resumes_with_orthogonalised_kernels():
  import numpy as np
  rng = np.random.default_rng(0)
  d = rng.normal(size=(64, 3))
  d /= np.linalg.norm(d, axis=-1, keepdims=True)
  batch = dict(origins=rng.normal(size=(64, 3)) * 0.1, directions=d, rgb=rng.random((64, 3)), metadata={'warp': rng.integers(0, 4, (64, 1))}, mask=np.zeros((64, 1)))
  extra = dict(nerf_alpha=8., warp_alpha=4., hyper_alpha=1., hyper_sheet_alpha=6., norm_input_alpha=4.)
  a, b = _trainer(optimizer='muon'), _trainer(optimizer='muon')
  a.step(batch, extra, 1e-3, seed=1)
  b.set_params(a.get_params())
  b.set_opt_state(*a.get_opt_state(), a.optimizer_step)
  for tr in (a, b):
    stats = tr.step(batch, extra, 1e-3, seed=2)
    assert math.isfinite(stats['loss/total']) and tr.optimizer_step == 2
  # The step's gradients are sums of float32 atomics, equal up to their order: 1e-5 of a kernel's gradient at the most, which the orthogonalisation
  # multiplies by 3.4445^5 = 485 at the most: 5e-3 of an element of O, times lr 0.2 sqrt(560) = 4.7e-3 (and again for the momentum: 5e-5)
  pa, pb = a._download(0), b._download(0)
  for name, off, rows, cols in a.leaves:
    if name in a.orthogonalized_leaves:
      assert np.abs(pa[off:off + rows * cols] - pb[off:off + rows * cols]).max() < 5e-5, name
  for kw in (dict(momentum=1.0), dict(momentum=-0.1), dict(steps=0), dict(steps=17), dict(weight_decay=-1.0), dict(weight_decay=float('nan')), dict(momentum=float('nan'))):
    with pytest.raises(ValueError):
      a.set_optimizer('muon', **kw)
  with pytest.raises(ValueError, match='unknown optimizer'):
    a.set_optimizer('sgd')
