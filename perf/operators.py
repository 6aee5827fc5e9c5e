"""Measured cases of the dense layer, the layer norm and the orthogonalised update: their plain forms (``own = False``: elementary torch
operations in 32 bits, rounded once at the end) and the calls a user makes of the framework (``own = True``)."""
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'nerf-ds_amd'))

own = False

DTYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
ACTIVATIONS = ('none', 'relu', 'sigmoid', 'softplus', 'silu', 'gelu')
EPS = 1e-6
# The quintic of the orthogonalisation: x <- a x + b x^3 + c x^5 on every singular value
COEFFS = (3.4445, -4.7750, 2.0315)

# [in, out] of the hidden kernels of the nerf_ds graph, each with how often it occurs: mask, warp and hyper-sheet networks (shared by the levels),
# then trunk, bottleneck and rgb branch of both levels
NERF_DS = (((44, 128), 1), ((128, 128), 6), ((172, 128), 1), ((33, 128), 1), ((128, 128), 4), ((161, 128), 1), ((45, 64), 1), ((64, 64), 4),
           ((109, 64), 1), ((52, 256), 2), ((256, 256), 12), ((308, 256), 2), ((256, 256), 2), ((560, 128), 2))


def listed():
  return [
      # one row through a wide layer, as a per-frame embedding head is evaluated while rendering: latency
      dict(name='dense_one_row', op='dense', m=1, k=1024, n=1024, dtype='bf16', act='silu', bias=True, residual=False, grads=False),
      # the rgb branch's first layer over the samples of 160 rays, ragged in every size, trained in f16
      dict(name='dense_ragged_f16', op='dense', m=20011, k=172, n=131, dtype='f16', act='relu', bias=True, residual=False, grads=True),
      # a hidden layer over the 128 samples of the reference's 512-ray batch, in the reference's own float32, trained
      dict(name='dense_batch_f32', op='dense', m=65536, k=256, n=256, dtype='f32', act='softplus', bias=True, residual=False, grads=True),
      # a residual trunk layer over 4096 rays x 128 samples, trained in bf16: bound by memory
      dict(name='dense_trunk_bf16', op='dense', m=524288, k=256, n=256, dtype='bf16', act='relu', bias=True, residual=True, grads=True),
      # a wide layer over rays, trained in bf16: bound by the matrix pipe
      dict(name='dense_wide_bf16', op='dense', m=8192, k=2048, n=4096, dtype='bf16', act='gelu', bias=True, residual=True, grads=True),
      # one row between two layers of such a head: latency
      dict(name='norm_one_row', op='norm', m=1, d=256, dtype='f32', grads=False),
      # odd width, odd row count, float32, trained
      dict(name='norm_ragged_f32', op='norm', m=10007, d=1023, dtype='f32', grads=True),
      # trunk width over 4096 rays x 128 samples in bf16, trained: bound by memory
      dict(name='norm_trunk_bf16', op='norm', m=524288, d=256, dtype='bf16', grads=True),
      # wide rows in f16, trained
      dict(name='norm_wide_f16', op='norm', m=16384, d=4096, dtype='f16', grads=True),
      # one kernel of the hyper-sheet network: latency
      dict(name='ortho_one_small', op='ortho', shapes='64x64', dtype='f32'),
      # every hidden kernel of the nerf_ds graph, as the trainer's update takes them
      dict(name='ortho_nerf_ds', op='ortho', shapes=' '.join('%dx%d' % s for s, c in NERF_DS for _ in range(c)), dtype='f32'),
      # four wide kernels in bf16, tall and wide ones
      dict(name='ortho_wide_bf16', op='ortho', shapes='1024x4096 4096x1024 1024x4096 2000x2047', dtype='bf16'),
  ]


def _log_int(rng, lo, hi):
  return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
  op = rng.choice(('dense', 'norm', 'ortho'))
  dtype = rng.choice(('f32', 'f16', 'bf16'))
  if op == 'dense':
    grads = rng.random() < 0.6
    # (a float32 relu is drawn forward only: the sign of a pre-activation next to 0 is the rounding's, and one flipped sign of 10^7 is 3e-4 of a gradient)
    act = rng.choice([a for a in ACTIVATIONS if not (grads and dtype == 'f32' and a == 'relu')])
    while True:
      m, k, n = _log_int(rng, 1, 524288), _log_int(rng, 1, 4096), _log_int(rng, 1, 4096)
      if m * k * n <= 8192 * 2048 * 4096 // (2 if dtype == 'f32' else 1) and m * max(k, n) <= 524288 * 256 // (2 if dtype == 'f32' else 1):
        break
    return dict(op=op, m=m, k=k, n=n, dtype=dtype, act=act, bias=rng.random() < 0.8, residual=rng.random() < 0.4, grads=grads)
  if op == 'norm':
    while True:
      m, d = _log_int(rng, 1, 524288), _log_int(rng, 8, 8192)
      if m * d <= 524288 * 256 // (2 if dtype == 'f32' else 1):
        break
    return dict(op=op, m=m, d=d, dtype=dtype, grads=rng.random() < 0.6)
  while True:
    shapes = [(_log_int(rng, 1, 2048), _log_int(rng, 1, 2048)) for _ in range(rng.choice((1, 1, 2, 5, 12, 40)))]
    if sum(min(s) ** 2 * max(s) for s in shapes) <= 4 * 1024 * 1024 * 4096 and sum(r * c for r, c in shapes) <= 1 << 24:
      return dict(op=op, shapes=' '.join('%dx%d' % s for s in shapes), dtype=dtype)


def _shapes(case):
  return [tuple(int(v) for v in s.split('x')) for s in case['shapes'].split()]


def prepare(case, seed):
  g = torch.Generator(device='cuda').manual_seed(seed)
  t = DTYPES[case['dtype']]

  def normal(*shape, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=g, device='cuda') * scale + shift).to(t)

  s = dict(case)
  if case['op'] == 'dense':
    m, k, n = case['m'], case['k'], case['n']
    s['x'] = normal(m, k)
    s['kernel'] = normal(k, n, scale=math.sqrt(2.0 / (k + n)))      # the initialiser of the framework's kernels has this variance
    s['b'] = normal(n, scale=0.1) if case['bias'] else None
    s['r'] = normal(m, n) if case['residual'] else None
    s['dy'] = normal(m, n) if case['grads'] else None
  elif case['op'] == 'norm':
    m, d = case['m'], case['d']
    s['x'] = normal(m, d, scale=1.5, shift=0.3)
    s['scale'] = normal(d, scale=0.2, shift=1.0)
    s['b'] = normal(d, scale=0.1)
    s['dy'] = normal(m, d) if case['grads'] else None
  else:
    # what an update of a kernel looks like: a few strong directions over a broad floor
    s['u'] = []
    for r, c in _shapes(case):
      q = max(1, min(r, c) // 8)
      s['u'].append(((torch.randn((r, q), generator=g, device='cuda') @ torch.randn((q, c), generator=g, device='cuda')) / math.sqrt(q) * 1e-3 +
                     torch.randn((r, c), generator=g, device='cuda') * 1e-3).to(t))
  if case['op'] != 'ortho' and case['grads']:
    for name in ('x', 'kernel', 'scale', 'b', 'r'):
      if s.get(name) is not None:
        s[name].requires_grad_(True)
  return s


# ---- the plain forms ----------------------------------------------------------------------------------------------------------------------
def _act(z, act):
  """(act(z), act'(z))."""
  if act == 'none':
    return z, None
  if act == 'relu':
    return z.clamp_min(0), (z > 0).to(z.dtype)
  if act == 'sigmoid':
    y = torch.sigmoid(z)
    return y, y * (1 - y)
  if act == 'softplus':
    return z.clamp_min(0) + torch.log1p(torch.exp(-z.abs())), torch.sigmoid(z)
  if act == 'silu':
    y = torch.sigmoid(z)
    return z * y, y * (1 + z * (1 - y))
  phi = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
  return z * phi, phi + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))


def _plain_dense(s):
  t = s['x'].dtype
  x, kernel = s['x'].detach().float(), s['kernel'].detach().float()
  z = x @ kernel
  if s['b'] is not None:
    z = z + s['b'].detach().float()
  y, dact = _act(z, s['act'])
  if s['r'] is not None:
    y = y + s['r'].detach().float()
  out = dict(y=y.to(t))
  if s['grads']:
    dy = s['dy'].float()
    dz = dy if dact is None else dy * dact
    out['dx'] = (dz @ kernel.t()).to(t)
    # (a float32 result that is a sum over more than 10^5 rows: in 64 bits, the 32-bit product loses a decimal there)
    out['dkernel'] = (x.t() @ dz if t != torch.float32 or s['m'] <= 100000 else x.double().t() @ dz.double()).to(t)
    if s['b'] is not None:
      out['db'] = dz.sum(0).to(t)
    if s['r'] is not None:
      out['dr'] = dy.to(t)
  return out


def _plain_norm(s):
  t = s['x'].dtype
  x, scale, b = s['x'].detach().float(), s['scale'].detach().float(), s['b'].detach().float()
  c = x - x.mean(1, keepdim=True)
  rstd = torch.rsqrt((c * c).mean(1, keepdim=True) + EPS)
  xh = c * rstd
  out = dict(y=(xh * scale + b).to(t))
  if s['grads']:
    dy = s['dy'].float()
    h = dy * scale
    out['dx'] = (rstd * (h - h.mean(1, keepdim=True) - xh * (h * xh).mean(1, keepdim=True))).to(t)
    out['dscale'] = (dy * xh).sum(0).to(t)
    out['db'] = dy.sum(0).to(t)
  return out


def _plain_ortho(s):
  a, b, c = COEFFS
  out = []
  for u in s['u']:
    x = u.double()
    x = (x / x.square().sum().sqrt().clamp_min(1e-30)).float()      # the norm is a long sum: in 64 bits
    if u.shape[0] > u.shape[1]:
      x = x.t()
    for _ in range(5):
      p = x @ x.t()
      x = a * x + (b * p + c * (p @ p)) @ x
    out.append((x.t() if u.shape[0] > u.shape[1] else x).contiguous().to(u.dtype))
  return out


# ---- the framework's calls ------------------------------------------------------------------------------------------------------------------
def _own(s):
  from nerfds_amd import layers, optim
  if s['op'] == 'ortho':
    return optim.orthogonalize(s['u'])
  if s['op'] == 'dense':
    wanted = [('dx', s['x']), ('dkernel', s['kernel']), ('db', s['b']), ('dr', s['r'])]
    y = layers.dense(s['x'], s['kernel'], s['b'], activation=s['act'], residual=s['r'])
  else:
    wanted = [('dx', s['x']), ('dscale', s['scale']), ('db', s['b'])]
    y = layers.layer_norm(s['x'], s['scale'], s['b'], epsilon=EPS)
  out = dict(y=y.detach())
  if s['grads']:
    wanted = [w for w in wanted if w[1] is not None]
    out.update(zip((w[0] for w in wanted), torch.autograd.grad(y, [w[1] for w in wanted], s['dy'])))
  return out


def run(state):
  if own:
    return _own(state)
  return {'dense': _plain_dense, 'norm': _plain_norm, 'ortho': _plain_ortho}[state['op']](state)


def work(case):
  e = 4 if case['dtype'] == 'f32' else 2
  if case['op'] == 'dense':
    m, k, n = case['m'], case['k'], case['n']
    cells = m * k + k * n + n * case['bias'] + m * n * (1 + case['residual'])
    flops = 2 * m * k * n
    if case['grads']:      # x and the kernel are counted once: the pass as a whole reads them at least once
      cells += m * n + m * k + k * n + n * case['bias']
      flops *= 3
    return dict(bytes=cells * e, flops=flops)
  if case['op'] == 'norm':
    m, d = case['m'], case['d']
    return dict(bytes=(2 * m * d + 2 * d + case['grads'] * (2 * m * d + 2 * d)) * e, flops=m * d * (20 if case['grads'] else 8))
  cells = flops = 0
  for r, c in _shapes(case):
    n, m = min(r, c), max(r, c)
    cells += 2 * r * c
    flops += 5 * (n * n * m + n ** 3 + 2 * n * n * m)      # the two symmetric products need half of their elements only
  return dict(bytes=cells * e, flops=flops)


def exact(case, seed):
  """The definitions in 64 bits."""
  s = prepare(case, seed)
  f = lambda v: None if v is None else v.detach().to(torch.float64)
  if case['op'] == 'ortho':
    out = []
    for u in s['u']:
      x = f(u)
      x = x / max(float(torch.linalg.vector_norm(x)), 1e-30)
      tall = x.shape[0] > x.shape[1]
      for _ in range(5):
        gram = x.t() @ x if tall else x @ x.t()
        poly = COEFFS[0] * torch.eye(gram.shape[0], dtype=gram.dtype, device=gram.device) + COEFFS[1] * gram + COEFFS[2] * (gram @ gram)
        x = x @ poly if tall else poly @ x
      out.append(x)
    return out
  if case['op'] == 'norm':
    x, scale, b, dy = f(s['x']), f(s['scale']), f(s['b']), f(s['dy'])
    d = x.shape[1]
    mu = x.sum(1, keepdim=True) / d
    sd = ((x - mu).square().sum(1, keepdim=True) / d + EPS).sqrt()
    hat = (x - mu) / sd
    out = dict(y=scale * hat + b)
    if dy is not None:
      w = dy * scale
      out['dx'] = (w - w.sum(1, keepdim=True) / d - hat * ((w * hat).sum(1, keepdim=True) / d)) / sd
      out['dscale'], out['db'] = (dy * hat).sum(0), dy.sum(0)
    return out
  x, kernel, b, r, dy = f(s['x']), f(s['kernel']), f(s['b']), f(s['r']), f(s['dy'])
  z = torch.matmul(x, kernel) + (0 if b is None else b)
  act = case['act']
  sig = 1 / (1 + torch.exp(-z))
  cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
  value = dict(none=lambda: z, relu=lambda: torch.where(z > 0, z, 0.0), sigmoid=lambda: sig, softplus=lambda: torch.logaddexp(z, torch.zeros_like(z)), silu=lambda: z * sig,
               gelu=lambda: z * cdf)[act]()
  out = dict(y=value if r is None else value + r)
  if dy is not None:
    slope = dict(none=lambda: torch.ones_like(z), relu=lambda: (z > 0).double(), sigmoid=lambda: sig * (1 - sig), softplus=lambda: sig, silu=lambda: sig + z * sig * (1 - sig),
                 gelu=lambda: cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi))[act]()
    dz = dy * slope
    out['dx'], out['dkernel'] = torch.matmul(dz, kernel.t()), torch.matmul(x.t(), dz)
    if b is not None:
      out['db'] = dz.sum(0)
    if r is not None:
      out['dr'] = dy
  return out
