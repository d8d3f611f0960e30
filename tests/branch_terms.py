"""The gradient of a residual branch term by term in 64 bits, and how far float32 arithmetic may take each of its values.

    yh = y r1,  b = yh A,  A = post_weight gate mask,  t = alpha x + b,  sh = t r2,  g = dh weight
    q = r2 (g - sh c1), c1 = mean(g sh),  dt = q + ds,  dx = alpha dt
    G = dt A,  dy = r1 (G - yh c2), c2 = mean(G yh)
    d_weight = sum dh sh,  d_post_weight = sum dt mask yh gate,  d_gate = sum dt mask yh post_weight

Bounds, with U = 2^-24 a rounding's share of a value, to first order (and 2 % more): a value's error is what its operands' errors
come to through its formula and U of each intermediate value.
  A root of a row: its sum takes at most 12 additions of a thread's, 6 in a warp and 5 over the warps, then 1 / d, the product and
  eps: 26 U of positive terms, half of it in the root, and rsqrtf's two units in the last place (4 U): ROOT = 20 U.
  yh: ROOT + U. A: 3 products. b: 27 U. t: 27 U |b| + U |alpha x| + U |t|, and r2 takes the root mean square of that times r2.
  A row's mean of products: at most 4 + 1 + 5 + 9 additions and the two of 1 / d: 24 U of the terms' absolute mean.
  A column's sum over rows: one addition for every row of a thread, those of up to 32 groups of threads and of the partials:
  rows / 64 + 128 at most, of the terms' absolute sum.
No term of another size than the value's own enters: a gradient without one of its two means is out of them at every width.
"""
import numpy as np
import torch

U = 2.0 ** -24
ROOT = 20 * U
F32, BF16 = torch.float32, torch.bfloat16


def inputs(shape, xd, yd, gate, wd, od, device, seed=0):
  """x, y, post_weight, weight, gate and the gradients of h and s, as a block's: values of order one in every row, the output's
  gradient partly along y and x, so that a row's means (c1, c2) are of order one too."""
  gen = torch.Generator(device=device).manual_seed(seed + shape[-1])
  rand = lambda *s: torch.randn(*s, device=device, generator=gen)  # noqa: E731
  d = shape[-1]
  x, y = rand(*shape).to(xd), (0.5 * rand(*shape)).to(yd)
  pw, w = ((1 + 0.2 * rand(d)).to(wd), (1 + 0.2 * rand(d)).to(wd)) if wd is not None else (None, None)
  gs = {None: None, "channel": (d,), "sample": shape[:-2] + (d,), "kept": shape[:-2] + (1, d), "value": shape}[gate]
  g = None if gs is None else (0.5 + 0.3 * rand(*gs)).to(yd if gate == "value" else F32)
  dh = (rand(*shape) + 0.5 * x.float() + 0.5 * y.float()).to(od)
  ds = (0.5 * rand(*shape) + 0.25 * y.float()).to(xd)
  return (x, y, pw, w, g), (dh, ds)


def mask_of(shape, p, seed, site, device):
  from oracle import dropout
  return torch.from_numpy(np.ascontiguousarray(dropout.factors(shape, p, seed, site))).to(device)


def gradients(ins, dh, ds, alpha, eps=1e-6, mask=None, without=()):
  """{name: (value, room)} of the gradients, float64. dh or ds may be None. `without`: "c1" or "c2" leaves that mean out."""
  x, y, pw, w, gate = [None if t is None else t.detach().double() for t in ins]
  shape, d = x.shape, x.shape[-1]
  rows = x.numel() // d
  one = torch.ones((), dtype=torch.float64, device=x.device)
  full = one if gate is None else gate.unsqueeze(-2) if gate.dim() == x.dim() - 1 and gate.dim() > 1 else gate
  p, m, wt = one if pw is None else pw, one if mask is None else mask, one if w is None else w
  mean = lambda v: v.mean(-1, keepdim=True)  # noqa: E731
  rms = lambda v: torch.sqrt(mean(v * v))  # noqa: E731
  r1 = 1 / torch.sqrt(mean(y * y) + eps)
  yh = y * r1
  a = (p * full * m).expand(shape)
  b = yh * a
  t = alpha * x + b
  r2 = 1 / torch.sqrt(mean(t * t) + eps)
  sh = t * r2
  zero = torch.zeros(shape, dtype=torch.float64, device=x.device)
  gh = zero if dh is None else dh.double()
  g = gh * wt
  c1 = mean(g * sh)
  diff = g - (0 if "c1" in without else sh * c1)
  q = r2 * diff
  dt = q + (zero if ds is None else ds.double())
  dx = alpha * dt
  G = dt * a
  c2 = mean(G * yh)
  diff2 = G - (0 if "c2" in without else yh * c2)
  dy = r1 * diff2

  root2 = ROOT + (28 * U * rms(b) + 2 * U * rms(alpha * x)) * r2 + U
  sh_off = r2 * (27 * U * b.abs() + U * t.abs()) + (root2 + 2 * U) * sh.abs()
  c1_off = mean(g.abs() * sh_off + U * (g * sh).abs()) + 24 * U * mean((g * sh).abs())
  q_off = r2 * (U * g.abs() + c1.abs() * sh_off + sh.abs() * c1_off + U * diff.abs()) + (root2 + U) * q.abs()
  dt_off = q_off + U * dt.abs()
  if dh is None:
    dt_off = zero
  G_off = a.abs() * dt_off + 5 * U * G.abs()
  c2_off = mean(yh.abs() * G_off + 21 * U * (G * yh).abs()) + 24 * U * mean((G * yh).abs())
  dy_off = r1 * (G_off + c2.abs() * 21 * U * yh.abs() + yh.abs() * c2_off + U * diff2.abs()) + 22 * U * dy.abs()
  steps = (rows / 64 + 128) * U
  out = {"x": (dx, abs(alpha) * dt_off + U * dx.abs()), "y": (dy, dy_off)}
  over = lambda v: v.reshape(-1, d).sum(0)  # noqa: E731
  if w is not None:
    out["weight"] = over(gh * sh), over(gh.abs() * sh_off) + steps * over((gh * sh).abs())
  e = dt * m * yh
  e_off = (m * yh).abs() * dt_off + 26 * U * e.abs()
  if pw is not None:
    out["post_weight"] = over(e * full), over(e_off * full.abs()) + steps * over((e * full).abs())
  if gate is not None:
    v, v_off = e * p, e_off * p.abs()
    if gate.shape == shape:
      out["gate"] = v, v_off
    elif gate.dim() == 1:
      out["gate"] = over(v), over(v_off) + steps * over(v.abs())
    else:
      out["gate"] = tuple(u.sum(-2).reshape(gate.shape) for u in (v, v_off + steps * v.abs()))
  return {k: (v, 1.02 * room) for k, (v, room) in out.items()}


def excess(got, want, room):
  """How far got (of some type) lies above its bound: half a step of the type and `room`; positive where it is out."""
  step = torch.finfo(got.dtype).eps / 2 * 1.0001
  off = (got.double() - want).abs() - step * want.abs() - room - 1e-38
  return torch.where(torch.isnan(off), torch.full_like(off, float("inf")), off).max().item()
