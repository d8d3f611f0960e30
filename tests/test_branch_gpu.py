"""GPU: dropout and the norms around a residual branch against their formulas in 64 bits, at the sizes, types, strides and
masks where they can go wrong; captured graphs, streams, refusals.

Tolerances. A result rounded to type t is off by finfo(t).eps / 2 of itself. Before that the kernels compute in float32: a
norm's root is good to (d / 64 + 16) 2^-24 (sums of d squares, over at least 8 threads in exchanges), a value is the product
of at most six factors and a sum of two or three terms: (d / 64 + 40) 2^-24 of the terms bounds it. The terms of s are
residual_scale x and the branch, which may cancel: with T the row's largest sum of their absolute values, s is off by
(d / 64 + 40) 2^-24 T at most, and what is divided by s's root mean square R by T / R times as much of itself (a row of one
column, or of a few, can have T far above R). Column sums add a term for each row in at most rows / 64 + 80 steps.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16, E4M3 = torch.float32, torch.bfloat16, torch.float8_e4m3fn
U = 2.0 ** -24


def _randn(seed):
  g = torch.Generator(device="cuda").manual_seed(seed)
  return lambda *s: torch.randn(*s, device="cuda", generator=g)


def _mask(shape, p, seed, site):
  from oracle import dropout
  return torch.from_numpy(np.ascontiguousarray(dropout.factors(shape, p, seed, site))).cuda()


def _close(got, want, room, label=""):
  """got, of some type, against float64: half a step of the type, and `room` (absolute, broadcast)."""
  assert got.shape == want.shape, label
  step = torch.finfo(got.dtype).eps / 2 * 1.0001
  off = (got.double() - want).abs() - step * want.abs() - room - 1e-38
  assert not (off > 0).any(), f"{label}: {off.max().item():.3e} above its bound"
  assert not torch.isnan(got.double()).any(), label


# ---- dropout --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (4096,), (4099,), (333, 515), (3, 5, 1001), (2, 8191)])
def test_dropout_values_and_gradient(cuda, dtype, shape):
  from faster_weathernext import branch
  rand = _randn(len(shape) + shape[-1])
  x, dy = rand(*shape).to(dtype).requires_grad_(), rand(*shape).to(dtype)
  y = branch.dropout(x, 0.3, 1234567890123, site=5)
  d_x, = torch.autograd.grad(y, x, dy)
  m = _mask(shape, 0.3, 1234567890123, 5)
  room = 0.0 if dtype is BF16 else 2 * U * m.max()
  _close(y.detach(), x.detach().double() * m, room * x.detach().abs().double())
  _close(d_x, dy.double() * m, room * dy.abs().double())
  assert torch.equal(y == 0, (m == 0) | (x == 0))


@pytest.mark.parametrize("p", [0.0, 2.0 ** -17, 2.0 ** -16, 0.5, 1 - 2.0 ** -16, 1.0])
def test_dropout_probabilities(cuda, p):
  from faster_weathernext import branch
  x = torch.ones(100_000, device="cuda")
  y = branch.dropout(x, p, 99)
  want = _mask((100_000,), p, 99, 0)
  assert torch.equal(y.double() == 0, want == 0)
  _close(y, want, 2 * U * want)


def test_dropout_values_off_bounds(cuda):
  """Dropped values are 0 whatever they were; kept infinities and NaN stay."""
  from faster_weathernext import branch
  x = torch.tensor([float("inf"), float("nan"), -float("inf")], device="cuda").repeat(1000)
  y = branch.dropout(x, 0.5, 3)
  m = _mask((3000,), 0.5, 3, 0) != 0
  assert (y[~m] == 0).all() and torch.equal(torch.isnan(y), torch.isnan(x) & m) and torch.equal(torch.isinf(y), torch.isinf(x) & m)
  assert (branch.dropout(x, 1.0, 3) == 0).all()


def test_dropout_seed_forms(cuda):
  """An int, a tensor of the same bits, and layouts: the mask goes by the value's place alone."""
  from faster_weathernext import branch
  rand = _randn(0)
  x = rand(64, 96)
  t = torch.tensor([-5], dtype=torch.int64, device="cuda")
  a, b = branch.dropout(x, 0.4, 2 ** 64 - 5), branch.dropout(x, 0.4, t)
  assert torch.equal(a, b)
  assert torch.equal(branch.dropout(x.t().contiguous().t(), 0.4, t), a)
  wide = rand(64, 200)
  wide[:, 3:99] = x
  assert torch.equal(branch.dropout(wide[:, 3:99], 0.4, t), a)
  assert torch.equal(branch.dropout(x.reshape(-1)[1:], 0.4, t)[8:] == 0, _mask((64 * 96 - 1,), 0.4, 2 ** 64 - 5, 0)[8:] == 0)
  assert not torch.equal(branch.dropout(x, 0.4, t, site=1) == 0, a == 0)
  assert branch.dropout(x[:0], 0.4, t).shape == (0, 96)
  assert branch.dropout(torch.tensor(2.0, device="cuda"), 0.0, t).shape == ()


def test_dropout_second_derivative_and_changed_seed(cuda):
  from faster_weathernext import branch
  x = _randn(1)(500).requires_grad_()
  y = branch.dropout(x * x, 0.25, 8)
  g, = torch.autograd.grad(y.sum(), x, create_graph=True)
  h, = torch.autograd.grad(g.sum(), x)
  _close(h, 2 * _mask((500,), 0.25, 8, 0), 1e-6)
  seed = torch.tensor([8], device="cuda")
  y = branch.dropout(x, 0.25, seed)
  seed.add_(1)
  with pytest.raises(RuntimeError, match="modified by an inplace"):
    y.sum().backward()


def test_dropout_in_a_graph_takes_new_masks(cuda):
  from faster_weathernext import branch
  x = torch.ones(10_000, device="cuda")
  seed = torch.tensor([1], device="cuda")
  branch.dropout(x, 0.5, seed)
  torch.cuda.synchronize()
  g = torch.cuda.CUDAGraph()
  with torch.cuda.graph(g):
    y = branch.dropout(x, 0.5, seed)
  for s in (1, 2, 77):
    seed.fill_(s)
    g.replay()
    assert torch.equal(y == 0, _mask((10_000,), 0.5, s, 0) == 0)


# ---- the norms around a branch --------------------------------------------------------------------------------------

def _inputs(shape, xd, yd, gate, wd, seed=0):
  rand = _randn(seed + shape[-1])
  d = shape[-1]
  x, y = (rand(*shape) * torch.exp(0.5 * rand(d))).to(xd), (0.5 * rand(*shape)).to(yd)
  pw, w = ((1 + 0.2 * rand(d)).to(wd), (1 + 0.2 * rand(d)).to(wd)) if wd is not None else (None, None)
  gs = {None: None, "channel": (d,), "sample": shape[:-2] + (d,), "kept": shape[:-2] + (1, d), "value": shape}[gate]
  g = None if gs is None else (0.5 + 0.3 * rand(*gs)).to(yd if gate == "value" else F32)
  return x, y, pw, w, g


def _formula(x, y, pw, w, gate, alpha, eps, mask):
  leaf = lambda t: None if t is None else t.detach().double().requires_grad_()  # noqa: E731
  v = [leaf(t) for t in (x, y, pw, w, gate)]
  d = x.shape[-1]
  b = v[1] / torch.sqrt((v[1] ** 2).sum(-1, keepdim=True) / d + eps)
  if v[2] is not None:
    b = b * v[2]
  if v[4] is not None:
    g = v[4]
    if g.shape != x.shape and g.dim() == x.dim() - 1 and g.dim() > 1:
      g = g.unsqueeze(-2)
    b = b * g
  if mask is not None:
    b = torch.where(mask != 0, b * mask, torch.zeros_like(b))
  s = alpha * v[0] + b
  h = s / torch.sqrt((s ** 2).sum(-1, keepdim=True) / d + eps)
  if v[3] is not None:
    h = h * v[3]
  return v, h, s


def _rows_room(t, d):
  return (d / 64 + 40) * U * t.abs().amax(-1, keepdim=True)


CASES = [
    ((1, 1), F32, BF16, "channel", F32, BF16, 1.0, 0.0),
    ((1, 8), BF16, BF16, None, None, F32, 0.5, 0.0),
    ((5, 64), F32, F32, "value", BF16, F32, 1.0, 0.2),
    ((2, 33, 100), F32, BF16, "sample", F32, BF16, 1.0, 0.1),
    ((3, 7, 65), BF16, F32, "sample", F32, F32, 1.25, 0.3),
    ((3, 40, 257), BF16, BF16, "value", F32, BF16, 1.0, 0.25),
    ((4, 50, 512), F32, BF16, "kept", F32, BF16, 1.0, 0.1),
    ((2, 2, 30, 512), BF16, BF16, "sample", BF16, BF16, 0.7, 0.0),
    ((700, 512), F32, F32, "channel", F32, F32, 1.0, 0.0),
    ((6, 5, 520), F32, BF16, "sample", BF16, BF16, -1.0, 0.5),
    ((150, 1001), BF16, BF16, "channel", F32, BF16, 1.25, 0.1),
    ((2, 3, 1001), F32, BF16, "sample", F32, BF16, 1.0, 0.1),   # fewer rows a gate than the start of a row repeats
    ((2, 90, 1001), F32, BF16, "sample", F32, F32, 1.0, 0.0),
    ((9, 2048), BF16, F32, "value", None, F32, 1.0, 0.0),
    ((5, 4099), F32, BF16, "value", BF16, BF16, 1.0, 0.4),
    ((4, 8192), BF16, BF16, "channel", F32, BF16, 1.0, 0.1),
    ((11, 8185), F32, F32, None, F32, F32, 0.0, 0.1),
    ((333, 192), F32, BF16, "channel", F32, BF16, 1.0, 0.1),
    ((700, 250), BF16, BF16, "channel", F32, BF16, 1.0, 0.1),
    ((300, 252), F32, F32, "value", F32, F32, 1.0, 0.0),
    ((1000, 1), F32, BF16, "channel", F32, F32, 1.0, 0.3),
    ((500, 3), BF16, BF16, "channel", F32, BF16, 1.0, 0.0),
    ((211, 9), F32, BF16, "value", F32, BF16, 1.0, 0.1),
    ((90, 333), BF16, F32, "channel", F32, BF16, 1.0, 0.0),
    ((2, 70, 760), F32, BF16, "sample", BF16, F32, 1.0, 0.1),
    ((33, 771), F32, BF16, "value", F32, BF16, 1.0, 0.1),
    ((40, 1152), BF16, BF16, "channel", F32, BF16, 1.0, 0.2),
    ((3, 9, 1700), F32, F32, "sample", F32, BF16, 1.0, 0.0),
    ((21, 5000), F32, BF16, "channel", F32, BF16, 1.0, 0.1),
    ((1000, 1, 64), F32, BF16, "sample", F32, BF16, 1.0, 0.1),
    ((301, 2, 24), F32, BF16, "sample", F32, BF16, 1.0, 0.1),
    ((40, 3, 13), F32, BF16, "sample", F32, BF16, 1.0, 0.1),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[0])) + f"-{c[3]}-{c[7]}")
def test_branch_norm_and_gradients(cuda, case):
  from faster_weathernext import branch
  shape, xd, yd, gate, wd, od, alpha, p = case
  ins = _inputs(shape, xd, yd, gate, wd)
  rand = _randn(99)
  dh, ds = rand(*shape).to(od), (0.5 * rand(*shape)).to(xd)
  for t in ins:
    if t is not None:
      t.requires_grad_()
  x, y, pw, w, g = ins
  h, s = branch.branch_norm(x, y, pw, w, gate=g, residual_scale=alpha, p=p, seed=42 if p else None, site=2, out_dtype=od)
  wanted = [t for t in ins if t is not None]
  got = torch.autograd.grad((h, s), wanted, (dh, ds))
  assert h.dtype is od and s.dtype is xd and all(a.dtype is b.dtype and a.shape == b.shape for a, b in zip(got, wanted))
  mask = _mask(shape, p, 42, 2) if p else None
  v, h64, s64 = _formula(x, y, pw, w, g, alpha, 1e-6, mask)
  d = shape[-1]
  terms = _terms(x, s64, alpha)
  amp = 1 + 2 * terms / torch.sqrt((s64.detach() ** 2).sum(-1, keepdim=True) / d + 1e-6)
  _close(s.detach(), s64.detach(), (d / 64 + 40) * U * terms, "s")
  _close(h.detach(), h64.detach(), amp * _rows_room(h64.detach(), d), "h")
  leaves = [t for t in v if t is not None]
  want = torch.autograd.grad((h64, s64), leaves, (dh.double(), ds.double()))
  names = [n for n, t in zip(("x", "y", "post_weight", "weight", "gate"), ins) if t is not None]
  rows = x.numel() // d
  with torch.no_grad():
    for name, a, b in zip(names, got, want):
      if name in ("x", "y") or (name == "gate" and a.shape == x.shape):
        # Gradients of a row: differences of terms of the size of the row's largest gradient times the factors' largest.
        room = (d / 64 + 60) * U * 8 * torch.maximum(b.abs().amax(-1, keepdim=True), _size_of_terms(y, s64, dh, ds, name, leaves, names)) * amp
        _close(a, b, room, "d_" + name)
      else:
        columns = _column_terms(name, x, y, dh, ds, v, alpha, mask, amp)
        _close(a, b, (rows / 64 + 200 + d / 8) * U * columns.view(b.shape), "d_" + name)


def _terms(x, s64, alpha):
  """The row's largest |residual_scale x| + |branch|."""
  ax = alpha * x.detach().double()
  return (ax.abs() + (s64.detach() - ax).abs()).amax(-1, keepdim=True)


def _size_of_terms(y, s64, dh, ds, name, leaves, names):
  """A bound of the terms that a row's gradient is made of, from the row's values (float64 [..., 1])."""
  d = y.shape[-1]
  r1 = 1 / torch.sqrt((y.detach().double() ** 2).sum(-1, keepdim=True) / d + 1e-6)
  r2 = 1 / torch.sqrt((s64.detach() ** 2).sum(-1, keepdim=True) / d + 1e-6)
  v = dict(zip(names, leaves))
  g = dh.abs().double().amax(-1, keepdim=True) * (v["weight"].abs().max() if "weight" in v else 1.0)
  dt = 2 * g * d ** 0.5 * r2 + ds.abs().double().amax(-1, keepdim=True)
  if name == "x":
    return dt
  f = (v["post_weight"].abs().max() if "post_weight" in v else 1.0) * (v["gate"].abs().max() if "gate" in v else 1.0)
  return dt * f * 4 * (r1 if name == "y" else d ** 0.5)


def _column_terms(name, x, y, dh, ds, v, alpha, mask, amp):
  """Sum over rows of the absolute terms of a column's sum, each with its row's `amp`."""
  d = x.shape[-1]
  xs, ys = x.double(), y.double()
  yhat = ys / torch.sqrt((ys ** 2).sum(-1, keepdim=True) / d + 1e-6)
  pw = v[2] if v[2] is not None else torch.ones(d, device="cuda", dtype=torch.float64)
  w = v[3] if v[3] is not None else torch.ones(d, device="cuda", dtype=torch.float64)
  g = v[4] if v[4] is not None else torch.ones(d, device="cuda", dtype=torch.float64)
  if g.shape != x.shape and g.dim() == x.dim() - 1 and g.dim() > 1:
    g = g.unsqueeze(-2)
  b = yhat * pw * g * (mask if mask is not None else 1.0)
  s = alpha * xs + b
  r2 = 1 / torch.sqrt((s ** 2).sum(-1, keepdim=True) / d + 1e-6)
  shat = s * r2
  gs = dh.double() * w
  dt = r2 * (gs.abs() + shat.abs() * (gs * shat).abs().mean(-1, keepdim=True)) + ds.double().abs()
  db = dt * amp * (mask if mask is not None else 1.0)
  if name == "weight":
    return (dh.double().abs() * shat.abs() * amp).reshape(-1, d).sum(0)
  if name == "post_weight":
    return (db * (yhat * g).abs()).reshape(-1, d).sum(0)
  t = db * (yhat * pw).abs()
  if v[4].dim() == 1:
    return t.reshape(-1, d).sum(0)
  return t.sum(-2).reshape(v[4].shape)


@pytest.mark.parametrize("d", [64, 515, 2048])
@pytest.mark.parametrize("xd", [F32, BF16])
def test_branch_norm_fp8(cuda, d, xd):
  from faster_weathernext import branch
  x, y, pw, w, g = _inputs((3, 21, d), xd, BF16, "sample", F32)
  values, scale, s = branch.branch_norm_fp8(x, y, pw, w, gate=g, residual_scale=0.5)
  _, h64, s64 = _formula(x, y, pw, w, g, 0.5, 1e-6, None)
  assert values.dtype is E4M3 and scale.shape == (3, 21)
  _close(s, s64.detach(), _rows_room(s64.detach(), d))
  _close(scale, h64.detach().abs().amax(-1) / 448, (d / 64 + 44) * U * scale.double())
  # A value is rounded to e4m3 (2^-4 of itself, 2^-10 where that is subnormal) after float32's own errors.
  want = h64.detach() / scale.double().unsqueeze(-1)
  off = (values.float().double() - want).abs()
  assert (off <= torch.maximum(want.abs() * 2.0 ** -4, torch.full_like(want, 2.0 ** -10)) + 448 * (d / 64 + 44) * U).all()


def test_branch_norm_fp8_rows_off_bounds(cuda):
  """A row of zeros: scale and values 0; a NaN stays in its row."""
  from faster_weathernext import branch
  x, y = torch.zeros(4, 64, device="cuda"), torch.zeros(4, 64, device="cuda", dtype=BF16)
  x[1] = 1.0
  x[2, 5] = float("nan")
  values, scale, _ = branch.branch_norm_fp8(x, y)
  assert scale[0] == 0 and (values[0].float() == 0).all() and scale[1] > 0 and torch.isnan(scale[2]) and scale[3] == 0


def test_nan_and_infinity_stay_in_their_rows(cuda):
  from faster_weathernext import branch
  x, y, pw, w, _ = _inputs((9, 512), F32, BF16, None, F32)
  clean_h, clean_s = branch.branch_norm(x, y, pw, w)
  x2, y2 = x.clone(), y.clone()
  x2[3, 7], y2[6, 100] = float("nan"), float("inf")
  leaves = [t.requires_grad_() for t in (x2, y2)]
  h, s = branch.branch_norm(x2, y2, pw, w)
  grads = torch.autograd.grad((h, s), leaves, (torch.ones_like(h), torch.ones_like(s)))
  keep = [r for r in range(9) if r not in (3, 6)]
  assert torch.equal(h[keep], clean_h[keep]) and torch.equal(s[keep], clean_s[keep])
  assert torch.isnan(h[3]).all() and torch.isnan(h[6]).any()
  assert all(torch.isfinite(t[keep]).all() for t in grads)


def test_a_dropped_value_counts_as_zero(cuda):
  """Where dropout takes a value that is not a number, the rest of the row goes on."""
  from faster_weathernext import branch
  x = torch.ones(1, 64, device="cuda")
  y = torch.ones(1, 64, device="cuda")
  gate = torch.ones(64, device="cuda")
  m = _mask((1, 64), 0.5, 4, 0)[0]
  gate[int((m == 0).nonzero()[0])] = float("inf")
  h, s = branch.branch_norm(x, y, gate=gate, p=0.5, seed=4)
  assert torch.isfinite(h).all() and torch.isfinite(s).all()


def test_strides_offsets_and_layouts(cuda):
  """Views of any stride and start give what their copies give, bit for bit where both take wide accesses."""
  from faster_weathernext import branch
  rand = _randn(5)
  base_x, base_y = rand(40, 2, 512), rand(40, 3, 512).to(BF16)
  x, y = base_x[:, 1], base_y[:, 2]
  want = branch.branch_norm(x.contiguous(), y.contiguous(), p=0.1, seed=1)
  got = branch.branch_norm(x, y, p=0.1, seed=1)
  assert all(torch.equal(a, b) for a, b in zip(got, want))
  flat = rand(40 * 512 + 1)
  off = flat[1:].view(40, 512)
  got = branch.branch_norm(off, y, p=0.1, seed=1)
  want = branch.branch_norm(off.clone(), y, p=0.1, seed=1)
  assert all(torch.equal(a, b) for a, b in zip(got, want))
  odd = rand(40, 700)[:, :333]
  got, want = branch.branch_norm(odd, y[:, :333]), branch.branch_norm(odd.clone(), y[:, :333].clone())
  assert all(torch.equal(a, b) for a, b in zip(got, want))
  turned = rand(512, 40).t()
  leaves = [turned.requires_grad_(), y.detach().requires_grad_()]
  h, s = branch.branch_norm(*leaves)
  dh = rand(512, 40).to(BF16).t()
  got = torch.autograd.grad(h, leaves, dh)
  twin = [t.detach().clone(memory_format=torch.contiguous_format).requires_grad_() for t in leaves]
  want = torch.autograd.grad(branch.branch_norm(*twin)[0], twin, dh.contiguous())
  assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_columns_off_their_alignment(cuda):
  """Weights and gates that start anywhere, of widths that are multiples of 8: the form for rows of any width."""
  from faster_weathernext import _lib, branch
  rand = _randn(21)
  x, y = rand(50, 64), rand(50, 64).to(BF16)
  pool = 1 + 0.1 * rand(200)
  odd = [pool[i:i + 64] for i in (1, 66, 131)]
  want = branch.branch_norm(x, y, odd[0].clone(), odd[1].clone(), gate=odd[2].clone())
  s, h = torch.empty_like(x), torch.empty(50, 64, device="cuda", dtype=BF16)
  desc = _lib.BranchDesc(50, 64, 64, 50, 64, _lib.DTYPE_F32, _lib.DTYPE_BF16, 1, 1, 1, _lib.DTYPE_BF16, 1e-6, 1.0, 0)
  _lib.check(_lib.lib().fwn_branch_norm(desc, x.data_ptr(), y.data_ptr(), *[t.data_ptr() for t in odd], s.data_ptr(), h.data_ptr(),
                                        None, None, torch.cuda.current_stream().cuda_stream))
  _close(h, want[0].double(), 2.0 ** -7 * want[0].double().abs())
  _close(s, want[1].double(), 8 * U * want[1].double().abs().amax())
  assert all(torch.equal(a, b) for a, b in zip(branch.branch_norm(x, y, odd[0], odd[1], gate=odd[2]), want))


def test_empty_and_partial_gradients(cuda):
  from faster_weathernext import branch
  x, y, pw, w, g = _inputs((2, 5, 64), F32, BF16, "sample", F32)
  for t in (x, y, pw, w, g):
    t.requires_grad_()
  h, s = branch.branch_norm(x, y, pw, w, gate=g)
  full = torch.autograd.grad((h, s), (x, y, pw, w, g), (torch.ones_like(h), torch.zeros_like(s)), retain_graph=True)
  only_h = torch.autograd.grad(h, (x, y, pw, w, g), torch.ones_like(h), retain_graph=True)
  assert all(torch.equal(a, b) for a, b in zip(full, only_h))
  only_s = torch.autograd.grad(s, (x, y, pw, w, g), torch.ones_like(s), allow_unused=True, retain_graph=True)
  assert torch.equal(only_s[0], torch.ones_like(x)) and (only_s[3] == 0).all()
  assert torch.equal(torch.autograd.grad(h, w, torch.ones_like(h))[0], full[3])
  e = [torch.zeros(0, 64, device="cuda", requires_grad=True), torch.zeros(0, 64, device="cuda"), torch.ones(64, device="cuda", requires_grad=True)]
  h, s = branch.branch_norm(e[0], e[1], e[2])
  assert h.shape == (0, 64)
  gx, gw = torch.autograd.grad((h, s), (e[0], e[2]), (torch.zeros_like(h), torch.zeros_like(s)))
  assert gx.shape == (0, 64) and (gw == 0).all()


@pytest.mark.parametrize("d", [64, 333, 1001])
@pytest.mark.parametrize("have", ["post_weight", "weight", "gate", "post_weight gate", "weight gate"])
def test_some_of_the_columns(cuda, d, have):
  """Either weight or the gate alone: what is not given counts as ones, and only what is given gets a gradient. The columns'
  sums of 51 terms may be added in another order (gate by gate where there are gates): each order is off by at most 51 2^-24
  of the terms' absolute sum."""
  from faster_weathernext import branch
  x, y, pw, w, g = _inputs((3, 17, d), F32, BF16, "sample", F32)
  kw = {"post_weight": pw, "weight": w, "gate": g}
  given = {k: v.requires_grad_() for k, v in kw.items() if k in have.split()}
  ones = {k: v if k in given else torch.ones_like(v) for k, v in kw.items()}
  x.requires_grad_()
  dh, ds = _randn(1)(3, 17, d).to(BF16), _randn(2)(3, 17, d)
  leaves = [x, *given.values()]
  a, b = branch.branch_norm(x, y, p=0.1, seed=1, **given), branch.branch_norm(x, y, p=0.1, seed=1, **ones)
  assert all(torch.equal(u, v) for u, v in zip(a, b))
  got, want = (torch.autograd.grad(o, leaves, (dh, ds)) for o in (a, b))
  assert torch.equal(got[0], want[0])
  mask = _mask((3, 17, d), 0.1, 1, 0)
  v = [t.detach().double() for t in (x, y, ones["post_weight"], ones["weight"], ones["gate"])]
  for name, u, o in zip(given, got[1:], want[1:]):
    terms = _column_terms(name, x.detach(), y, dh, ds, v, 1.0, mask, 1.0)
    assert ((u.double() - o.double()).abs() <= 2 * 51 * U * terms.view(u.shape)).all(), name


@pytest.mark.parametrize("d", [65, 250, 1001, 2047])
def test_one_gradient_of_odd_rows(cuda, d):
  """Rows that start anywhere, with the gradient of one output alone: the other one's is not there to read."""
  from faster_weathernext import branch
  for xd, yd in ((F32, BF16), (BF16, F32)):
    ins = _inputs((2, 21, d), xd, yd, "sample", F32)
    for t in ins:
      t.requires_grad_()
    h, s = branch.branch_norm(*ins[:4], gate=ins[4], p=0.2, seed=3)
    dh, ds = _randn(1)(2, 21, d).to(BF16), _randn(2)(2, 21, d).to(xd)
    only_h = torch.autograd.grad(h, ins, dh, retain_graph=True)
    both = torch.autograd.grad((h, s), ins, (dh, torch.zeros_like(ds)), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(only_h, both))
    only_s = torch.autograd.grad(s, ins, ds, allow_unused=True, retain_graph=True)
    both = torch.autograd.grad((h, s), ins, (torch.zeros_like(dh), ds))
    assert all(torch.equal(a, b) for a, b in zip(only_s, both))


@pytest.mark.parametrize("d", [64, 65, 100, 250, 1001])
@pytest.mark.parametrize("gate", ["sample", "value"])
def test_nan_stays_with_its_gate(cuda, d, gate):
  """A sample's NaN reaches no other sample's rows nor its gate's gradient."""
  from faster_weathernext import branch
  ins = _inputs((4, 9, d), F32, BF16, gate, F32)
  dh, ds = _randn(1)(4, 9, d).to(BF16), _randn(2)(4, 9, d)
  for t in ins:
    t.requires_grad_()
  want = torch.autograd.grad(branch.branch_norm(*ins[:4], gate=ins[4]), (ins[0], ins[1], ins[4]), (dh, ds))
  with torch.no_grad():
    for t in ins[:2]:
      t[2] = float("nan")
    dh[2], ds[2] = float("nan"), float("nan")
  got = torch.autograd.grad(branch.branch_norm(*ins[:4], gate=ins[4]), (ins[0], ins[1], ins[4]), (dh, ds))
  assert all(torch.equal(a[[0, 1, 3]], b[[0, 1, 3]]) for a, b in zip(got, want))


@pytest.mark.parametrize("shape,gate", [((0, 64), (64,)), ((3, 0, 64), (3, 64)), ((0, 5, 64), (0, 64)), ((0, 64), (0, 64))])
def test_gates_of_no_rows(cuda, shape, gate):
  from faster_weathernext import branch
  x, g = torch.zeros(shape, device="cuda", requires_grad=True), torch.ones(gate, device="cuda", requires_grad=True)
  torch.full((1 << 20,), 7.0, device="cuda")  # memory that is not zero
  h, _ = branch.branch_norm(x, torch.zeros(shape, device="cuda"), gate=g)
  d_gate, = torch.autograd.grad(h, g, torch.zeros_like(h))
  assert d_gate.shape == gate and (d_gate == 0).all()


def test_gradient_against_differences(cuda):
  """The kernels' own forward, moved along a random direction, in float32."""
  from faster_weathernext import branch
  x, y, pw, w, g = _inputs((2, 9, 96), F32, F32, "sample", F32)
  ins = [t.requires_grad_() for t in (x, y, pw, w, g)]
  rand = _randn(12)
  a, b = rand(2, 9, 96), rand(2, 9, 96)

  def value(v):
    h, s = branch.branch_norm(*v[:4], gate=v[4], residual_scale=0.8, p=0.2, seed=6, out_dtype=F32)
    return (h.double() * a).sum() + (s.double() * b).sum()

  grads = torch.autograd.grad(value(ins), ins)
  step = 1e-2
  for i, gr in enumerate(grads):
    direction = rand(*gr.shape)
    moved = lambda f: [t.detach() + f * step * direction if i == j else t.detach() for j, t in enumerate(ins)]  # noqa: E731, B023
    # Fourth-order differences: an error of step^4 times the fifth derivative, and float32's noise over the step.
    slope = (8 * (value(moved(1)) - value(moved(-1))) - (value(moved(2)) - value(moved(-2)))) / (12 * step)
    want = (gr.double() * direction).sum()
    size = (gr.double().norm() * direction.double().norm())
    assert abs(slope - want) <= 1e-3 * size, (i, slope.item(), want.item())


def test_deterministic_and_repeated(cuda):
  from faster_weathernext import branch
  x, y, pw, w, g = _inputs((4, 3001, 512), F32, BF16, "sample", F32)
  ins = [t.requires_grad_() for t in (x, y, pw, w, g)]
  runs = []
  for _ in range(3):
    h, s = branch.branch_norm(*ins[:4], gate=g, p=0.1, seed=3)
    runs.append([h.detach(), s.detach(), *torch.autograd.grad((h, s), ins, (torch.ones_like(h), torch.ones_like(s)))])
  assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))


def test_streams_and_graphs(cuda):
  """Another stream than the inputs'; a training step captured and replayed with new inputs and seeds, beside an eager one."""
  from faster_weathernext import branch
  x, y, pw, w, g = _inputs((2, 100, 512), F32, BF16, "sample", F32)
  ins = [t.requires_grad_() for t in (x, y, pw, w, g)]
  seed = torch.tensor([5], device="cuda")

  def step():
    h, s = branch.branch_norm(*ins[:4], gate=g, p=0.1, seed=seed)
    return [h.detach(), s.detach(), *torch.autograd.grad((h, s), ins, (torch.ones_like(h), torch.ones_like(s)))]

  want = step()
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    got = step()
  torch.cuda.current_stream().wait_stream(side)
  assert all(torch.equal(a, b) for a, b in zip(got, want))
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = step()
  with torch.no_grad():
    x.add_(1.0)
  seed.fill_(9)
  graph.replay()
  want = step()
  assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals(cuda):
  from faster_weathernext import branch
  x, y = torch.zeros(2, 3, 8, device="cuda"), torch.zeros(2, 3, 8, device="cuda")
  seed = torch.tensor([1], device="cuda")
  for bad in (-0.1, 1.1, float("nan")):
    with pytest.raises(ValueError):
      branch.dropout(x, bad, 1)
    with pytest.raises(ValueError):
      branch.branch_norm(x, y, p=bad, seed=1)
  with pytest.raises(TypeError):
    branch.branch_norm(x, y, p=0.1)
  with pytest.raises(TypeError):
    branch.dropout(x, 0.1, 1.0)
  with pytest.raises(TypeError):
    branch.dropout(x, 0.1, seed.int())
  with pytest.raises(ValueError):
    branch.dropout(x, 0.1, seed.cpu())
  with pytest.raises(ValueError):
    branch.dropout(x, 0.1, seed.repeat(2))
  for s in (-1, 2 ** 64):
    with pytest.raises(ValueError):
      branch.dropout(x, 0.1, s)
  with pytest.raises(ValueError):
    branch.dropout(x, 0.1, 1, site=2 ** 32)
  with pytest.raises(TypeError):
    branch.dropout(x.half(), 0.1, 1)
  with pytest.raises(ValueError):
    branch.branch_norm(x, y[:1])
  with pytest.raises(ValueError):
    branch.branch_norm(x, y, torch.ones(7, device="cuda"))
  for shape in ((3, 8), (2, 3), (3, 1, 8), (1, 3, 8), (8, 2)):
    with pytest.raises(ValueError):
      branch.branch_norm(x, y, gate=torch.ones(shape, device="cuda"))
  with pytest.raises(ValueError):
    branch.branch_norm(x, y, out_dtype=torch.float16)
  with pytest.raises(TypeError):
    branch.branch_norm(x, y, residual_scale=torch.ones(8, device="cuda"))
  with pytest.raises(TypeError):
    branch.branch_norm(x, y, gate=torch.ones(8, device="cuda", dtype=torch.float16))
  with pytest.raises(NotImplementedError):
    branch.branch_norm(torch.zeros(2, 8200, device="cuda"), torch.zeros(2, 8200, device="cuda"))
  with pytest.raises(NotImplementedError):
    branch.branch_norm(torch.zeros(2, 8191, device="cuda"), torch.zeros(2, 8191, device="cuda"))
  with pytest.raises(NotImplementedError):
    branch.branch_norm_fp8(x.clone().requires_grad_(), y)
  a = x.clone().requires_grad_()
  with pytest.raises(NotImplementedError):
    torch.autograd.grad(branch.branch_norm(a, y)[0].float().sum(), a, create_graph=True)
  from torch.autograd import forward_ad
  with forward_ad.dual_level():
    dual = forward_ad.make_dual(x, torch.ones_like(x))
    for call in (lambda: branch.dropout(dual, 0.1, 1), lambda: branch.branch_norm(dual, y)):
      with pytest.raises(NotImplementedError):
        call()


def test_gradients_of_saved_tensors_that_come_back_elsewhere(cuda):
  """Saved tensors may be moved between forward and backward (torch.autograd.graph's hooks): rows with a stride come back
  without one, the seed at another address. The same bits as without."""
  from faster_weathernext import branch
  r = _randn(61)
  wide, y, pw, w, gate = r(33, 160), r(33, 72).to(BF16), r(72), r(72).to(BF16), r(33, 72)
  dh, ds = r(33, 72).to(BF16), r(33, 72)
  seed = torch.tensor([77], dtype=torch.int64, device="cuda")

  def grads(seed):
    leaves = [t.clone().requires_grad_() for t in (wide, y, pw, w, gate)]
    h, s = branch.branch_norm(leaves[0][:, 8:80], *leaves[1:4], gate=leaves[4], p=0.25, seed=seed)
    return torch.autograd.grad((h, s), leaves, (dh, ds))

  for used in (seed, 77):
    want = grads(used)
    with torch.autograd.graph.save_on_cpu():
      got = grads(used)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
