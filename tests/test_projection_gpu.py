"""GPU: the pre-norm projections (faster_weathernext.projection) against plain float64 torch on the same inputs.

Bounds, in relative 2-norm. A result rounded once to bf16 is off by at most half a step of each value, 2^-9 to 2^-8 of it,
in the mean square over many values below 2^-9; fewer than 64 values are held to half a step each. A gradient through the
bf16 pre-activation gradient has a second rounding of that size, whose errors are independent over the sum: twice the
bound. float32 norms: about ten roundings of 2^-24. float32 products: every 768 of k accumulate in the tensor core, 16
(bf16) or 32 (e4m3) at a step, each step truncating 2^-24 of the running sum on average, 48 * 2^-24 = 2.9e-6. Column sums
over rows in float32: 2^-24 times the square root of the terms, with a margin of ten. e4m3: half a step is 2^-4 of a
normal value, 2^-10 below 2^-6."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32, E4 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
TOL = {BF: 2.0 ** -9 + 1e-5, F32: 1e-6}
TOL_PRODUCT = {BF: 2.0 ** -9 + 1e-5, F32: 4e-6}
TOL_GRAD = {BF: 2 * 2.0 ** -9, F32: 1e-5}
C0, C1 = math.sqrt(2.0 / math.pi), 0.044715


def _pr():
  from faster_weathernext import projection
  return projection


def _gen(seed):
  return torch.Generator(device="cuda").manual_seed(seed)


def _rel(x, ref):
  x, ref = x.double(), ref.double()
  assert x.shape == ref.shape
  assert bool(torch.isfinite(x).all())
  return float((x - ref).norm() / ref.norm().clamp_min(1e-30))


def _check(x, ref, tol):
  """_rel within tol; a bf16 tensor of fewer than 64 values: each within half a step of bf16 (and tol's share of 2^-9)."""
  if x.dtype == BF and x.numel() < 64:
    step = torch.exp2(torch.floor(torch.log2(ref.abs().clamp_min(1e-30))) - 7)
    assert x.shape == ref.shape
    assert bool(((x.double() - ref).abs() <= 0.5 * step * (tol / 2.0 ** -9) + 1e-6 * ref.abs().max()).all())
  else:
    assert _rel(x, ref) <= tol


def _no_device_error():
  from faster_weathernext import _lib
  torch.cuda.synchronize()
  assert _lib.device_error(torch.cuda.current_stream().cuda_stream) == 0


def _act64(x, act):
  if act == "gelu":
    return 0.5 * x * (1.0 + torch.tanh(C0 * (x + C1 * x ** 3)))
  return x * torch.sigmoid(x) if act == "swish" else x


def _rms64(x, w, r, eps):
  s = x if r is None else x + r
  h = s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
  return (h if w is None else h * w), s


def _check_fp8(values, scale, h):
  """values e4m3 and scale against h (float64): the scale to float32, each value to half an e4m3 step."""
  top = h.abs().amax(-1)
  assert float(((scale.double() - top / 448.0).abs() / (top / 448.0).clamp_min(1e-300)).max()) <= 1e-6
  want = h / (top / 448.0)[..., None]
  err = (values.double() - want).abs()
  assert bool((err <= want.abs() * 2.0 ** -4 * 1.001 + 2.0 ** -10 * 1.001).all())
  assert float(values.double().abs().max()) == 448.0


# ---- rms_norm -------------------------------------------------------------------------------------------------------

WIDTHS = [(1, 1), (3, 7), (12, 64), (5, 256), (9, 257), (42, 512), (33, 1000), (17, 1024), (2, 1025), (5, 2048),
          (3, 4104), (2, 8192), (3, 8200), (2, 16384), (1, 16383)]


@pytest.mark.parametrize("rows,d", WIDTHS)
@pytest.mark.parametrize("x_dtype,r_dtype,w_dtype", [(F32, BF, F32), (BF, BF, BF), (BF, F32, F32), (F32, None, None),
                                                     (F32, F32, BF), (BF, None, F32)])
def test_rms_norm_forward(cuda, rows, d, x_dtype, r_dtype, w_dtype):
  pr, g = _pr(), _gen(rows * 7 + d)
  x = (torch.randn(rows, d, device=cuda, generator=g) * 3).to(x_dtype)
  r = None if r_dtype is None else torch.randn(rows, d, device=cuda, generator=g).to(r_dtype)
  w = None if w_dtype is None else (1 + 0.2 * torch.randn(d, device=cuda, generator=g)).to(w_dtype)
  dbl = lambda t: None if t is None else t.double()  # noqa: E731
  h64, s64 = _rms64(x.double(), dbl(w), dbl(r), 1e-6)
  for out in (BF, F32):
    got = pr.rms_norm(x, w, r, out_dtype=out)
    h = got if r is None else got[0]
    assert h.dtype == out
    _check(h, h64, TOL[out])
    if r is not None:
      assert got[1].dtype == x_dtype
      _check(got[1], s64, TOL[x_dtype])
  got = pr.rms_norm_fp8(x, w, r)
  assert got[0].dtype == E4 and got[1].shape == (rows,)
  _check_fp8(got[0], got[1], h64)
  if r is not None:
    _check(got[2], s64, TOL[x_dtype])


@pytest.mark.parametrize("rows,d", [(1, 1), (3, 7), (42, 512), (1001, 515), (333, 1024), (300, 1030), (40, 4096),
                                    (7, 9001), (3, 16384)])
@pytest.mark.parametrize("x_dtype,r_dtype,w_dtype,out", [(F32, BF, F32, BF), (BF, BF, BF, BF), (BF, F32, F32, F32),
                                                         (F32, None, F32, BF), (F32, F32, None, F32)])
def test_rms_norm_gradients(cuda, rows, d, x_dtype, r_dtype, w_dtype, out):
  pr, g = _pr(), _gen(rows + d)
  x = (torch.randn(rows, d, device=cuda, generator=g) * 2).to(x_dtype).requires_grad_()
  r = None if r_dtype is None else torch.randn(rows, d, device=cuda, generator=g).to(r_dtype).requires_grad_()
  w = None if w_dtype is None else (1 + 0.2 * torch.randn(d, device=cuda, generator=g)).to(w_dtype).requires_grad_()
  dh = torch.randn(rows, d, device=cuda, generator=g).to(out)
  ds = torch.randn(rows, d, device=cuda, generator=g).to(x_dtype)
  ins = [t for t in (x, w, r) if t is not None]
  got = pr.rms_norm(x, w, r, out_dtype=out, eps=1e-5)
  outs, seeds = ((got,), (dh,)) if r is None else (got, (dh, ds))
  grads = torch.autograd.grad(outs, ins, seeds)
  again = torch.autograd.grad(pr.rms_norm(x, w, r, out_dtype=out, eps=1e-5), ins, seeds)
  ref = [t.detach().double().requires_grad_() for t in ins]
  it = iter(ref)
  x64, w64, r64 = next(it), (next(it) if w is not None else None), (next(it) if r is not None else None)
  h64, s64 = _rms64(x64, w64, r64, 1e-5)
  want = torch.autograd.grad((h64,) if r is None else (h64, s64), ref, [s.double() for s in seeds])
  for t, a, b, c in zip(ins, grads, again, want):
    assert a.dtype == t.dtype and a.shape == t.shape
    assert torch.equal(a, b)                                   # fixed order: the same bits
    if t.dtype == BF and d > 1:
      _check(a, c, TOL[BF])
    else:
      # d = 1: dx is what is left of a full cancellation; measured against what cancels.
      scale = max(float(c.norm()), float(dh.double().norm()) if d == 1 else 0.0)
      assert float((a.double() - c).norm()) / scale <= (TOL[BF] if t.dtype == BF else TOL_GRAD[F32])


def test_rms_norm_gradient_against_differences(cuda):
  """Directional differences of the kernel's own float32 output: step 1e-2, error O(step^2) of the third derivative."""
  pr, g = _pr(), _gen(5)
  rows, d, t = 16, 640, 1e-2
  x, r, c = (torch.randn(rows, d, device=cuda, generator=g) for _ in range(3))
  w = 1 + 0.1 * torch.randn(d, device=cuda, generator=g)
  dirs = [torch.randn(rows, d, device=cuda, generator=g), torch.randn(d, device=cuda, generator=g)]
  loss = lambda xx, ww: float((pr.rms_norm(xx, ww, r, out_dtype=F32)[0].double() * c.double()).sum())  # noqa: E731
  xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
  h, _ = pr.rms_norm(xg, wg, r, out_dtype=F32)
  gx, gw = torch.autograd.grad(h, (xg, wg), c)
  for grad, dx, dw in ((gx, dirs[0], 0 * dirs[1]), (gw, 0 * dirs[0], dirs[1])):
    diff = (loss(x + t * dx, w + t * dw) - loss(x - t * dx, w - t * dw)) / (2 * t)
    exact = float((grad.double() * (dx if dx.abs().sum() > 0 else dw).double()).sum())
    assert abs(diff - exact) <= 2e-3 * float(c.norm())


def test_rms_norm_only_the_stored_sum_or_the_norm_is_used(cuda):
  pr, g = _pr(), _gen(1)
  x = torch.randn(9, 128, device=cuda, generator=g).requires_grad_()
  r = torch.randn(9, 128, device=cuda, generator=g).to(BF).requires_grad_()
  w = torch.ones(128, device=cuda).requires_grad_()
  _, s = pr.rms_norm(x, w, r)
  gx, gw, gr = torch.autograd.grad(s.sum(), (x, w, r))
  assert bool((gx == 1).all()) and bool((gw == 0).all()) and bool((gr == 1).all()) and gr.dtype == BF
  h, _ = pr.rms_norm(x, w, r, out_dtype=F32)
  gx, gr = torch.autograd.grad(h.square().sum(), (x, r))
  assert bool(torch.isfinite(gx).all()) and torch.equal(gx.to(BF), gr)


@pytest.mark.parametrize("d", [7, 512, 1001, 2048, 9000])
def test_rms_norm_special_rows(cuda, d):
  """Zero rows give 0 (and an 8-bit scale of 0); a NaN or infinity stays in its row; an 8-bit row with one has a NaN
  scale or values, never a number that hides it."""
  pr = _pr()
  x = torch.randn(6, d, device=cuda, generator=_gen(d))
  x[1] = 0
  x[2, d // 2] = float("nan")
  x[3, 0] = float("inf")
  x[4] = 1e-38
  good = [0, 5]
  h = pr.rms_norm(x, out_dtype=F32)
  assert bool((h[1] == 0).all()) and bool(torch.isnan(h[2]).all()) and bool(torch.isnan(h[3]).any())
  assert _rel(h[good], _rms64(x[good].double(), None, None, 1e-6)[0]) <= 1e-6
  v, s = pr.rms_norm_fp8(x)
  assert float(s[1]) == 0 and bool((v[1].float() == 0).all())
  assert bool(torch.isnan(v[2].float() * s[2]).all()) and bool(torch.isnan(v[3].float() * s[3]).any())
  _check_fp8(v[good], s[good], _rms64(x[good].double(), None, None, 1e-6)[0])
  v, s = pr.quantize_fp8(x)
  assert float(s[4]) == 0 and bool((v[4].float() == 0).all())      # below 2^-100
  assert math.isnan(float(s[2])) and bool(torch.isnan(v[3].float() * s[3]).any())
  _check_fp8(v[good], s[good], x[good].double())


def test_rms_norm_strides_views_and_broadcast(cuda):
  pr, g = _pr(), _gen(3)
  big = torch.randn(40, 700, device=cuda, generator=g)
  w = torch.randn(600, device=cuda, generator=g)
  for x in (big[:, :600], big[::2, 8:608], big[:, 1:601], big[:, :600].t().contiguous().t(), big[:1, :600].expand(40, 600),
            big.view(4, 10, 700)[:, 2:9, 4:604]):
    h64, _ = _rms64(x.double(), w.double(), None, 1e-6)
    assert _rel(pr.rms_norm(x, w, out_dtype=F32), h64) <= 1e-6
    r = (0.5 * x).to(BF)
    h, s = pr.rms_norm(x, w, r, out_dtype=F32)
    assert _rel(s, x.double() + r.double()) <= 1e-6 and s.shape == x.shape
  # A broadcast input's gradient is the sum over its copies.
  row = big[:1, :600].clone().requires_grad_()
  pr.rms_norm(row.expand(40, 600), w, out_dtype=F32).square().sum().backward()
  ref = big[:1, :600].double().requires_grad_()
  _rms64(ref.expand(40, 600), w.double(), None, 1e-6)[0].square().sum().backward()
  assert float((row.grad.double() - ref.grad).norm()) <= 1e-4 * float(w.double().square().sum())


def test_rms_norm_empty_and_refusals(cuda):
  pr = _pr()
  x = torch.randn(4, 64, device=cuda)
  e = torch.empty(0, 64, device=cuda, requires_grad=True)
  w = torch.ones(64, device=cuda, requires_grad=True)
  h = pr.rms_norm(e, w)
  assert h.shape == (0, 64)
  gw, = torch.autograd.grad(h.sum(), w)
  assert bool((gw == 0).all())
  assert pr.rms_norm_fp8(e.detach())[1].shape == (0,)
  for bad in (lambda: pr.rms_norm(x, torch.ones(63, device=cuda)), lambda: pr.rms_norm(x, None, x[:3]),
              lambda: pr.rms_norm(x, eps=-1.0), lambda: pr.rms_norm(x, out_dtype=torch.float16),
              lambda: pr.rms_norm(x.cpu()), lambda: pr.rms_norm(x, torch.ones(64)),
              lambda: pr.rms_norm(torch.empty(4, 0, device=cuda))):
    with pytest.raises(ValueError):
      bad()
  for bad in (lambda: pr.rms_norm(x.half()), lambda: pr.rms_norm(x, w.detach().double()),
              lambda: pr.rms_norm(x, None, x.half())):
    with pytest.raises(TypeError):
      bad()
  with pytest.raises(NotImplementedError):
    pr.rms_norm(torch.empty(1, 16385, device=cuda))


def test_rms_norm_offsets_past_32_bits(cuda):
  """140,000 rows of 16,384 bf16 (2.3e9 values): the last rows against float64."""
  pr = _pr()
  rows, d = 140_000, 16_384
  x = torch.empty(rows, d, device=cuda, dtype=BF)
  x[:] = torch.randn(d, device=cuda, generator=_gen(2)).to(BF)
  x[-3:] = torch.randn(3, d, device=cuda, generator=_gen(3)).to(BF)
  v, s = pr.rms_norm_fp8(x)
  h64, _ = _rms64(x[-3:].double(), None, None, 1e-6)
  _check_fp8(v[-3:], s[-3:], h64)
  assert torch.equal(v[0], v[-4]) and float(s[0]) == float(s[-4])


# ---- linear ---------------------------------------------------------------------------------------------------------

def _problem(m, k, n, seed, layout="nk"):
  g = _gen(seed)
  a = torch.randn(m, k, device="cuda", generator=g).to(BF)
  w = (torch.randn(n, k, device="cuda", generator=g) * k ** -0.5).to(BF)
  if layout == "kn":
    w = w.t().contiguous().t()
  b = 0.3 * torch.randn(n, device="cuda", generator=g)
  r = torch.randn(m, n, device="cuda", generator=g)
  return a, w, b, r


def _linear64(a, w, b, r, act):
  y = a.double() @ w.double().t()
  y = _act64(y if b is None else y + b.double(), act)
  return y if r is None else y + r.double()


SHAPES = [(1, 1, 1), (1, 512, 2048), (2, 100, 77), (5, 2048, 512), (8, 333, 1000), (9, 64, 64), (42, 512, 2048),
          (128, 64, 128), (129, 65, 129), (130, 1001, 515), (255, 2048, 72), (257, 4096, 200), (700, 192, 2500),
          (2562, 515, 131), (5000, 512, 2048), (9001, 520, 1000), (3, 8192, 40), (20000, 72, 8)]


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("layout", ["nk", "kn"])
@pytest.mark.parametrize("act,bias,residual,out", [(None, None, False, BF), ("gelu", F32, False, BF),
                                                   ("swish", BF, True, BF), (None, F32, True, F32),
                                                   ("gelu", None, False, F32)])
def test_linear_forward(cuda, m, k, n, layout, act, bias, residual, out):
  pr = _pr()
  a, w, b, r = _problem(m, k, n, m + k + n, layout)
  b = None if bias is None else b.to(bias)
  r = r.to(out) if residual else None
  y = pr.linear(a, w, b, r, activation=act, out_dtype=out)
  assert y.dtype == out and y.shape == (m, n)
  assert _rel(y, _linear64(a, w, b, r, act)) <= TOL_PRODUCT[out]
  assert torch.equal(y, pr.linear(a, w, b, r, activation=act, out_dtype=out))
  _no_device_error()


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("act,residual,out", [(None, False, F32), ("gelu", True, BF), ("swish", True, F32)])
def test_linear_fp8_forward(cuda, m, k, n, act, residual, out):
  """On the 8-bit operands' own values: the product of what they stand for."""
  pr = _pr()
  a, w, b, r = _problem(m, k, n, m + 2 * k + n)
  a8, sa = pr.quantize_fp8(a)
  w8, sw = pr.quantize_fp8(w)
  r = r.to(out) if residual else None
  y = pr.linear_fp8(a8, sa, w8, sw, b, r, activation=act, out_dtype=out)
  a64, w64 = a8.double() * sa.double()[:, None], w8.double() * sw.double()[:, None]
  assert _rel(y, _linear64(a64, w64, b, r, act)) <= TOL_PRODUCT[out]
  _no_device_error()


@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 512, 77), (3, 700, 300), (8, 64, 2048), (42, 512, 256), (130, 1001, 515),
                                   (700, 192, 2500), (2562, 515, 131), (9001, 520, 1000)])
@pytest.mark.parametrize("layout", ["nk", "kn"])
@pytest.mark.parametrize("act,bias,residual,out", [(None, F32, True, BF), ("gelu", F32, True, F32), ("swish", BF, False, BF),
                                                   (None, BF, True, F32), ("gelu", None, False, BF)])
def test_linear_gradients(cuda, m, k, n, layout, act, bias, residual, out):
  pr = _pr()
  a, w, b, r = _problem(m, k, n, m + k, layout)
  b = None if bias is None else b.to(bias).requires_grad_()
  r = r.to(out).requires_grad_() if residual else None
  a.requires_grad_()
  w.requires_grad_()
  dy = torch.randn(m, n, device=cuda, generator=_gen(n)).to(out)
  ins = [t for t in (a, w, b, r) if t is not None]
  grads = torch.autograd.grad(pr.linear(a, w, b, r, activation=act, out_dtype=out), ins, dy)
  again = torch.autograd.grad(pr.linear(a, w, b, r, activation=act, out_dtype=out), ins, dy)
  ref = [t.detach().double().requires_grad_() for t in ins]
  it = iter(ref)
  args = [next(it), next(it), next(it) if b is not None else None, next(it) if r is not None else None]
  want = torch.autograd.grad(_linear64(*args, act), ref, dy.double())
  for t, x, z, c in zip(ins, grads, again, want):
    assert x.dtype == t.dtype and x.shape == t.shape and torch.equal(x, z)
    assert _rel(x, c) <= (TOL_GRAD[BF] if t.dtype == BF else TOL_GRAD[F32])
  _no_device_error()


def test_linear_gradient_against_differences(cuda):
  """Differences of the kernel's own float32 output. Without an activation the output is linear in each input, so a step
  of one (exact in bf16 here: small integers) gives the gradient up to rounding; with GELU, central differences over the
  float32 bias, step 1e-2."""
  pr, g = _pr(), _gen(8)
  m, k, n = 40, 96, 72
  ints = lambda *s: torch.randint(-3, 4, s, device=cuda, generator=g).to(BF)  # noqa: E731
  a, w, c = ints(m, k), ints(n, k), ints(m, n).float()
  da, dw = ints(m, k), ints(n, k)
  b = torch.randn(n, device=cuda, generator=g)
  ag, wg, bg = a.clone().requires_grad_(), w.clone().requires_grad_(), b.clone().requires_grad_()
  ga, gw = torch.autograd.grad(pr.linear(ag, wg, b, out_dtype=F32), (ag, wg), c)
  f = lambda aa, ww: (pr.linear(aa, ww, b, out_dtype=F32).double() * c.double()).sum()  # noqa: E731
  size = float(c.norm()) * k ** 0.5 * 4
  assert abs(float(f(a + da, w) - f(a, w)) - float((ga.double() * da.double()).sum())) <= 2.0 ** -8 * size
  assert abs(float(f(a, w + dw) - f(a, w)) - float((gw.double() * dw.double()).sum())) <= 2.0 ** -8 * size
  a, w = 0.1 * a, 0.2 * w
  gb, = torch.autograd.grad(pr.linear(a, w, bg, activation="gelu", out_dtype=F32), bg, c)
  db, t = torch.randn(n, device=cuda, generator=g), 1e-2
  f = lambda bb: (pr.linear(a, w, bb, activation="gelu", out_dtype=F32).double() * c.double()).sum()  # noqa: E731
  diff = float(f(b + t * db) - f(b - t * db)) / (2 * t)
  assert abs(diff - float((gb.double() * db.double()).sum())) <= 1e-3 * float(c.norm()) * float(db.norm())


@pytest.mark.parametrize("m,k,n", [(9001, 520, 1000), (9001, 64, 1000), (20000, 2048, 512), (9001, 1040, 333)])
@pytest.mark.parametrize("out", [BF, F32])
def test_linear_many_tiles_again_and_again(cuda, m, k, n, out):
  """Tiles that follow one another in a block reuse its slots, accumulators and biases: thirty calls, the same bits."""
  pr = _pr()
  a, w, b, r = _problem(m, k, n, m + k)
  r = r.to(out)
  y = pr.linear(a, w, b, r, activation="swish", out_dtype=out)
  assert _rel(y, _linear64(a, w, b, r, "swish")) <= TOL_PRODUCT[out]
  for _ in range(30):
    assert torch.equal(y, pr.linear(a, w, b, r, activation="swish", out_dtype=out))


@pytest.mark.parametrize("act", ["gelu", "swish"])
def test_linear_activation_over_its_range(cuda, act):
  """Each pre-activation from -40 to 40 (the bias, with a zero product) and +-1e4: values to bf16 and float32 accuracy
  (absolutely below the smallest value that counts), slopes to float32."""
  pr = _pr()
  b = torch.cat([torch.linspace(-40, 40, 4001, device=cuda), torch.tensor([-1e4, 1e4, 0.0], device=cuda)])
  n = b.numel()
  a, w = torch.zeros(16, 64, device=cuda, dtype=BF), torch.zeros(n, 64, device=cuda, dtype=BF)
  b64 = b.double().requires_grad_()
  want = _act64(b64, act)
  slope, = torch.autograd.grad(want.sum(), b64)
  y = pr.linear(a, w, b, activation=act, out_dtype=F32)
  # The exponential's argument reaches 80 log2(e): its relative error is that times 2^-24 and a few roundings.
  assert bool(((y.double() - want).abs() <= 1e-5 * want.abs() + 1e-12).all())
  bg = b.clone().requires_grad_()
  one = torch.zeros(16, n, device=cuda)
  one[3] = 1
  got, = torch.autograd.grad(pr.linear(a, w, bg, activation=act, out_dtype=F32), bg, one)
  assert float((got.double() - slope).abs().max()) <= 2e-6


def test_linear_strides_views_and_broadcast(cuda):
  """Operands that TMA cannot address (odd strides, bases off 16 bytes) or that overlap, residuals and weights in views;
  leading dimensions."""
  pr, g = _pr(), _gen(4)
  buf = torch.randn(300, 1111, device=cuda, generator=g).to(BF)
  wbuf = torch.randn(333, 1111, device=cuda, generator=g).to(BF)
  rbuf = torch.randn(300, 999, device=cuda, generator=g).to(BF)
  for a in (buf[:, 3:515], buf[:, :512], buf[::3, 8:520], buf[:1, :512].expand(300, 512), buf.t()[:512, :300].t(),
            buf[:4, 1:513], buf[:300, :1024:2]):
    for w in (wbuf[:200, :512], wbuf[1:130, 5:517], wbuf.t()[:512, :200].t(), wbuf[:1, :512].expand(72, 512)):
      m, n = a.shape[0], w.shape[0]
      r = rbuf[:m, 1:n + 1]
      y = pr.linear(a, w, None, r, activation="swish")
      assert _rel(y, _linear64(a, w, None, r, "swish")) <= TOL_PRODUCT[BF]
      y = pr.linear(a, w, None, rbuf[:1, :n].expand(m, n))
      assert _rel(y, _linear64(a, w, None, rbuf[:1, :n], None)) <= TOL_PRODUCT[BF]
  a3 = buf[:24, :512].reshape(2, 12, 512)
  y = pr.linear(a3, wbuf[:77, :512], out_dtype=F32)
  assert y.shape == (2, 12, 77) and _rel(y, a3.double() @ wbuf[:77, :512].double().t()) <= TOL_PRODUCT[F32]
  # A gradient that is one value broadcast (sum().backward()) and one through a shared operand.
  w = wbuf[:130, :512].clone().requires_grad_()
  a = buf[:100, :512].clone().requires_grad_()
  (pr.linear(a, w).float().sum() + pr.linear(a, w, activation="gelu").float().sum()).backward()
  aa, ww = a.detach().double().requires_grad_(), w.detach().double().requires_grad_()
  p = aa @ ww.t()
  (p.sum() + _act64(p, "gelu").sum()).backward()
  assert _rel(a.grad, aa.grad) <= TOL_GRAD[BF] and _rel(w.grad, ww.grad) <= TOL_GRAD[BF]
  _no_device_error()


def test_linear_writes_nothing_past_its_rows(cuda):
  """Through the C ABI into a larger tensor: the rows and columns around the output stay."""
  import ctypes
  from faster_weathernext import _lib
  lib = _lib.lib()
  for m, k, n, ld in ((300, 128, 200, 256), (257, 128, 129, 131), (5, 64, 33, 40), (40, 128, 72, 80)):
    a, w, b, r = _problem(m, k, n, m)
    big = torch.full((m + 4, ld), 7.0, device=cuda, dtype=BF)
    desc = _lib.LinearDesc(m, n, k, _lib.DTYPE_BF16, _lib.DTYPE_BF16, _lib.DTYPE_F32, 0, _lib.ACT_NONE, 0, k, k, 0, ld)
    size = ctypes.c_size_t(0)
    _lib.check(lib.fwn_linear_workspace_size(ctypes.byref(desc), a.data_ptr(), w.data_ptr(), ctypes.byref(size)))
    ws = torch.empty(max(1, size.value), device=cuda, dtype=torch.uint8)
    _lib.check(lib.fwn_linear(ctypes.byref(desc), a.data_ptr(), None, w.data_ptr(), None, b.data_ptr(), None,
                              big[2:].data_ptr(), None, ws.data_ptr(), size.value, torch.cuda.current_stream().cuda_stream))
    assert _rel(big[2:m + 2, :n], _linear64(a, w, b, None, None)) <= TOL_PRODUCT[BF]
    big[2:m + 2, :n] = 7.0
    assert bool((big == 7.0).all())


def test_linear_nan_and_infinity_stay_in_their_rows(cuda):
  pr = _pr()
  a, w, b, r = _problem(200, 512, 300, 1)
  a[7, 100] = float("nan")
  a[9, 3] = float("inf")
  y = pr.linear(a, w, b, activation="swish")
  keep = [i for i in range(200) if i not in (7, 9)]
  assert bool(torch.isnan(y[7].float()).all()) and not bool(torch.isfinite(y[9].float()).all())
  assert _rel(y[keep], _linear64(a, w, b, None, "swish")[keep]) <= TOL_PRODUCT[BF]


def test_linear_empty_and_refusals(cuda):
  pr = _pr()
  a, w, b, r = _problem(12, 64, 40, 2)
  e = torch.empty(0, 64, device=cuda, dtype=BF, requires_grad=True)
  wg, bg = w.clone().requires_grad_(), b.clone().requires_grad_()
  y = pr.linear(e, wg, bg, activation="gelu")
  assert y.shape == (0, 40)
  ge, gw, gb = torch.autograd.grad(y.float().sum(), (e, wg, bg))
  assert ge.shape == (0, 64) and bool((gw == 0).all()) and bool((gb == 0).all())
  a8, sa = pr.quantize_fp8(a)
  w8, sw = pr.quantize_fp8(w)
  for bad in (lambda: pr.linear(a, w[:, :63]), lambda: pr.linear(a, w, b[:39]), lambda: pr.linear(a, w, None, r[:, :39].to(BF)),
              lambda: pr.linear(a, w, activation="relu"), lambda: pr.linear(a, w, out_dtype=torch.float16),
              lambda: pr.linear(a.cpu(), w), lambda: pr.linear(a, w.cpu()), lambda: pr.linear(a, w[0]),
              lambda: pr.linear_fp8(a8, sa[:5], w8, sw), lambda: pr.linear_fp8(a8, sa, w8, sw[:5])):
    with pytest.raises(ValueError):
      bad()
  for bad in (lambda: pr.linear(a.float(), w), lambda: pr.linear(a, w.float()), lambda: pr.linear(a, w, None, r),
              lambda: pr.linear(a, w, b.double()), lambda: pr.linear_fp8(a, sa, w8, sw),
              lambda: pr.linear_fp8(a8, sa.double(), w8, sw)):
    with pytest.raises(TypeError):
      bad()


def test_linear_offsets_past_32_bits(cuda):
  """1,100,000 rows by 2,048 columns of output (2.3e9 values): the last rows against float64."""
  pr = _pr()
  m, k, n = 1_100_000, 64, 2048
  a, w, b, _ = _problem(1, k, n, 3)
  a = torch.randn(m, k, device=cuda, generator=_gen(9)).to(BF)
  y = pr.linear(a, w, b, activation="gelu")
  for rows in (slice(0, 2), slice(m // 2, m // 2 + 2), slice(m - 130, m)):
    assert _rel(y[rows], _linear64(a[rows], w, b, None, "gelu")) <= TOL_PRODUCT[BF]


def test_projection_on_another_stream(cuda):
  """Inputs written, and calls made, on a side stream; the workspaces come from that stream's memory."""
  pr = _pr()
  st = torch.cuda.Stream()
  a, w, b, r = _problem(700, 515, 333, 6)
  x, wr = torch.randn(700, 515, device=cuda, generator=_gen(1)), torch.ones(515, device=cuda)
  torch.cuda.synchronize()
  with torch.cuda.stream(st):
    for _ in range(20):
      x2 = x * 2
      h = pr.rms_norm(x2, wr)
      y = pr.linear(h, w, b, activation="gelu")
  st.synchronize()
  h64, _ = _rms64(2 * x.double(), None, None, 1e-6)
  assert _rel(h, h64) <= TOL[BF]
  assert _rel(y, _linear64(h, w, b, None, "gelu")) <= TOL_PRODUCT[BF]
