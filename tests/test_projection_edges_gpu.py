"""GPU: the pre-norm projections where one value is not a number or infinite and where an activation's
tail counts. Every case runs on each way a product takes: few rows (m <= 8), one tile, split k, many tiles on pairs of SMs.

Bounds. Columns beside a NaN: those of the same products without one (test_projection_gpu.py). An activation's value,
each by itself, as a bf16 result: half a bf16 step, at most 2^-8 of the value; 1e-5 of it for the arithmetic (the
exponential's argument reaches 80 log2(e), times 2^-24 and a few roundings); and absolutely 6e-9 (GELU) or 2.1e-8
(swish): the value at -5.5 or -21, below which it is held there, is within that."""
import pytest
import torch

from test_projection_gpu import BF, F32, TOL_GRAD, TOL_PRODUCT, _act64, _gen, _linear64, _no_device_error, _pr, _problem, _rel

pytestmark = pytest.mark.gpu

TAIL = {"gelu": 6e-9, "swish": 2.1e-8}
# m, k, n: few rows; one tile; split k, of bf16 and of e4m3; few tiles; pairs of SMs, short k, odd rows and long k.
PATHS = [(5, 256, 130), (42, 256, 130), (42, 2048, 512), (42, 4096, 512), (300, 256, 130), (9001, 520, 1000),
         (9001, 1040, 333), (9001, 1536, 1000)]


def _operands(kind, a, w):
  """(call with these operands, their values in float64)."""
  pr = _pr()
  if kind == "bf16":
    return lambda *rest, **kw: pr.linear(a, w, *rest, **kw), a.double(), w.double()
  a8, sa = pr.quantize_fp8(a)
  w8, sw = pr.quantize_fp8(w)
  return (lambda *rest, **kw: pr.linear_fp8(a8, sa, w8, sw, *rest, **kw), a8.double() * sa.double()[:, None],
          w8.double() * sw.double()[:, None])


# ---- a NaN stays in its column --------------------------------------------------------------------------------------

@pytest.mark.parametrize("m,k,n", PATHS)
@pytest.mark.parametrize("kind,out", [("bf16", BF), ("bf16", F32), ("fp8", BF), ("fp8", F32)])
@pytest.mark.parametrize("act", ["gelu", "swish"])
def test_a_nan_in_a_bias_or_weight_row_stays_in_its_column(cuda, m, k, n, kind, out, act):
  a, w, b, _ = _problem(m, k, n, m + n)
  b[17] = float("nan")
  w[66, 3] = float("nan")
  call, a64, w64 = _operands(kind, a, w)
  y = call(b, activation=act, out_dtype=out)
  keep = [i for i in range(n) if i not in (17, 66)]
  assert bool(torch.isnan(y[:, [17, 66]].float()).all())
  assert _rel(y[:, keep], _linear64(a64, w64, b, None, act)[:, keep]) <= TOL_PRODUCT[out]


@pytest.mark.parametrize("m,k,n", PATHS)
@pytest.mark.parametrize("act", ["gelu", "swish"])
def test_a_nan_in_a_bias_or_weight_row_stays_in_its_gradients(cuda, m, k, n, act):
  """d_weight's rows and d_bias's entries of the columns with a NaN are NaN, all others numbers; d_a, a sum over all
  columns, is NaN."""
  pr = _pr()
  a, w, b, _ = _problem(m, k, n, m + k)
  b[17] = float("nan")
  w[66, 3] = float("nan")
  dy = torch.randn(m, n, device=cuda, generator=_gen(n)).to(BF)
  ins = [t.requires_grad_() for t in (a, w, b)]
  d_a, d_w, d_b = torch.autograd.grad(pr.linear(*ins, activation=act), ins, dy)
  ref = [t.detach().double().requires_grad_() for t in ins]
  _, want_w, want_b = torch.autograd.grad(_linear64(*ref, None, act), ref, dy.double())
  keep = [i for i in range(n) if i not in (17, 66)]
  assert bool(torch.isnan(d_a.float()).all()) and bool(torch.isnan(d_w[[17, 66]].float()).all())
  assert bool(torch.isnan(d_b[[17, 66]]).all())
  assert _rel(d_w[keep], want_w[keep]) <= TOL_GRAD[BF] and _rel(d_b[keep], want_b[keep]) <= TOL_GRAD[F32]


# ---- activations over their range -----------------------------------------------------------------------------------

@pytest.mark.parametrize("m,k,n", [(1, 64, 4003), (16, 64, 4003), (300, 64, 4003), (3000, 64, 4003), (40, 2048, 515),
                                   (40, 4096, 515), (9001, 1536, 515), (9001, 1536, 1000)])
@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("act", ["gelu", "swish"])
def test_bf16_results_of_an_activation_over_its_range(cuda, m, k, n, kind, act):
  """Pre-activations from -40 to 40 and beyond (the bias, with a zero product), each value by itself, for bf16 and 8-bit
  operands and on every way a product takes: a row's values do not depend on the rows it came with."""
  b = torch.cat([torch.linspace(-40, 40, n - 6, device=cuda),
                 torch.tensor([-1e4, 1e4, 0.0, -3.0, -4.0, -8.0], device=cuda)])
  a = torch.zeros(m, k, device=cuda, dtype=BF)
  w = torch.randn(n, k, device=cuda, generator=_gen(k)).to(BF)
  want = _act64(b.double(), act)
  y = _operands(kind, a, w)[0](b, activation=act).double()
  assert bool(((y - want).abs() <= (2.0 ** -8 + 1e-5) * want.abs() + TAIL[act]).all())
  _no_device_error()


@pytest.mark.parametrize("m,k,n", PATHS)
@pytest.mark.parametrize("kind,out", [("bf16", BF), ("bf16", F32), ("fp8", BF), ("fp8", F32)])
@pytest.mark.parametrize("act", ["gelu", "swish"])
def test_infinite_pre_activations_give_the_limits(cuda, m, k, n, kind, out, act):
  """A bias of infinity gives infinity, one of -infinity (a unit that is switched off) 0, on every way a product takes."""
  a, w, b, _ = _problem(m, k, n, m + n)
  b[17], b[66] = float("inf"), float("-inf")
  call, a64, w64 = _operands(kind, a, w)
  y = call(b, activation=act, out_dtype=out)
  keep = [i for i in range(n) if i not in (17, 66)]
  assert bool((y[:, 17].float() == float("inf")).all()) and bool((y[:, 66].float().abs() <= TAIL[act]).all())
  assert _rel(y[:, keep], _linear64(a64, w64, b, None, act)[:, keep]) <= TOL_PRODUCT[out]


@pytest.mark.parametrize("m,k,n", PATHS)
@pytest.mark.parametrize("act", ["gelu", "swish"])
def test_infinite_pre_activations_give_the_slopes_limits(cuda, m, k, n, act):
  """Slope 1 at infinity, 0 at -infinity (held at that of -5.5 or -21: below 5e-8), the other columns' as without them."""
  pr = _pr()
  a, w, b, _ = _problem(m, k, n, m + k)
  b[17], b[66] = float("inf"), float("-inf")
  dy = torch.randn(m, n, device=cuda, generator=_gen(n)).to(BF)
  ins = [t.requires_grad_() for t in (a, w, b)]
  _, d_w, d_b = torch.autograd.grad(pr.linear(*ins, activation=act), ins, dy)
  ref = [t.detach().double().requires_grad_() for t in ins]
  _, want_w, want_b = torch.autograd.grad(_linear64(*ref, None, act), ref, dy.double())
  keep = [i for i in range(n) if i not in (17, 66)]
  assert _rel(d_w[keep], want_w[keep]) <= TOL_GRAD[BF] and _rel(d_b[keep], want_b[keep]) <= TOL_GRAD[F32]
  assert abs(float(d_b[17]) - float(dy[:, 17].double().sum())) <= 1e-5 * float(dy[:, 17].double().norm())
  assert abs(float(d_b[66])) <= 5e-8 * float(dy[:, 66].double().abs().sum())


# ---- derivatives that cannot be given are refused -------------------------------------------------------------------

def test_8_bit_calls_refuse_inputs_that_require_a_gradient(cuda):
  """Their results would be cut off from the input; under no_grad, and for a weight laid out once, they are constants."""
  pr = _pr()
  a, w, b, r = _problem(40, 64, 48, 1)
  x, wn = torch.randn(40, 64, device=cuda), torch.ones(64, device=cuda)
  a8, sa = pr.quantize_fp8(a)
  w8, sw = pr.quantize_fp8(w.clone().requires_grad_())
  assert not w8.requires_grad and not sw.requires_grad
  r = r.to(BF)
  leaf = lambda t: t.clone().requires_grad_()  # noqa: E731
  calls = (lambda: pr.rms_norm_fp8(leaf(x), wn), lambda: pr.rms_norm_fp8(x, leaf(wn)),
           lambda: pr.rms_norm_fp8(x, None, leaf(x)), lambda: pr.linear_fp8(a8, leaf(sa), w8, sw),
           lambda: pr.linear_fp8(a8, sa, w8, leaf(sw)), lambda: pr.linear_fp8(a8, sa, w8, sw, leaf(b)),
           lambda: pr.linear_fp8(a8, sa, w8, sw, None, leaf(r)))
  for call in calls:
    with pytest.raises(NotImplementedError):
      call()
    with torch.no_grad():
      call()


def test_forward_mode_is_refused(cuda):
  """A tangent of any input, in forward calls and in gradients, under no_grad too; calls without one pass at a dual level."""
  from torch.autograd import forward_ad as fw
  pr = _pr()
  a, w, b, r = _problem(40, 64, 48, 1)
  x, wn = torch.randn(40, 64, device=cuda), torch.ones(64, device=cuda)
  a8, sa = pr.quantize_fp8(a)
  w8, sw = pr.quantize_fp8(w)
  r = r.to(BF)
  ag, xg = a.clone().requires_grad_(), x.clone().requires_grad_()
  y, h = pr.linear(ag, w, b, activation="gelu"), pr.rms_norm(xg, wn)
  with fw.dual_level():
    dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
    calls = (lambda f: pr.linear(f(a), w), lambda f: pr.linear(a, f(w)), lambda f: pr.linear(a, w, f(b)),
             lambda f: pr.linear(a, w, None, f(r)), lambda f: pr.rms_norm(f(x)), lambda f: pr.rms_norm(x, f(wn)),
             lambda f: pr.rms_norm(x, wn, f(x)), lambda f: pr.rms_norm_fp8(f(x)),
             lambda f: pr.linear_fp8(a8, sa, w8, sw, f(b)), lambda f: pr.linear_fp8(a8, sa, w8, sw, None, f(r)),
             lambda f: torch.autograd.grad(y, ag, f(torch.ones_like(y)), retain_graph=True),
             lambda f: torch.autograd.grad(h, xg, f(torch.ones_like(h)), retain_graph=True))
    for call in calls:
      with pytest.raises(NotImplementedError):
        call(dual)
      call(lambda t: t)
    for call in calls[:10]:
      with torch.no_grad(), pytest.raises(NotImplementedError):
        call(dual)


def test_second_derivatives_are_refused(cuda):
  """A gradient that keeps a graph through a product or norm is refused, whether or not what comes in has a graph; what a
  residual or the stored sum passes through alone has its own, right, graph."""
  pr = _pr()
  a, w, b, r = _problem(40, 64, 48, 1)
  ins = [t.requires_grad_() for t in (a, w, b, r)]
  for f in (lambda y: y.sum(), lambda y: y.square().sum()):
    y = pr.linear(a, w, b, r, activation="gelu", out_dtype=F32)
    with pytest.raises(NotImplementedError):
      torch.autograd.grad(f(y), ins, retain_graph=True, create_graph=True)
    torch.autograd.grad(f(y), ins)
  y = pr.linear(a.detach(), w.detach(), b.detach(), r, out_dtype=F32)
  g, = torch.autograd.grad(y.pow(3).sum(), r, create_graph=True)
  assert torch.allclose(torch.autograd.grad(g.sum(), r)[0], 6 * y)
  x, s, wn = torch.randn(40, 64, device=cuda), torch.randn(40, 64, device=cuda), torch.ones(64, device=cuda)
  ins = [t.requires_grad_() for t in (x, s, wn)]
  for f in (lambda h: h.sum(), lambda h: h.square().sum()):
    h, total = pr.rms_norm(x, wn, s, out_dtype=F32)
    with pytest.raises(NotImplementedError):
      torch.autograd.grad(f(h), ins, retain_graph=True, create_graph=True)
    torch.autograd.grad(f(h), ins, retain_graph=True)
  g, = torch.autograd.grad(total.pow(3).sum(), x, create_graph=True)
  assert torch.allclose(torch.autograd.grad(g.sum(), x)[0], 6 * total)
