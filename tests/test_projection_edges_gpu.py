"""GPU: the pre-norm projections where one value is not a number. Every case runs on each way a product takes: few rows
(m <= 8), one tile, split k, many tiles on pairs of SMs.

Bounds. Columns beside a NaN: those of the same products without one (test_projection_gpu.py)."""
import pytest
import torch

from test_projection_gpu import BF, F32, TOL_GRAD, TOL_PRODUCT, _gen, _linear64, _pr, _problem, _rel

pytestmark = pytest.mark.gpu

# m, k, n: few rows; one tile; split k; few tiles; pairs of SMs, short k and long.
PATHS = [(5, 256, 130), (42, 256, 130), (42, 2048, 512), (300, 256, 130), (9001, 520, 1000), (9001, 1040, 333)]


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
