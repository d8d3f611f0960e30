"""GPU: the routing of rows to experts and back against its definition: choices, ties, places, gradients, values off bounds,
every size of block, graphs, refusals.

Tolerances: weights are quotients of sums of at most 16 exponentials in float32 (20 units of the last place, with exp's 2 and
the difference's rounding times the logits' span of about 10); sums of at most 16 products in float32 and a dot product of d
terms, (d / 32 + 40) 2^-24 of the absolute terms' sum, then half a step of the type.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24


def _randn(seed):
  g = torch.Generator(device="cuda").manual_seed(seed)
  return lambda *s: torch.randn(*s, device="cuda", generator=g)


def _close(got, want, room, label=""):
  assert got.shape == want.shape, label
  off = (got.double() - want).abs() - torch.finfo(got.dtype).eps / 2 * 1.0001 * want.abs() - room - 1e-38
  assert not (off > 0).any() and torch.isfinite(got.double()).all(), f"{label}: {off.max().item():.3e} above its bound"


def _order(logits, k):
  """The choice by NumPy: largest first, equal ones by index, NaN largest."""
  x = logits.detach().double().cpu().numpy()
  x = np.where(np.isnan(x), np.inf, x) + 0.0
  nan = np.isnan(logits.detach().double().cpu().numpy())
  idx = np.stack([np.lexsort((np.arange(x.shape[1]), -row, ~bad)) for row, bad in zip(x, nan)]) if x.shape[0] else np.zeros(x.shape, np.int64)
  return idx[:, :k]


def _check_plan(r, idx, e):
  rows, k = idx.shape
  assert np.array_equal(r.experts.cpu().numpy(), idx)
  flat = idx.reshape(-1)
  order = np.argsort(flat, kind="stable")
  assert np.array_equal(r.order.cpu().numpy(), order)
  position = np.empty_like(order)
  position[order] = np.arange(rows * k)
  assert np.array_equal(r.position.cpu().numpy(), position.reshape(rows, k))
  assert np.array_equal(r.offsets.cpu().numpy(), np.concatenate(([0], np.cumsum(np.bincount(flat, minlength=e)))))
  assert all(t.dtype is torch.int32 for t in (r.experts, r.position, r.order, r.offsets))


@pytest.mark.parametrize("rows,e,k", [(1, 1, 1), (1, 64, 4), (3, 8, 8), (127, 5, 3), (128, 8, 2), (129, 8, 2), (1000, 9, 1),
                                      (1000, 16, 16), (513, 17, 3), (2000, 33, 8), (700, 64, 2), (700, 128, 5), (400, 200, 12),
                                      (400, 300, 2), (260, 1023, 16), (100, 1023, 7), (40000, 8, 2), (300, 65, 4), (129, 10, 10), (1000, 31, 6), (128, 300, 3)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_route(cuda, rows, e, k, dtype):
  from faster_weathernext import experts
  rand = _randn(rows + e)
  logits = (2 * rand(rows, e)).to(dtype).requires_grad_()   # bf16: equal logits are common
  r = experts.route(logits, k)
  idx = _order(logits, k)
  _check_plan(r, idx, e)
  l64 = logits.detach().double().requires_grad_()
  w64 = torch.softmax(torch.gather(l64, 1, torch.from_numpy(idx).cuda()), 1)
  _close(r.weights.detach(), w64.detach(), 40 * U * w64.detach(), "weights")
  dw = rand(rows, k)
  got, = torch.autograd.grad(r.weights, logits, dw)
  want, = torch.autograd.grad(w64, l64, dw.double())
  assert got.dtype is dtype
  size = (w64.detach() * (dw.double().abs() + (w64.detach() * dw.double().abs()).sum(1, keepdim=True))).sum(1, keepdim=True)
  _close(got, want, 80 * U * size, "d_logits")


@pytest.mark.parametrize("times", [1, 40])
def test_ties_and_special_logits(cuda, times):
  """Few rows (one block, several lanes a row) and many (a thread a row)."""
  from faster_weathernext import experts
  inf, nan = float("inf"), float("nan")
  logits = torch.tensor([[0.0, -0.0, 0.0, 0.0], [1, 1, 1, 1], [-inf, 3, -inf, -inf], [-inf] * 4, [2, nan, 5, nan],
                         [-3.4e38, -inf, -3.4e38, -inf], [3.4e38, 3.4e38, 0, -3.4e38]], device="cuda").repeat(times, 1).requires_grad_()
  r = experts.route(logits, 2)
  _check_plan(r, np.tile(np.array([[0, 1], [0, 1], [1, 0], [0, 1], [1, 3], [0, 2], [0, 1]]), (times, 1)), 4)
  w = r.weights.detach()
  half = torch.tensor([0.5, 0.5], device="cuda")
  assert torch.equal(w[0], half) and torch.equal(w[1], half) and torch.equal(w[5], half) and torch.equal(w[6], half)
  assert torch.equal(w[2], torch.tensor([1.0, 0.0], device="cuda")) and (w[3] == 0).all() and torch.isnan(w[4]).all()
  g, = torch.autograd.grad(r.weights, logits, torch.tensor([[1.0, 2.0]], device="cuda").repeat(7 * times, 1))
  assert (g[2] == 0).all() and (g[3] == 0).all() and torch.isfinite(g[[0, 1, 5, 6]]).all() and torch.equal(g[0], torch.tensor([-0.25, 0.25, 0, 0], device="cuda"))


@pytest.mark.parametrize("rows,e,k,d", [(1, 4, 2, 2048), (7, 4, 1, 8), (130, 8, 2, 512), (333, 6, 3, 65), (257, 16, 4, 1000), (90, 32, 8, 129),
                                        (50, 20, 16, 264), (12, 4, 2, 1), (2000, 8, 2, 515), (301, 8, 2, 514), (77, 8, 8, 128), (77, 8, 3, 120),
                                        (1001, 12, 12, 64), (33, 20, 9, 56), (9, 4, 1, 250)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_there_and_back(cuda, rows, e, k, d, dtype):
  from faster_weathernext import experts
  rand = _randn(rows + d)
  logits = rand(rows, e).requires_grad_()
  x, y = rand(rows, d).to(dtype).requires_grad_(), rand(rows * k, d).to(dtype).requires_grad_()
  r = experts.route(logits, k)
  moved, back = experts.dispatch(x, r), experts.combine(y, r)
  d_moved, d_back = rand(rows * k, d).to(dtype), rand(rows, d).to(dtype)
  d_x, d_y, d_w = torch.autograd.grad((moved, back), (x, y, r.weights), (d_moved, d_back))
  source, pos = (r.order // k).long(), r.position.long()
  assert torch.equal(moved.detach(), x.detach()[source])
  w = r.weights.detach().double()
  parts = y.detach().double()[pos.reshape(-1)].view(rows, k, d)
  _close(back.detach(), (w[:, :, None] * parts).sum(1), 20 * U * (w[:, :, None] * parts).abs().sum(1), "combine")
  dm = d_moved.double()[pos.reshape(-1)].view(rows, k, d)
  _close(d_x, dm.sum(1), 20 * U * dm.abs().sum(1), "d_x")
  want = torch.empty(rows * k, d, dtype=torch.float64, device="cuda")
  want[pos.reshape(-1)] = (w[:, :, None] * d_back.double()[:, None, :]).reshape(-1, d)
  _close(d_y, want, 2 * U * want.abs(), "d_y")
  terms = parts * d_back.double()[:, None, :]
  _close(d_w, terms.sum(2), (d / 32 + 40) * U * terms.abs().sum(2), "d_weights")


def test_partial_gradients_and_strides(cuda):
  from faster_weathernext import experts
  rand = _randn(4)
  wide = rand(50, 40)
  logits = wide[:, 3:11].detach().requires_grad_()
  r = experts.route(logits, 2)
  same = experts.route(logits.detach().clone(), 2)
  assert torch.equal(r.order, same.order) and torch.equal(r.weights, same.weights)
  x = rand(64, 50).t().detach().requires_grad_()
  assert torch.equal(experts.dispatch(x, r).detach(), experts.dispatch(x.detach().contiguous(), r))
  strided = rand(50, 3, 64).to(BF16)[:, 1]
  assert torch.equal(experts.dispatch(strided, r), experts.dispatch(strided.contiguous(), r))
  y = rand(100, 64)
  only_w, = torch.autograd.grad(experts.combine(y, r), r.weights, torch.ones(50, 64, device="cuda"), retain_graph=True)
  y.requires_grad_()
  both = torch.autograd.grad(experts.combine(y, r), (y, r.weights), torch.ones(50, 1, device="cuda").expand(50, 64), retain_graph=True)
  assert torch.equal(both[1], only_w)
  only_y, = torch.autograd.grad(experts.combine(y, same), y, torch.ones(50, 64, device="cuda"))
  assert torch.equal(only_y, both[0])


def test_empty(cuda):
  from faster_weathernext import experts
  logits = torch.zeros(0, 5, device="cuda", requires_grad=True)
  x = torch.zeros(0, 16, device="cuda", requires_grad=True)
  r = experts.route(logits, 2)
  assert r.offsets.tolist() == [0] * 6 and r.order.shape == (0,)
  out = experts.combine(experts.dispatch(x, r), r)
  gx, gl = torch.autograd.grad(out, (x, logits), torch.zeros(0, 16, device="cuda"))
  assert gx.shape == (0, 16) and gl.shape == (0, 5)


def test_nan_rows_stay_apart(cuda):
  from faster_weathernext import experts
  rand = _randn(8)
  logits, x = rand(200, 8), rand(200, 64)
  x[17] = float("nan")
  r = experts.route(logits, 2)
  out = experts.combine(experts.dispatch(x, r), r)
  assert torch.isnan(out[17]).all() and torch.isfinite(out[torch.arange(200, device="cuda") != 17]).all()


def test_positions_outside_are_reported(cuda):
  from faster_weathernext import _lib, experts
  rand = _randn(9)
  r = experts.route(rand(20, 4), 2)
  bad = r.position.clone()
  bad[3, 1], bad[4, 0] = 40, -1
  wrong = r._replace(position=bad)
  x = rand(20, 64)
  out = experts.combine(rand(40, 64), wrong)
  assert out.shape == (20, 64) and _lib.device_error() == _lib.FWN_ERR_INVALID_ARGUMENT
  experts.dispatch(x, wrong)
  assert _lib.device_error() == _lib.FWN_ERR_INVALID_ARGUMENT and _lib.device_error() == 0


def test_graph_and_repeats(cuda):
  from faster_weathernext import experts
  rand = _randn(10)
  logits, x = rand(3000, 16).requires_grad_(), rand(3000, 128).to(BF16).requires_grad_()

  def step():
    r = experts.route(logits, 3)
    out = experts.combine(experts.dispatch(x, r), r)
    return [r.experts, r.order, r.offsets, out.detach(), *torch.autograd.grad(out, (logits, x), torch.ones_like(out))]

  first = step()
  assert all(torch.equal(a, b) for a, b in zip(first, step()))
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = step()
  with torch.no_grad():
    logits.copy_(rand(3000, 16))
  graph.replay()
  assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_refusals(cuda):
  from faster_weathernext import experts
  rand = _randn(11)
  logits, x = rand(10, 4), rand(10, 8)
  r = experts.route(logits, 2)
  for bad in (lambda: experts.route(logits, 0), lambda: experts.route(logits, 5), lambda: experts.route(logits, 2.0),
              lambda: experts.route(logits[0], 1), lambda: experts.route(logits[:, :0], 1), lambda: experts.dispatch(x[:9], r),
              lambda: experts.combine(x, r), lambda: experts.dispatch(x[:, :0], r), lambda: experts.dispatch(x[0], r),
              lambda: experts.combine(rand(20, 8), r._replace(weights=r.weights[:5])),
              lambda: experts.dispatch(x, r._replace(position=r.position.cpu()))):
    with pytest.raises(ValueError):
      bad()
  for bad in (lambda: experts.route(logits.double(), 2), lambda: experts.dispatch(x.half(), r),
              lambda: experts.dispatch(x, r._replace(position=r.position.long()))):
    with pytest.raises(TypeError):
      bad()
  for bad in (lambda: experts.route(rand(4, 1024), 2), lambda: experts.route(rand(4, 40), 17)):
    with pytest.raises(NotImplementedError):
      bad()
  lg, xx = logits.clone().requires_grad_(), x.clone().requires_grad_()
  for f, leaf in ((lambda: experts.route(lg, 2).weights, lg), (lambda: experts.dispatch(xx, r), xx),
                  (lambda: experts.combine(experts.dispatch(xx, r), r), xx)):
    with pytest.raises(NotImplementedError):
      torch.autograd.grad(f().sum(), leaf, create_graph=True)
  from torch.autograd import forward_ad
  with forward_ad.dual_level():
    for call in (lambda: experts.route(forward_ad.make_dual(logits, logits), 2), lambda: experts.dispatch(forward_ad.make_dual(x, x), r)):
      with pytest.raises(NotImplementedError):
        call()
