"""GPU: forms of the pre-norm projections' kernels that take sizes of their own, against plain float64 torch, and the calls
as a program makes them: captured in CUDA graphs, from two threads, on a middle mesh. Bounds as test_projection_gpu.py's
and test_rms_processor_gpu.py's."""
import threading

import pytest
import torch

import test_projection_gpu as base
import test_rms_processor_gpu as processor_base
from test_projection_gpu import BF, F32, TOL, TOL_GRAD, _check, _gen, _no_device_error, _pr, _problem, _rel, _rms64

pytestmark = pytest.mark.gpu


# ---- rms_norm -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,d", [(33, 640), (9, 768), (17, 1280), (301, 1536), (9, 2560), (70, 2944)])
@pytest.mark.parametrize("x_dtype,r_dtype,w_dtype", [(F32, BF, F32), (BF, BF, BF), (BF, F32, F32), (F32, None, None),
                                                     (BF, None, F32)])
def test_rms_norm_forward_at_three_groups_a_thread(cuda, rows, d, x_dtype, r_dtype, w_dtype):
  base.test_rms_norm_forward(cuda, rows, d, x_dtype, r_dtype, w_dtype)


@pytest.mark.parametrize("rows,d", [(40, 600), (301, 600), (33, 2500), (9, 9001), (3, 16383)])
@pytest.mark.parametrize("x_dtype,r_dtype,out", [(F32, BF, BF), (BF, BF, F32), (BF, None, BF), (F32, F32, F32)])
def test_rms_norm_gradients_of_views(cuda, rows, d, x_dtype, r_dtype, out):
  """x and the residual as columns of wider tensors whose rows start anywhere."""
  pr, g = _pr(), _gen(rows + d)
  wide = (torch.randn(rows, d + 7, device=cuda, generator=g) * 2).to(x_dtype).requires_grad_()
  r_wide = None if r_dtype is None else torch.randn(rows, d + 3, device=cuda, generator=g).to(r_dtype).requires_grad_()
  w = (1 + 0.2 * torch.randn(d, device=cuda, generator=g)).requires_grad_()
  dh = torch.randn(rows, d, device=cuda, generator=g).to(out)
  ds = torch.randn(rows, d, device=cuda, generator=g).to(x_dtype)
  ins = [t for t in (wide, w, r_wide) if t is not None]

  def run(norm, x, w, r):
    got = norm(x[:, 1:d + 1], w, None if r is None else r[:, 2:d + 2])
    return (got,) if r is None else got

  seeds = (dh,) if r_dtype is None else (dh, ds)
  grads = torch.autograd.grad(run(lambda x, w, r: pr.rms_norm(x, w, r, out_dtype=out), wide, w, r_wide), ins, seeds)
  ref = [t.detach().double().requires_grad_() for t in ins]
  outs = run(lambda x, w, r: _rms64(x, w, r, 1e-6)[:1 if r is None else 2], ref[0], ref[1],
             ref[2] if r_dtype is not None else None)
  want = torch.autograd.grad(outs[0] if r_dtype is None else outs, ref, [s.double() for s in seeds])
  for t, a, c in zip(ins, grads, want):
    assert a.dtype == t.dtype
    if t.dtype == BF:
      _check(a, c, TOL[BF])
    else:
      assert _rel(a, c) <= TOL_GRAD[F32]


# ---- linear ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("m,k,n", [(9001, 1024, 1000), (4000, 1024, 1024), (9001, 1280, 1000), (9001, 2048, 512)])
@pytest.mark.parametrize("act", ["gelu", "swish"])
@pytest.mark.parametrize("bias,out", [(F32, BF), (F32, F32), (BF, BF), (BF, F32)])
def test_linear_gradients_of_wide_layers(cuda, m, k, n, act, bias, out):
  """Many rows at widths of 1,024 to 2,048: the gradient of the pre-activation on pairs of SMs, with k added in chunks
  (float32 bias) and at once (bf16 bias), in its forms for short and for long k."""
  base.test_linear_gradients(cuda, m, k, n, "nk", act, bias, False, out)


# ---- as a program makes the calls -----------------------------------------------------------------------------------

def _captured(call):
  """(graph, outputs) of call, captured after runs on a side stream."""
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    for _ in range(2):
      call()
  torch.cuda.current_stream().wait_stream(side)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    outs = call()
  return graph, outs


@pytest.mark.parametrize("m", [1, 42, 3000])
def test_forecast_calls_in_a_cuda_graph(cuda, m):
  """All five functions in one graph: new inputs in the same tensors, replayed, give the bits of plain calls."""
  pr = _pr()
  a, w, b, r = _problem(m, 515, 512, m)
  x, wn = torch.randn(m, 515, device=cuda, generator=_gen(1)), torch.ones(515, device=cuda)

  def call():
    h, s = pr.rms_norm(x, wn, a)
    y = pr.linear(h, w, b, r.to(BF), activation="gelu")
    v, sc, s8 = pr.rms_norm_fp8(x, wn, a)
    w8, sw = pr.quantize_fp8(w)
    return h, s, y, v.float(), sc, s8, pr.linear_fp8(v, sc, w8, sw, b, r, activation="swish", out_dtype=F32)

  graph, outs = _captured(call)
  for seed in (2, 3):
    x.copy_(torch.randn(m, 515, device=cuda, generator=_gen(seed)))
    r.copy_(torch.randn(m, 512, device=cuda, generator=_gen(seed + 9)))
    graph.replay()
    got = [t.clone() for t in outs]
    for p, q in zip(got, call()):
      assert torch.equal(p, q)
  _no_device_error()


@pytest.mark.parametrize("m,k,n", [(42, 512, 512), (2562, 515, 333)])
def test_a_training_step_in_a_cuda_graph(cuda, m, k, n):
  pr = _pr()
  a, w, b, _ = _problem(m, k, n, m)
  x, wn = torch.randn(m, k, device=cuda, generator=_gen(1)), torch.ones(k, device=cuda)
  dy = torch.randn(m, n, device=cuda, generator=_gen(2)).to(BF)
  ins = [t.requires_grad_() for t in (x, wn, w, b)]

  def call():
    h, s = pr.rms_norm(x, wn, a)
    y = pr.linear(h, w, b, activation="gelu")
    return (y, *torch.autograd.grad((y, s), ins, (dy, s.detach())))

  graph, outs = _captured(call)
  with torch.no_grad():
    x.copy_(torch.randn(m, k, device=cuda, generator=_gen(3)))
    dy.copy_(torch.randn(m, n, device=cuda, generator=_gen(4)))
  graph.replay()
  got = [t.detach().clone() for t in outs]
  for p, q in zip(got, call()):
    assert torch.equal(p, q.detach())
  _no_device_error()


def test_calls_from_two_threads(cuda):
  """Each thread with its own stream and shapes: the bits of calls made one after another."""
  pr = _pr()
  problems = [_problem(700, 515, 333, 1), _problem(3000, 512, 1024, 2)]

  def step(problem):
    a, w, b, _ = problem
    ins = [t.detach().clone().requires_grad_() for t in (a, w, b)]
    y = pr.linear(*ins, activation="gelu")
    h = pr.rms_norm(y, torch.ones(y.shape[1], device=cuda))
    return [y.detach(), *torch.autograd.grad(h, ins, torch.ones_like(h))]

  want, wrong = [step(p) for p in problems], []
  torch.cuda.synchronize()

  def work(i):
    try:
      with torch.cuda.stream(torch.cuda.Stream()):
        for _ in range(10):
          got = step(problems[i])
          torch.cuda.current_stream().synchronize()
          if not all(torch.equal(p, q) for p, q in zip(got, want[i])):
            wrong.append(i)
    except Exception as e:  # a thread's own exception would pass unseen
      wrong.append(e)

  threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
  for t in threads:
    t.start()
  for t in threads:
    t.join()
  assert not wrong
  _no_device_error()


def test_rms_processor_on_a_middle_mesh(cuda):
  """2,562 nodes (two members: 5,124 rows), training and forecasts against plain torch."""
  from faster_weathernext import mesh
  from faster_weathernext import tiled_attn as ta
  from faster_weathernext.rms_processor import RmsProcessor
  xyz, _ = mesh.icosphere(4)
  lat, lon = mesh.latlon(xyz)
  m = mesh.permute(mesh.great_circle_mask(xyz, 0.15), mesh.morton_order(lat, lon))
  model = RmsProcessor(processor_base._cfg(d_model=256, heads=4, mlp_hidden=1024), seed=3, device=cuda)
  x = torch.randn(2, m.shape[0], 256, device=cuda, generator=_gen(5))
  tiles, mask = ta.AttentionTiles.from_mask(m, device=cuda), torch.from_numpy(m.toarray()).to(cuda)
  y = model(x, tiles)
  t = torch.randn_like(x)
  grads = torch.autograd.grad(torch.nn.functional.mse_loss(y, t), list(model.parameters()))
  want = processor_base._plain(model, x, mask)
  ref = torch.autograd.grad(torch.nn.functional.mse_loss(want, t), list(model.parameters()))
  assert processor_base._rel(y.detach(), want.detach()) < 2e-2
  grads, ref = (torch.cat([v.reshape(-1) for v in s]) for s in (grads, ref))
  assert float((grads - ref).norm() / ref.norm()) < 5e-2
  assert processor_base._rel(model.forecast(x, tiles, model.forecast_plan(eight_bit=False)), want.detach()) < 2e-2
  assert processor_base._rel(model.forecast(x, tiles, model.forecast_plan()), want.detach()) < 1e-1
