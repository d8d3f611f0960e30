"""GPU: matrix products grouped by expert against their formula in 64 bits: ragged, empty and missing experts, odd sizes,
strides, both weight layouts, all gradients, what lies in rows of no expert, graphs, streams, refusals.

Tolerances. A result is rounded once to its type (finfo.eps / 2 of itself). Before that a sum of k products of bf16 values in
float32, whose running sum the tensor core may cut by a unit of its last place at each step of 16: (k / 16 + 16) 2^-23 of the
sum of the products' absolute values; the activations' slopes lie between -0.13 and 1.13, and they are good to 2^-20 of
themselves. The gradients go through the gradient of the pre-activation rounded to bf16: 2^-8 of each term more.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _randn(seed):
  g = torch.Generator(device="cuda").manual_seed(seed)
  return lambda *s: torch.randn(*s, device="cuda", generator=g)


def _offsets(sizes, start=0):
  return torch.tensor(np.concatenate(([start], start + np.cumsum(sizes))), dtype=torch.int32, device="cuda")


def _act(x, act):
  if act == "gelu":
    return torch.nn.functional.gelu(x, approximate="tanh")
  return torch.nn.functional.silu(x) if act == "swish" else x


def _close(got, want, room, label=""):
  assert got.shape == want.shape, label
  off = (got.double() - want).abs() - torch.finfo(got.dtype).eps / 2 * 1.0001 * want.abs() - room - 1e-30
  assert not (off > 0).any() and torch.isfinite(got.double()).all(), f"{label}: {off.max().item():.3e} above its bound"


def _inputs(m, e, k, n, bias, layout, seed=0):
  rand = _randn(seed + m + k)
  a = rand(m, k).to(BF16)
  w = (rand(e, n, k) * k ** -0.5).to(BF16)
  if layout == "kn":
    w = w.transpose(1, 2).contiguous().transpose(1, 2)
  return a, w, None if bias is None else (0.3 * rand(e, n)).to(bias)


def _check(sizes, k, n, act=None, bias=F32, out=BF16, layout="nk", start=0, tail=0, grads=True, a=None, w=None):
  from faster_weathernext import experts
  m, e = start + sum(sizes) + tail, len(sizes)
  a0, w0, b = _inputs(m, e, k, n, bias, layout)
  a, w = a0 if a is None else a, w0 if w is None else w
  offsets = _offsets(sizes, start)
  ins = [t for t in (a, w, b) if t is not None]
  if grads:
    for t in ins:
      t.requires_grad_()
  y = experts.linear_grouped(a, w, offsets, b, activation=act, out_dtype=out)
  assert y.dtype is out and y.shape == (m, n)
  dy = _randn(7)(m, n).to(out)
  got = torch.autograd.grad(y, ins, dy) if grads else []
  want_y, room_y = torch.zeros(m, n, dtype=torch.float64, device="cuda"), torch.zeros(m, n, dtype=torch.float64, device="cuda")
  want = [torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in ins]
  room = [torch.zeros_like(t) for t in want]
  at = start
  for i, size in enumerate(sizes):
    if size == 0:
      continue
    r = slice(at, at + size)
    at += size
    v = [a.detach()[r].double().requires_grad_(), w.detach()[i].double().requires_grad_()]
    if b is not None:
      v.append(b.detach()[i].double().requires_grad_())
    pre = v[0] @ v[1].t() + (v[2] if b is not None else 0.0)
    y64 = _act(pre, act)
    want_y[r] = y64.detach()
    terms = v[0].detach().abs() @ v[1].detach().abs().t() + (v[2].detach().abs() if b is not None else 0.0)
    cut = (k / 16 + 16) * 2.0 ** -23 * terms
    room_y[r] = 1.13 * cut + 2.0 ** -20 * y64.detach().abs() + 2e-8
    if grads:
      d_pre, = torch.autograd.grad(y64, pre, dy[r].double(), retain_graph=True)
      g = torch.autograd.grad(y64, v, dy[r].double())
      # d_pre: the slope's own error (2^-20 and 0.8 of an error of the pre-activation), then its rounding to bf16.
      d_off = dy[r].double().abs() * (2.0 ** -20 + 1.6 * cut if act else 0.0)
      d_sum = d_pre.abs() + d_off
      step = d_off + (2.0 ** -8 * d_sum if act or out is F32 else 0.0)
      want[0][r] = g[0]
      room[0][r] = step @ v[1].detach().abs() + (n / 16 + 16) * 2.0 ** -23 * (d_sum @ v[1].detach().abs())
      want[1][i] = g[1]
      room[1][i] = step.t() @ v[0].detach().abs() + (size / 16 + 64) * 2.0 ** -23 * (d_sum.t() @ v[0].detach().abs())
      if b is not None:
        want[2][i] = g[2]
        room[2][i] = d_off.sum(0) + (size / 32 + 64) * 2.0 ** -23 * d_sum.sum(0)
  _close(y.detach(), want_y, room_y, "y")
  for name, t, g, x, o in zip(("a", "weight", "bias"), ins, got, want, room):
    assert g.dtype is t.dtype
    _close(g, x, o, "d_" + name)
  from faster_weathernext import _lib
  torch.cuda.synchronize()
  assert _lib.device_error() == 0
  return y.detach(), got


FORMS = [
    # sizes, k, n, activation, bias, out, layout, rows before and behind
    ([300, 200, 524], 256, 256, None, None, BF16, "nk", 0, 0),
    ([300, 0, 200, 13], 64, 128, "gelu", F32, BF16, "nk", 0, 0),
    ([1, 2, 3, 0, 700, 5], 512, 520, "swish", BF16, BF16, "kn", 0, 0),
    ([0, 0, 40, 0], 200, 72, "gelu", F32, F32, "nk", 0, 0),
    ([129, 127, 128, 256, 257], 1001, 515, "swish", F32, BF16, "nk", 3, 60),
    ([33, 500], 1000, 513, "gelu", BF16, F32, "kn", 17, 5),
    ([1000], 320, 2048, "gelu", F32, BF16, "nk", 0, 1),
    ([2000, 3000, 100], 512, 1024, None, F32, BF16, "kn", 0, 0),
    ([2000, 3000, 100], 2048, 512, None, F32, F32, "nk", 0, 0),
    ([700] * 16, 128, 256, "swish", None, F32, "nk", 0, 0),
    ([5, 0, 9, 1] * 16, 96, 200, "gelu", F32, BF16, "nk", 2, 3),
    ([64], 1, 1, "gelu", F32, BF16, "nk", 0, 0),
    ([70, 3], 7, 9, None, BF16, BF16, "kn", 1, 1),
    ([4, 1], 512, 300, "gelu", F32, BF16, "nk", 0, 0),           # few rows
    ([0, 3, 0, 2], 100, 77, "swish", BF16, F32, "nk", 1, 2),
    ([2, 2], 264, 64, "gelu", F32, BF16, "kn", 0, 0),
    ([1], 2048, 512, None, F32, F32, "nk", 0, 0),
    ([0, 0, 0], 64, 64, "gelu", F32, BF16, "nk", 0, 9),          # no expert has a row
    ([0, 0, 0], 64, 64, "gelu", F32, BF16, "nk", 2, 3),
]


@pytest.mark.parametrize("form", FORMS, ids=lambda f: f"{sum(f[0])}of{len(f[0])}-{f[1]}x{f[2]}-{f[3]}-{f[6]}")
def test_values_and_gradients(cuda, form):
  sizes, k, n, act, bias, out, layout, start, tail = form
  _check(sizes, k, n, act, bias, out, layout, start, tail)


@pytest.mark.parametrize("form", FORMS, ids=lambda f: f"{sum(f[0])}of{len(f[0])}-{f[1]}x{f[2]}-{f[3]}-{f[6]}")
def test_values_without_gradients(cuda, form):
  sizes, k, n, act, bias, out, layout, start, tail = form
  _check(sizes, k, n, act, bias, out, layout, start, tail, grads=False)


def test_large_ragged(cuda):
  """Every tile form of the forward and of the gradients at sizes that fill the SMs, several tiles a block."""
  _check([9000, 1, 20000, 0, 7777, 128], 512, 2048, "gelu", F32, BF16, "kn")
  _check([15000, 30000], 2048, 512, None, F32, F32, "nk")


def test_many_experts(cuda):
  rng = np.random.default_rng(0)
  sizes = rng.integers(0, 9, 1023).tolist()
  _check(sizes, 64, 72, "swish", F32, BF16, "nk", 0, 4)


def test_one_expert_is_linear(cuda):
  """One expert of all rows gives projection.linear's result, whose kernel it is."""
  from faster_weathernext import experts, projection
  a, w, b = _inputs(5000, 1, 512, 768, F32, "nk")
  y = experts.linear_grouped(a, w, _offsets([5000]), b, activation="gelu")
  assert torch.equal(y, projection.linear(a, w[0], b[0], activation="gelu"))


def test_weight_views(cuda):
  """Experts apart by any stride, and weights that TMA cannot address."""
  rand = _randn(3)
  sizes = [100, 30, 270]
  pool = (rand(3, 2, 64, 128) * 0.1).to(BF16)
  _check(sizes, 128, 64, "gelu", w=pool[:, 1].detach())
  inter = (rand(64, 3, 128) * 0.1).to(BF16)
  _check(sizes, 128, 64, "gelu", w=inter.transpose(0, 1).detach())
  cut = (rand(3, 64, 140) * 0.1).to(BF16)
  _check(sizes, 128, 64, None, w=cut[:, :, 5:133].detach())
  wide = rand(400, 300).to(BF16)
  _check(sizes, 128, 64, "swish", a=wide[:, 11:139].detach())
  _check(sizes, 128, 64, "swish", a=rand(128, 400).to(BF16).t().detach())


def test_rows_of_no_expert_are_not_read(cuda):
  """Whatever lies before the first expert's rows and behind the last one's (NaN here) reaches nothing, and gives zeros."""
  from faster_weathernext import experts
  sizes, start, tail = [100, 0, 37, 200], 5, 50
  m = start + sum(sizes) + tail
  for k, n, layout, out in ((128, 256, "nk", BF16), (77, 45, "kn", F32)):
    a, w, b = _inputs(m, 4, k, n, F32, layout)
    dy = _randn(2)(m, n).to(out)
    offsets = _offsets(sizes, start)
    outside = torch.ones(m, dtype=torch.bool, device="cuda")
    outside[start:m - tail] = False

    def run(fill, a=a, w=w, b=b, dy=dy, offsets=offsets, outside=outside, out=out):
      a2, dy2 = a.clone(), dy.clone()
      a2[outside], dy2[outside] = fill, fill
      ins = [t.detach().requires_grad_() for t in (a2, w, b)]
      y = experts.linear_grouped(ins[0], ins[1], offsets, ins[2], activation="gelu", out_dtype=out)
      return [y.detach(), *torch.autograd.grad(y, ins, dy2)]

    for x, z in zip(run(float("nan")), run(0.0)):
      assert torch.equal(x, z)
    assert (run(1.0)[0][outside] == 0).all() and (run(1.0)[1][outside] == 0).all()


def test_nan_stays_with_its_expert(cuda):
  from faster_weathernext import experts
  sizes = [70, 130, 64]
  a, w, b = _inputs(264, 3, 96, 160, F32, "nk")
  a[80, 3] = float("nan")
  ins = [t.requires_grad_() for t in (a, w, b)]
  y = experts.linear_grouped(*ins[:2], _offsets(sizes), b, activation="swish")
  d_a, d_w, d_b = torch.autograd.grad(y, ins, torch.ones_like(y))
  keep = [i for i in range(264) if i != 80]
  assert torch.isnan(y[80]).all() and torch.isfinite(y[keep]).all() and torch.isfinite(d_a[keep]).all()
  assert torch.isfinite(d_w[[0, 2]]).all() and torch.isfinite(d_b[[0, 2]]).all() and torch.isnan(d_b[1]).all()


def test_infinite_preactivations(cuda):
  from faster_weathernext import experts
  b = torch.tensor([[float("-inf"), float("inf"), 0.0, 1.0] * 2], device="cuda")
  for m in (2, 40):
    a, w, _ = _inputs(m, 1, 16, 8, None, "nk")
    for act in ("gelu", "swish"):
      y = experts.linear_grouped(a, w, _offsets([m]), b, activation=act)
      assert (y[:, 0].abs() <= 2e-8).all() and torch.isinf(y[:, 1]).all() and torch.isfinite(y[:, 2:4]).all()


def test_empty_inputs(cuda):
  from faster_weathernext import experts
  a, w, b = _inputs(0, 3, 64, 32, F32, "kn")
  ins = [t.requires_grad_() for t in (a, w, b)]
  y = experts.linear_grouped(a, w, _offsets([0, 0, 0]), b)
  assert y.shape == (0, 32)
  d_a, d_w, d_b = torch.autograd.grad(y, ins, torch.zeros_like(y))
  assert d_a.shape == (0, 64) and (d_w == 0).all() and (d_b == 0).all() and d_w.shape == w.shape


def test_partial_gradients(cuda):
  from faster_weathernext import experts
  full = {}
  for need in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1)):
    a, w, b = _inputs(300, 3, 128, 64, F32, "nk")
    ins = (a, w, b)
    for t, f in zip(ins, need):
      t.requires_grad_(bool(f))
    for act in ("gelu", None):
      y = experts.linear_grouped(a, w, _offsets([100, 150, 50]), b, activation=act)
      got = torch.autograd.grad(y, [t for t, f in zip(ins, need) if f], torch.ones_like(y))
      if sum(need) == 3:
        full[act] = got
      else:
        assert torch.equal(got[0], full[act][need.index(1)])


def test_offsets_out_of_order_are_reported(cuda):
  """Offsets that decrease or leave the tensor are brought into order; the call's memory stays its own."""
  from faster_weathernext import _lib, experts
  a, w, b = _inputs(200, 3, 64, 64, F32, "nk")
  want = experts.linear_grouped(a, w, _offsets([90, 0, 110]), b)
  bad = torch.tensor([0, 90, 40, 5000], dtype=torch.int32, device="cuda")
  got = experts.linear_grouped(a, w, bad, b)
  torch.cuda.synchronize()
  assert _lib.device_error() == _lib.FWN_ERR_INVALID_ARGUMENT and _lib.device_error() == 0
  assert torch.equal(got, want)
  experts.linear_grouped(a[:4], w, torch.tensor([0, 3, 1, 4], dtype=torch.int32, device="cuda"), b)
  assert _lib.device_error() == _lib.FWN_ERR_INVALID_ARGUMENT
  experts.linear_grouped(a[:4], w, torch.tensor([-3, 0, 1, 4], dtype=torch.int32, device="cuda"), b)
  assert _lib.device_error() == _lib.FWN_ERR_INVALID_ARGUMENT


def test_graph_takes_new_offsets(cuda):
  """A captured training step replayed with other rows, sizes and weights gives what an eager step gives."""
  from faster_weathernext import experts
  a, w, b = _inputs(1000, 4, 256, 320, F32, "kn")
  offsets = _offsets([400, 100, 0, 500])
  ins = [t.requires_grad_() for t in (a, w, b)]
  dy = torch.ones(1000, 320, device="cuda", dtype=BF16)

  def step():
    y = experts.linear_grouped(a, w, offsets, b, activation="gelu")
    return [y.detach(), *torch.autograd.grad(y, ins, dy)]

  step()
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = step()
  for sizes in ([400, 100, 0, 500], [0, 1, 999, 0], [250, 250, 250, 200]):
    with torch.no_grad():
      offsets.copy_(_offsets(sizes))
      a.mul_(1.01)
    graph.replay()
    assert all(torch.equal(x, y) for x, y in zip(out, step()))


@pytest.mark.parametrize("m,e,n,k", [(20000, 2, 64, 96), (3000, 40, 72, 64)])
def test_c_entry_with_results_that_start_anywhere(cuda, m, e, n, k):
  """Results at addresses of whole elements alone (the first shape sums its weights' gradient in runs, the second at once)."""
  from faster_weathernext import _lib, experts
  lib = _lib.lib()
  a, w, b = _inputs(m, e, k, n, F32, "nk")
  offsets = _offsets([m // e] * e)
  dy = _randn(1)(m, n).to(BF16)
  ins = [t.requires_grad_() for t in (a, w, b)]
  y = experts.linear_grouped(a, w, offsets, b, activation="gelu")
  want = [y.detach(), *torch.autograd.grad(y, ins, dy)]
  pool = [torch.zeros(t.numel() + 8, device="cuda", dtype=t.dtype) for t in want]
  got = [p[1:1 + t.numel()].view(t.shape) for p, t in zip(pool, want)]
  desc = _lib.GroupedDesc(m, e, n, k, 0, 1, 0, _lib.ACT_GELU_TANH, 0, k, k, n * k, n)
  stream = torch.cuda.current_stream().cuda_stream
  import ctypes
  size = ctypes.c_size_t(0)
  _lib.check(lib.fwn_linear_grouped_workspace_size(desc, size))
  ws = torch.empty(size.value, dtype=torch.uint8, device="cuda")
  _lib.check(lib.fwn_linear_grouped(desc, a.data_ptr(), w.data_ptr(), b.data_ptr(), offsets.data_ptr(), got[0].data_ptr(),
                                    ws.data_ptr(), size.value, stream))
  _lib.check(lib.fwn_linear_grouped_bwd_workspace_size(desc, dy.data_ptr(), size))
  ws = torch.empty(size.value, dtype=torch.uint8, device="cuda")
  _lib.check(lib.fwn_linear_grouped_bwd(desc, a.data_ptr(), w.data_ptr(), b.data_ptr(), offsets.data_ptr(), dy.data_ptr(),
                                        got[1].data_ptr(), got[2].data_ptr(), got[3].data_ptr(), ws.data_ptr(), size.value, stream))
  for g, t, p in zip(got, want, pool):
    assert (g.float() - t.float()).abs().max() <= 2.0 ** -7 * t.float().abs().max()   # other tiles: a step of the type
    assert p[0] == 0 and (p[1 + t.numel():] == 0).all()


def test_streams_and_repeats(cuda):
  from faster_weathernext import experts
  a, w, b = _inputs(3000, 8, 512, 512, F32, "nk")
  offsets = _offsets([375] * 8)
  ins = [t.requires_grad_() for t in (a, w, b)]

  def step():
    y = experts.linear_grouped(a, w, offsets, b, activation="swish")
    return [y.detach(), *torch.autograd.grad(y, ins, torch.ones_like(y))]

  want = step()
  torch.cuda.synchronize()
  streams = [torch.cuda.Stream() for _ in range(2)]
  got = []
  for s in streams * 3:
    with torch.cuda.stream(s):
      got.append(step())
  torch.cuda.synchronize()
  assert all(torch.equal(x, y) for g in got for x, y in zip(g, want))


def test_gradient_against_differences(cuda):
  """The float32 result, moved along a direction that bf16 holds exactly."""
  from faster_weathernext import experts
  a, w, b = _inputs(60, 3, 64, 48, F32, "nk")
  a, w = a.float().sign().mul_(0.5).to(BF16), (w.float().sign() * 0.0625).to(BF16)
  offsets = _offsets([25, 5, 30])
  weight_of = _randn(5)(60, 48)
  value = lambda *v: (experts.linear_grouped(v[0], v[1], offsets, v[2], activation="gelu", out_dtype=F32).double() * weight_of).sum()  # noqa: E731
  ins = [t.requires_grad_() for t in (a, w, b)]
  grads = torch.autograd.grad(value(*ins), ins)
  rand = _randn(6)
  for i, (t, g) in enumerate(zip(ins, grads)):
    direction = rand(*t.shape).sign() * (2.0 ** -6 if i == 0 else 2.0 ** -9 if i == 1 else 2.0 ** -6)
    at = lambda f: [(x.detach().double() + f * direction.double()).to(x.dtype) if i == j else x.detach() for j, x in enumerate(ins)]  # noqa: E731, B023
    slope = (8 * (value(*at(1)) - value(*at(-1))) - (value(*at(2)) - value(*at(-2)))) / 12
    want = (g.double() * direction).sum()
    assert abs(slope - want) <= 6e-3 * g.double().norm() * direction.double().norm(), i


def test_refusals(cuda):
  from faster_weathernext import experts
  a, w, b = _inputs(20, 2, 64, 32, F32, "nk")
  o = _offsets([10, 10])
  call = experts.linear_grouped
  for bad in (lambda: call(a[0], w, o), lambda: call(a, w[0], o), lambda: call(a[:, :63], w, o), lambda: call(a, w, o[:2]),
              lambda: call(a, w, o, b[:1]), lambda: call(a, w, o, b, activation="relu"), lambda: call(a, w, o, out_dtype=torch.half),
              lambda: call(a, w, o.cpu()), lambda: call(a, w[:, :0], o)):
    with pytest.raises(ValueError):
      bad()
  for bad in (lambda: call(a.float(), w, o), lambda: call(a, w.float(), o), lambda: call(a, w, o.long()), lambda: call(a, w, o, b.half())):
    with pytest.raises(TypeError):
      bad()
  with pytest.raises(NotImplementedError):
    call(a, w[:1].expand(1024, 32, 64), torch.zeros(1025, dtype=torch.int32, device="cuda"))
  x = a.clone().requires_grad_()
  with pytest.raises(NotImplementedError):
    torch.autograd.grad(call(x, w, o).float().sum(), x, create_graph=True)
  from torch.autograd import forward_ad
  with forward_ad.dual_level(), pytest.raises(NotImplementedError):
    call(forward_ad.make_dual(a, torch.ones_like(a)), w, o)
