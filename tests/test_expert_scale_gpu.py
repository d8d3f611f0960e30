"""GPU: the branches, the products grouped by expert and the routing where a tensor has more than 2^31 values, and from two
threads at once. The last rows of the large tensors have to be what the same calls give for those rows alone."""
import threading

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _large(rows, d, seed):
  """rows x d bf16 values, the last 64 rows random, the others a small pattern."""
  g = torch.Generator(device="cuda").manual_seed(seed)
  t = torch.empty(rows, d, device="cuda", dtype=BF16)
  t[:] = torch.randn(1, d, device="cuda", generator=g)
  t[-64:] = torch.randn(64, d, device="cuda", generator=g)
  return t


@pytest.mark.parametrize("d", [2048, 2047])
def test_branches_past_32_bits(cuda, d):
  from faster_weathernext import branch
  from oracle import dropout
  rows = 2 ** 31 // d + 1000
  x, y = _large(rows, d, 1), _large(rows, d, 2)
  first = (rows - 64) * d
  lead = first % 8
  m = torch.from_numpy(dropout.factors((64 * d + lead,), 0.25, 9, 1, first=first - lead)[lead:].reshape(64, d)).cuda()
  z = branch.dropout(x, 0.25, 9, site=1)
  assert torch.equal(z[-64:], (x[-64:].double() * m).to(BF16))
  del z
  h, s = branch.branch_norm(x, y)
  want = branch.branch_norm(x[-64:].clone(), y[-64:].clone())
  assert torch.equal(h[-64:], want[0]) and torch.equal(s[-64:], want[1])
  del h, s
  x.requires_grad_()
  h, s = branch.branch_norm(x, y)
  dh = y
  d_x, = torch.autograd.grad(h, x, dh)
  tail = x.detach()[-64:].clone().requires_grad_()
  want, = torch.autograd.grad(branch.branch_norm(tail, y[-64:].clone())[0], tail, dh[-64:].clone())
  assert torch.equal(d_x[-64:], want)


def test_grouped_past_32_bits(cuda):
  from faster_weathernext import experts
  k, n, m = 1024, 64, 2 ** 31 // 1024 + 5000
  a = _large(m, k, 3)
  g = torch.Generator(device="cuda").manual_seed(4)
  w = (torch.randn(3, n, k, device="cuda", generator=g) * k ** -0.5).to(BF16)
  offsets = torch.tensor([0, 1000, m - 64, m], dtype=torch.int32, device="cuda")
  a.requires_grad_()
  y = experts.linear_grouped(a, w, offsets, activation="gelu")
  d_a, = torch.autograd.grad(y, a, torch.ones_like(y))
  tail = a.detach()[-64:].clone().requires_grad_()
  one = torch.tensor([0, 64], dtype=torch.int32, device="cuda")
  want = experts.linear_grouped(tail, w[2:], one, activation="gelu")
  want_a, = torch.autograd.grad(want, tail, torch.ones_like(want))
  # Another tile's form may add k in another order: a step of the result's type, rarely.
  assert (y[-64:].float() - want.float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()
  assert (d_a[-64:].float() - want_a.float()).abs().max() <= 2.0 ** -6 * want_a.float().abs().max()


def test_routing_past_32_bits(cuda):
  from faster_weathernext import experts
  d, rows = 2048, 2 ** 30 // 2048 + 3000
  x = _large(rows, d, 5)
  logits = torch.randn(rows, 4, device="cuda", generator=torch.Generator(device="cuda").manual_seed(6))
  r = experts.route(logits, 2)
  moved = experts.dispatch(x, r)
  assert moved.numel() > 2 ** 31
  places = r.position[-64:].long().reshape(-1)
  assert torch.equal(moved[places], x[-64:].repeat_interleave(2, 0))
  assert torch.equal(moved[-8:], x[(r.order[-8:] // 2).long()])
  back = experts.combine(moved, r)
  want = (x[-64:].double()[:, None] * r.weights[-64:].double()[:, :, None]).sum(1)
  assert ((back[-64:].double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-6).all()


def test_two_threads(cuda):
  """Each on a stream of its own, captured sizes of workspaces and all: what one thread alone gives."""
  from faster_weathernext import branch, experts

  def step(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    logits, x = rand(700 + seed, 8).requires_grad_(), rand(700 + seed, 256).to(BF16).requires_grad_()
    w, stream = (rand(8, 256, 256) / 16).to(BF16).requires_grad_(), rand(700 + seed, 256).requires_grad_()
    r = experts.route(logits, 2)
    y = experts.combine(experts.linear_grouped(experts.dispatch(x, r), w, r.offsets, activation="swish"), r)
    h, s = branch.branch_norm(stream, y, p=0.1, seed=seed)
    return [h.detach(), s.detach(), *torch.autograd.grad((h, s), (logits, x, w, stream), (torch.ones_like(h), torch.ones_like(s)))]

  want = {seed: step(seed) for seed in (1, 2)}
  torch.cuda.synchronize()
  got, errors = {1: [], 2: []}, []

  def work(seed):
    try:
      with torch.cuda.stream(torch.cuda.Stream()):
        for _ in range(10):
          got[seed].append(step(seed))
    except Exception as e:  # noqa: BLE001
      errors.append(e)

  threads = [threading.Thread(target=work, args=(seed,)) for seed in (1, 2)]
  for t in threads:
    t.start()
  for t in threads:
    t.join()
  torch.cuda.synchronize()
  assert not errors
  assert all(torch.equal(a, b) for seed in (1, 2) for run in got[seed] for a, b in zip(run, want[seed]))
  assert np.isfinite(float(got[1][0][0].float().sum()))
