"""The gradient of the residual branch at every width against bounds that no wrong gradient meets: on the CPU, that a gradient
without one of its means, of zeros or negated is out of them; on the GPU, that the kernels' are within."""
import pytest
import torch

import branch_terms
from test_branch_gpu import CASES

F32, BF16 = torch.float32, torch.bfloat16
# x, y, gate, weights, h, residual scale, dropout: the sizes of the values' test, each of its gradients of a size to be wrong in,
# and wide rows more.
WIDE = [
    ((7, 2048), F32, F32, "value", F32, F32, 1.0, 0.0),
    ((7, 4096), BF16, BF16, "value", F32, BF16, 1.0, 0.1),
    ((3, 4, 8192), F32, F32, "sample", F32, F32, 1.0, 0.1),
    ((5, 8185), BF16, BF16, "value", BF16, F32, 1.0, 0.0),
    ((6, 3001), F32, F32, "channel", F32, F32, -0.5, 0.0),
    ((1300, 1152), F32, BF16, "channel", F32, BF16, 1.0, 0.1),   # several rows a block
    ((9000, 72), F32, F32, "channel", F32, F32, 1.0, 0.1),
    ((3000, 333), F32, F32, "channel", F32, F32, 1.0, 0.1),
]
SHAPES = [c[:6] + (c[6] or 0.5,) + c[7:] for c in CASES] + WIDE
ids = lambda c: "x".join(map(str, c[0])) + f"-{c[3]}-{c[7]}"  # noqa: E731


def _setup(case, device):
  shape, xd, yd, gate, wd, od, alpha, p = case
  ins, grads = branch_terms.inputs(shape, xd, yd, gate, wd, od, device)
  return ins, grads, alpha, branch_terms.mask_of(shape, p, 42, 2, device) if p else None


@pytest.mark.parametrize("case", SHAPES, ids=ids)
def test_wrong_gradients_are_out_of_bounds(case):
  ins, (dh, ds), alpha, mask = _setup(case, "cpu")
  given = dict(zip(("x", "y", "post_weight", "weight", "gate"), ins))
  right = branch_terms.gradients(ins, dh, ds, alpha, mask=mask)
  out = lambda name, v: branch_terms.excess(v.to(given[name].dtype), *right[name]) > 0  # noqa: E731
  for name, (v, _) in right.items():
    assert not out(name, v), name
    assert out(name, torch.zeros_like(v)) and out(name, -v), name
  for term, name in (("c1", "x"), ("c2", "y")):
    assert out(name, branch_terms.gradients(ins, dh, ds, alpha, mask=mask, without=(term,))[name][0]), term


def test_terms_are_the_formula():
  """The terms add up to what torch differentiates."""
  ins, (dh, ds) = branch_terms.inputs((2, 5, 24), F32, F32, "sample", F32, F32, "cpu")
  mask = branch_terms.mask_of((2, 5, 24), 0.2, 3, 0, "cpu")
  x, y, pw, w, gate = v = [t.double().requires_grad_() for t in ins]
  norm = lambda t: t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6)  # noqa: E731
  s = 0.75 * x + norm(y) * pw * gate.unsqueeze(-2) * mask
  want = torch.autograd.grad((norm(s) * w, s), v, (dh.double(), ds.double()))
  got = branch_terms.gradients(ins, dh, ds, 0.75, mask=mask)
  for name, t in zip(("x", "y", "post_weight", "weight", "gate"), want):
    assert (got[name][0] - t).abs().max() <= 1e-12 * t.abs().max(), name


@pytest.mark.gpu
@pytest.mark.parametrize("case", SHAPES, ids=ids)
def test_gradients(cuda, case):
  from faster_weathernext import branch
  ins, (dh, ds), alpha, mask = _setup(case, cuda)
  given = {k: t.requires_grad_() for k, t in zip(("x", "y", "post_weight", "weight", "gate"), ins) if t is not None}
  h, s = branch.branch_norm(*ins[:4], gate=ins[4], residual_scale=alpha, p=case[7], seed=42 if case[7] else None, site=2,
                            out_dtype=case[5])
  for a, b in ((dh, ds), (dh, None), (None, ds)):
    got = torch.autograd.grad([t for t, u in ((h, a), (s, b)) if u is not None], list(given.values()),
                              [u for u in (a, b) if u is not None], retain_graph=True)
    want = branch_terms.gradients(ins, a, b, alpha, mask=mask)
    for name, g in zip(given, got):
      assert branch_terms.excess(g, *want[name]) <= 0, (name, a is None, b is None)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [1001, 2048, 8185])
@pytest.mark.parametrize("gate", ["channel", "value"])
def test_wide_gradients_against_differences(cuda, d, gate):
  """The kernels' own forward, moved along a random direction and along each input itself. Along y the row's norm takes no part
  of the step, along x the next norm takes part of it: there a gradient without a mean is off by c d a row, c the mean, of order
  one here. Fourth-order differences of a step of 1e-2: 1e-8 of the fifth derivative, and float32's noise, 2^-20 of values of
  order one over the step: 1e-4 each, where they add up: 1e-3 of the two norms' product holds both."""
  from faster_weathernext import branch
  ins, (a, b) = branch_terms.inputs((3, d), F32, F32, gate, F32, F32, cuda)
  leaves = [t.requires_grad_() for t in ins]

  def value(v):
    h, s = branch.branch_norm(*v[:4], gate=v[4], residual_scale=0.8, p=0.2, seed=6, out_dtype=F32)
    return (h.double() * a).sum() + (s.double() * b).sum()

  grads = torch.autograd.grad(value(leaves), leaves)
  gen = torch.Generator(device="cuda").manual_seed(d)
  step = 1e-2
  for i, g in enumerate(grads):
    for direction in (torch.randn(g.shape, device="cuda", generator=gen), leaves[i].detach()):
      moved = lambda f: [t.detach() + f * step * direction if i == j else t.detach() for j, t in enumerate(leaves)]  # noqa: E731, B023
      slope = (8 * (value(moved(1)) - value(moved(-1))) - (value(moved(2)) - value(moved(-2)))) / (12 * step)
      want = (g.double() * direction).sum()
      assert abs(slope - want) <= 1e-3 * g.double().norm() * direction.double().norm(), (i, slope.item(), want.item())
