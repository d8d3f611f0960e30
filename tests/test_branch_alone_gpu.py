"""GPU: the gradient of a residual branch's stream alone. It does not depend on the stream's values (s = residual_scale x +
branch, and h is not used): whatever x holds, in rows whose gradient is zero also what is not a number."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("xd", [F32, BF16])
@pytest.mark.parametrize("d,gate", [(64, "sample"), (100, "value"), (333, "channel"), (512, "value"), (1001, "sample"), (2048, "sample")])
def test_gradients_do_not_depend_on_the_stream(cuda, d, gate, xd):
  from faster_weathernext import branch
  gen = torch.Generator(device="cuda").manual_seed(d)
  r = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
  x, y, pw, w, ds = r(2, 40, d).to(xd), r(2, 40, d).to(BF16), r(d), r(d), r(2, 40, d).to(xd)
  g = r(*{"channel": (d,), "sample": (2, d), "value": (2, 40, d)}[gate])
  ds[1, 30:] = 0.0  # rows that are padding
  odd = x.clone()
  odd[0, 3] = 0.0
  odd[1, 30], odd[1, 31, 5], odd[1, 32, 7] = float("nan"), float("inf"), float("-inf")
  odd[1, 33] = 3e38

  def grads(x):
    leaves = [t.detach().requires_grad_() for t in (x, y, pw, w, g)]
    _, s = branch.branch_norm(*leaves[:4], gate=leaves[4], residual_scale=0.5, p=0.1, seed=9)
    return torch.autograd.grad(s, leaves, ds, allow_unused=True)

  for name, a, b in zip(("x", "y", "post_weight", "weight", "gate"), grads(odd), grads(x)):
    assert torch.isfinite(a).all() and torch.equal(a, b), name
  assert torch.equal(grads(odd)[0], 0.5 * ds)


def test_a_branch_that_is_not_a_number(cuda):
  """x's gradient of the stream alone is the stream's, whatever the branch holds."""
  from faster_weathernext import branch
  x, y = torch.ones(4, 64, device="cuda", requires_grad=True), torch.ones(4, 64, device="cuda")
  y[1], y[2, 3] = float("nan"), float("inf")
  d_x, = torch.autograd.grad(branch.branch_norm(x, y)[1], x, torch.full_like(x, 3.0))
  assert torch.equal(d_x, torch.full_like(x, 3.0))
