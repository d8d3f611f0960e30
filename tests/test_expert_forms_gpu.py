"""GPU: sizes of the experts' block that the other tests pass over: one expert of nearly all rows among many, and the 8-bit
branch of enough rows that every block walks several."""
import pytest
import torch

from test_branch_gpu import E4M3, F32, BF16, U, _close, _formula, _inputs
from test_grouped_gpu import _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("others,k,n,act,layout", [(63, 512, 1024, "gelu", "kn"), (63, 256, 520, None, "nk"), (7, 1024, 512, "swish", "nk"),
                                                   (300, 65, 64, "gelu", "nk")])
@pytest.mark.parametrize("where", [0, 0.5, 1])
def test_one_expert_of_nearly_all_rows(cuda, others, k, n, act, layout, where):
  small = [(7 * i + 3) % 50 for i in range(others)]
  at = int(where * others)
  _check(small[:at] + [20_000] + small[at:], k, n, act, F32, BF16, layout, 0, 11)


@pytest.mark.parametrize("rows,d", [(9001, 64), (5003, 250), (2501, 515), (2001, 576), (3001, 2048), (601, 8185)])
@pytest.mark.parametrize("xd", [F32, BF16])
def test_branch_norm_fp8_of_many_rows(cuda, rows, d, xd):
  """Several rows a group of threads and gates that change between them. A row's scale: its values' float32 errors (the terms of
  s may cancel: their sum over the row's root mean square times as much), then the maximum and its quotient."""
  from faster_weathernext import branch
  x, y, pw, w, g = _inputs((2, rows, d), xd, BF16, "sample", F32)
  values, scale, s = branch.branch_norm_fp8(x, y, pw, w, gate=g, residual_scale=0.5)
  _, h64, s64 = _formula(x, y, pw, w, g, 0.5, 1e-6, None)
  h64, s64 = h64.detach(), s64.detach()
  ax = 0.5 * x.double()
  terms = (ax.abs() + (s64 - ax).abs()).amax(-1, keepdim=True)
  amp = 1 + 2 * terms / torch.sqrt((s64 ** 2).mean(-1, keepdim=True) + 1e-6)
  assert values.dtype is E4M3 and scale.shape == (2, rows)
  _close(s, s64, 60 * U * terms, "s")
  most = h64.abs().amax(-1, keepdim=True)
  _close(scale, most.squeeze(-1) / 448, (64 * U * amp * most / 448).squeeze(-1), "scale")
  # A value is rounded to e4m3 (2^-4 of itself, 2^-10 where that is subnormal) after float32's own errors.
  want = h64 / scale.double().unsqueeze(-1)
  off = (values.float().double() - want).abs()
  assert (off <= torch.maximum(want.abs() * 2.0 ** -4, torch.full_like(want, 2.0 ** -10)) + 448 * 64 * U * amp).all()
