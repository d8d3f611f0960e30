"""GPU: gradients where saved tensors come back in other places between forward and backward (torch.autograd.graph's hooks
move them): rows with a stride come back without one, or every value with one. What the kernels take is laid out again."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _randn(seed):
  g = torch.Generator(device="cuda").manual_seed(seed)
  return lambda *s: torch.randn(*s, device="cuda", generator=g)


def _spread():
  """Every saved tensor comes back as a view whose neighbouring values are two apart, the ones between being others."""
  return torch.autograd.graph.saved_tensors_hooks(lambda t: torch.stack((t, t.flip(0)), -1), lambda t: t[..., 0])


HOOKS = {"cpu": torch.autograd.graph.save_on_cpu, "spread": _spread}


def _same(step, hooks, room=0.0):
  want = step()
  with HOOKS[hooks]():
    got = step()
  assert len(got) == len(want)
  for a, b in zip(got, want):
    assert a.shape == b.shape and a.dtype is b.dtype
    if room:
      assert (a.double() - b.double()).abs().max() <= room * b.double().abs().max()
    else:
      assert torch.equal(a, b)


@pytest.mark.parametrize("hooks", HOOKS)
@pytest.mark.parametrize("k,n,layout,act", [(65, 33, "nk", "gelu"), (1001, 515, "nk", None), (128, 64, "nk", "swish"),
                                            (65, 40, "kn", "gelu"), (64, 35, "kn", None)])
def test_grouped(cuda, hooks, k, n, layout, act):
  """Padded copies of odd widths, wide rows and transposed weights. The transposed come back the other way round, whose
  gradient may take other tiles: another order of the float32 sums, a step of bf16."""
  from faster_weathernext import experts
  r = _randn(k)
  wide, w, b = r(210, k + 9).to(BF16), (r(3, n, k) * k ** -0.5).to(BF16), r(3, n)
  if layout == "kn":
    w = w.transpose(1, 2).contiguous().transpose(1, 2)
  offsets = torch.tensor([2, 102, 102, 200], dtype=torch.int32, device="cuda")
  dy = r(210, n).to(BF16)

  def step():
    leaves = [t.detach().requires_grad_() for t in (wide, w, b)]
    y = experts.linear_grouped(leaves[0][:, 3:3 + k], leaves[1], offsets, leaves[2], activation=act)
    return torch.autograd.grad(y, leaves, dy)

  _same(step, hooks, 2.0 ** -7 if layout == "kn" else 0.0)


@pytest.mark.parametrize("hooks", HOOKS)
@pytest.mark.parametrize("rows,d", [(37, 64), (300, 65)])
def test_routing(cuda, hooks, rows, d):
  from faster_weathernext import experts
  r = _randn(rows)
  x, y, logits, d_rows, d_out = r(rows, d), r(rows * 3, d), r(rows, 7), r(rows * 3, d), r(rows, d)

  def step():
    leaves = [t.detach().requires_grad_() for t in (x, y, logits)]
    routing = experts.route(leaves[2], 3)
    return torch.autograd.grad((experts.dispatch(leaves[0], routing), experts.combine(leaves[1], routing)), leaves, (d_rows, d_out))

  _same(step, hooks)


@pytest.mark.parametrize("hooks", HOOKS)
@pytest.mark.parametrize("d", [72, 333])
def test_branch(cuda, hooks, d):
  from faster_weathernext import branch
  r = _randn(d)
  wide, y, pw, w, gate = r(33, d + 88), r(33, d).to(BF16), r(d), r(d).to(BF16), r(33, d)
  dh, ds = r(33, d).to(BF16), r(33, d)
  seed = torch.tensor([77], dtype=torch.int64, device="cuda")

  def step():
    leaves = [t.detach().requires_grad_() for t in (wide, y, pw, w, gate)]
    h, s = branch.branch_norm(leaves[0][:, 8:8 + d], *leaves[1:4], gate=leaves[4], p=0.25, seed=seed)
    dropped = branch.dropout(leaves[1], 0.5, seed, site=1)
    return torch.autograd.grad((h, s, dropped), leaves, (dh, ds, dh))

  _same(step, hooks)


@pytest.mark.parametrize("hooks", HOOKS)
@pytest.mark.parametrize("k,n", [(64, 48), (65, 33)])
def test_projection(cuda, hooks, k, n):
  from faster_weathernext import projection
  r = _randn(n)
  x, w, b, nw, a = r(90, k), (r(n, k) * k ** -0.5).to(BF16), r(n), r(k), r(90, k)
  dy, ds = r(90, n).to(BF16), r(90, k)

  def step():
    leaves = [t.detach().requires_grad_() for t in (x, w, b, nw, a)]
    h, s = projection.rms_norm(leaves[0], leaves[3], residual=leaves[4])
    y = projection.linear(h, leaves[1], leaves[2], activation="gelu")
    return torch.autograd.grad((y, s), leaves, (dy, ds))

  _same(step, hooks)


@pytest.mark.parametrize("hooks", HOOKS)
@pytest.mark.parametrize("fused", [False, True])
def test_attention(cuda, hooks, fused):
  from faster_weathernext import mesh, tiled_attn
  mask, _, _ = mesh.config_mask(1)
  tiles = tiled_attn.AttentionTiles.from_mask(mask, device=cuda)
  r = _randn(4)
  qkv, dy = r(1, mask.shape[0], 2, 3, 64).to(BF16), r(1, mask.shape[0], 2, 64).to(BF16)

  def step():
    leaf = qkv.detach().requires_grad_()
    if fused:
      y = tiled_attn.attention_qkv(leaf, tiles, scale=0.125)
    else:
      y = tiled_attn.attention(*leaf.unbind(3), tiles, scale=0.125)
    return torch.autograd.grad(y, leaf, dy)

  _same(step, hooks)


@pytest.mark.parametrize("hooks", HOOKS)
def test_expert_processor(cuda, hooks):
  """A training step of the operators together, at an odd width of the experts' MLPs. Transposed weights come back the other way
  round, so that products may be summed in another order: each run is within the processor's bound for gradients of bf16
  products, 5e-2 of their norm, and so are the two of each other."""
  from faster_weathernext import mesh, tiled_attn
  from faster_weathernext.expert_processor import ExpertProcessor
  from faster_weathernext.processor import ProcessorConfig
  cfg = ProcessorConfig(layers=2, d_model=128, heads=2, head_dim=64, mlp_hidden=251, cond_dim=8)
  mask, _, _ = mesh.config_mask(1)
  r = _randn(1)
  model = ExpertProcessor(cfg, seed=3, device=cuda, dropout=0.1)
  x, cond, dy = r(1, mask.shape[0], 128), r(1, 8), r(1, mask.shape[0], 128)
  tiles = tiled_attn.AttentionTiles.from_mask(mask, device=cuda)
  leaves = [x.requires_grad_(), *model.parameters()]
  step = lambda: torch.autograd.grad(model(x, tiles, cond, seed=5), leaves, dy)  # noqa: E731
  want = step()
  with HOOKS[hooks]():
    got = step()
  for a, b in zip(got, want):
    assert (a.double() - b.double()).norm() <= 5e-2 * b.double().norm()


@pytest.mark.parametrize("hooks", HOOKS)
def test_processor(cuda, hooks):
  """The processor's own functions (torch's products around them take moved operands in another order of their sums)."""
  from faster_weathernext import processor
  r = _randn(2)
  x, a, so, dx, dh = r(84, 128), r(84, 128).to(BF16), r(2, 256), r(84, 128), r(84, 128).to(BF16)
  w1, b1, w2, b2 = r(128, 256) * 0.1, r(256), r(256, 128) * 0.1, r(128)

  def step():
    leaves = [t.detach().requires_grad_() for t in (x, a, so, w1, b1, w2, b2)]
    added, h = processor._CondNorm.apply(*leaves[:3], 42, BF16)
    first = processor._CondNorm.apply(leaves[0], None, leaves[2], 42, F32)
    y = processor._GeluMLP.apply(h, *leaves[3:])
    return torch.autograd.grad((added, y, first), leaves, (dx, dh, dx))

  _same(step, hooks)
