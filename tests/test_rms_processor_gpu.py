"""GPU: rms_processor.RmsProcessor, the RMS-norm blocks on the pre-norm projections around the attention kernels, against
the same blocks in plain float32 torch with a dense masked softmax. Bounds: bf16 products and attention as
test_processor_gpu.py's (2e-2 outputs, 5e-2 all gradients); an 8-bit product's operands are each off by 2.6e-2 (the mean
square of e4m3 rounding), so 3.7e-2 of a product and, over the four 8-bit products of two blocks, at most 7.4e-2 of the
output: 1e-1."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _cfg(**kw):
  from faster_weathernext.processor import ProcessorConfig
  return ProcessorConfig(**{**dict(layers=2, d_model=128, heads=2, head_dim=64, mlp_hidden=256, cond_dim=8), **kw})


def _rel(a, b):
  a, b = a.double(), b.double()
  return float(torch.sqrt(torch.mean((a - b) ** 2)) / b.std())


def _plain(model, x, mask):
  cfg, eps = model.cfg, model.eps
  norm = lambda t, w: t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps) * w  # noqa: E731
  for blk in model.blocks:
    b, n, _ = x.shape
    qkv = (norm(x, blk.norm1) @ blk.w_qkv).view(b, n, cfg.heads, 3, cfg.head_dim)
    q, k, v = (qkv[:, :, :, i].permute(0, 2, 1, 3) for i in range(3))
    s = (q @ k.transpose(-1, -2)) * cfg.head_dim ** -0.5
    o = torch.softmax(s.masked_fill(~mask, float("-inf")), -1) @ v
    x = x + o.permute(0, 2, 1, 3).reshape(b, n, -1) @ blk.w_out
    x = x + torch.nn.functional.gelu(norm(x, blk.norm2) @ blk.w1 + blk.b1, approximate="tanh") @ blk.w2 + blk.b2
  return norm(x, model.norm_final)


def _setup(cuda, cfg, seed=1):
  from faster_weathernext import mesh
  from faster_weathernext import tiled_attn as ta
  from faster_weathernext.rms_processor import RmsProcessor
  m, _, _ = mesh.config_mask(1)
  model = RmsProcessor(cfg, seed=3, device=cuda)
  g = torch.Generator(device=cuda).manual_seed(seed)
  with torch.no_grad():
    for p in model.parameters():
      if p.dim() == 1:
        p.add_(0.1 * torch.randn(p.shape, device=cuda, generator=g))
  x = torch.randn(2, m.shape[0], cfg.d_model, device=cuda, generator=g)
  return model, x, ta.AttentionTiles.from_mask(m, device=cuda), torch.from_numpy(m.toarray()).to(cuda)


@pytest.mark.parametrize("cfg", [{}, {"d_model": 120, "mlp_hidden": 250}])
def test_forward_and_gradients_match_plain_torch(cuda, cfg):
  model, x, tiles, mask = _setup(cuda, _cfg(**cfg))
  t = torch.randn_like(x)
  ya = model(x, tiles)
  ga = torch.autograd.grad(torch.nn.functional.mse_loss(ya, t), list(model.parameters()))
  yb = _plain(model, x, mask)
  gb = torch.autograd.grad(torch.nn.functional.mse_loss(yb, t), list(model.parameters()))
  assert ya.dtype == torch.float32 and _rel(ya, yb) < 2e-2
  ga, gb = (torch.cat([v.reshape(-1) for v in s]) for s in (ga, gb))
  assert float((ga - gb).norm() / gb.norm()) < 5e-2


def test_forecast_matches_plain_torch_in_bf16_and_8_bits(cuda):
  model, x, tiles, mask = _setup(cuda, _cfg())
  with torch.no_grad():
    want = _plain(model, x, mask)
    assert _rel(model.forecast(x, tiles, model.forecast_plan(eight_bit=False)), want) < 2e-2
    plan = model.forecast_plan()
    got = model.forecast(x, tiles, plan)
    assert _rel(got, want) < 1e-1
    assert torch.equal(got, model.forecast(x, tiles, plan))
    # The plan keeps its weights when the model's change.
    model.blocks[0].w1.zero_()
    assert torch.equal(got, model.forecast(x, tiles, plan))


def test_refusals(cuda):
  model, x, tiles, _ = _setup(cuda, _cfg())
  for bad in (x[0], x[..., :64], x.bfloat16()):
    with pytest.raises(ValueError):
      model(bad, tiles)
    with pytest.raises(ValueError):
      model.forecast(bad, tiles, model.forecast_plan())
