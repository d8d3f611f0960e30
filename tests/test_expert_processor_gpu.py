"""GPU: expert_processor.ExpertProcessor, the residual branches, the routing and the products grouped by expert together
around the attention kernels, against the same blocks in plain float32 torch with a dense masked softmax, on the choices that
the model made (a logit's rounding may decide between two experts). Bounds as test_rms_processor_gpu.py's: 2e-2 of the
outputs and 5e-2 of all gradients for bf16 products; 1e-1 with 8-bit operands."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _generators_as_they_were():
  """What these tests draw from torch's default generators does not move the values of the tests after them."""
  with torch.random.fork_rng():
    yield


def _cfg(**kw):
  from faster_weathernext.processor import ProcessorConfig
  return ProcessorConfig(**{**dict(layers=2, d_model=128, heads=2, head_dim=64, mlp_hidden=256, cond_dim=8), **kw})


def _rel(a, b):
  a, b = a.double(), b.double()
  return float(torch.sqrt(torch.mean((a - b) ** 2)) / b.std())


def _setup(cuda, cfg, seed=1, **kw):
  from faster_weathernext import mesh
  from faster_weathernext import tiled_attn as ta
  from faster_weathernext.expert_processor import ExpertProcessor
  m, _, _ = mesh.config_mask(1)
  model = ExpertProcessor(cfg, seed=3, device=cuda, **kw)
  g = torch.Generator(device=cuda).manual_seed(seed)
  with torch.no_grad():
    for name, p in model.named_parameters():
      if p.dim() == 1 or ".b" in name:
        p.add_(0.1 * torch.randn(p.shape, device=cuda, generator=g))
      elif "w_gate" in name:
        p.add_(0.05 * torch.randn(p.shape, device=cuda, generator=g))
  x = torch.randn(2, m.shape[0], cfg.d_model, device=cuda, generator=g)
  cond = torch.randn(2, cfg.cond_dim, device=cuda, generator=g)
  return model, x, cond, ta.AttentionTiles.from_mask(m, device=cuda), torch.from_numpy(m.toarray()).to(cuda)


def _choices(monkeypatch):
  """Collects the experts that the model chooses."""
  from faster_weathernext import experts
  seen, route = [], experts.route

  def watched(logits, top_k):
    r = route(logits, top_k)
    seen.append(r.experts.long())
    return r

  monkeypatch.setattr(experts, "route", watched)
  return seen


def _plain(model, x, mask, cond, chosen, seed=None):
  from oracle import dropout
  cfg, eps = model.cfg, model.eps
  b, n, d = x.shape
  norm = lambda t, w: t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps) * w  # noqa: E731

  def end(x, y, post, gate, w_gate, site):
    z = norm(y, post) * (gate if cond is None else gate + cond @ w_gate)[..., None, :] if cond is not None else norm(y, post) * gate
    if seed is not None:
      z = z * torch.from_numpy(dropout.factors((b, n, d), model.dropout, seed, site)).to(z)
    return model.residual_scale * x + z

  h = norm(x, model.norm_first)
  for i, blk in enumerate(model.blocks):
    qkv = (h @ blk.w_qkv).view(b, n, cfg.heads, 3, cfg.head_dim)
    q, k, v = (qkv[:, :, :, j].permute(0, 2, 1, 3) for j in range(3))
    s = (q @ k.transpose(-1, -2)) * cfg.head_dim ** -0.5
    o = torch.softmax(s.masked_fill(~mask, float("-inf")), -1) @ v
    x = end(x, o.permute(0, 2, 1, 3).reshape(b, n, -1) @ blk.w_out, blk.post1, blk.gate1, blk.w_gate1, 2 * i)
    h = norm(x, blk.norm1).reshape(b * n, d)
    idx = chosen[i]
    w = torch.softmax(torch.gather(h @ blk.w_router, 1, idx), 1)
    all_out = torch.stack([torch.nn.functional.gelu(h @ w1 + b1, approximate="tanh") @ w2 + b2
                           for w1, b1, w2, b2 in zip(blk.w1, blk.b1, blk.w2, blk.b2)], 1)
    m = (w[:, :, None] * torch.gather(all_out, 1, idx[:, :, None].expand(-1, -1, d))).sum(1)
    x = end(x, m.view(b, n, d), blk.post2, blk.gate2, blk.w_gate2, 2 * i + 1)
    h = norm(x, blk.norm2)
  return h


@pytest.mark.parametrize("kw", [dict(), dict(dropout=0.2, residual_scale=0.8), dict(experts=5, top_k=3, cond=False),
                                dict(cfg=dict(d_model=120, mlp_hidden=250), dropout=0.1)])
def test_forward_and_gradients_match_plain_torch(cuda, monkeypatch, kw):
  kw = dict(kw)
  cfg, with_cond = kw.pop("cfg", {}), kw.pop("cond", True)
  model, x, cond, tiles, mask = _setup(cuda, _cfg(**cfg), **kw)
  cond = cond if with_cond else None
  seen = _choices(monkeypatch)
  t = torch.randn_like(x)
  seed = 77 if model.dropout else None
  ya = model(x, tiles, cond, seed=seed)
  params = [p for name, p in model.named_parameters() if with_cond or "w_gate" not in name]
  ga = torch.autograd.grad(torch.nn.functional.mse_loss(ya, t), params)
  yb = _plain(model, x, mask, cond, seen, seed)
  gb = torch.autograd.grad(torch.nn.functional.mse_loss(yb, t), params)
  assert ya.dtype == torch.float32 and _rel(ya, yb) < 2e-2
  ga, gb = (torch.cat([v.reshape(-1) for v in s]) for s in (ga, gb))
  assert _rel(ga, gb) < 5e-2
  from faster_weathernext import _lib
  assert _lib.device_error() == 0


@pytest.mark.parametrize("eight_bit", [False, True])
def test_forecast(cuda, monkeypatch, eight_bit):
  model, x, cond, tiles, mask = _setup(cuda, _cfg(), dropout=0.3)
  model.eval()
  plan = model.forecast_plan(eight_bit)
  seen = _choices(monkeypatch)
  got = model.forecast(x, tiles, plan, cond)
  want = _plain(model, x, mask, cond, seen)
  assert _rel(got, want) < (1e-1 if eight_bit else 2e-2)
  if not eight_bit:
    with torch.no_grad():
      assert _rel(model(x, tiles, cond), got) < 2e-2


def test_single_node(cuda):
  """One node: every call's form for few rows."""
  from scipy import sparse
  from faster_weathernext import tiled_attn as ta
  model, _, cond, _, _ = _setup(cuda, _cfg())
  tiles = ta.AttentionTiles.from_mask(sparse.csr_matrix([[True]]), device=cuda)
  x = torch.randn(1, 1, 128, device=cuda)
  model.eval()
  a, b = model.forecast(x, tiles, model.forecast_plan(False), cond[:1]), model(x, tiles, cond[:1])
  assert a.shape == (1, 1, 128) and _rel(a.detach(), b.detach()) < 2e-2


def test_training_step_in_a_graph(cuda):
  """A captured step replayed with a new seed is the eager step of that seed."""
  model, x, cond, tiles, _ = _setup(cuda, _cfg(), dropout=0.1)
  seed = torch.tensor([1], device=cuda)
  params = list(model.parameters())

  def step():
    y = model(x, tiles, cond, seed=seed)
    return [y.detach(), *torch.autograd.grad(y.square().mean(), params)]

  step()
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = step()
  for s in (1, 5):
    seed.fill_(s)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_no_blocks_and_refusals(cuda):
  model, x, cond, tiles, _ = _setup(cuda, _cfg(layers=0), dropout=0.1)
  assert torch.equal(model(x, tiles, cond, seed=1), model.forecast(x, tiles, model.forecast_plan(), cond))
  from faster_weathernext.expert_processor import ExpertProcessor
  with pytest.raises(ValueError):
    ExpertProcessor(_cfg(), experts=2, top_k=3)
  with pytest.raises(ValueError):
    model(x, tiles, cond)            # dropout without a seed
  with pytest.raises(ValueError):
    model(x[0], tiles, cond, seed=1)
  with pytest.raises(ValueError):
    model(x, tiles, cond[:1], seed=1)
