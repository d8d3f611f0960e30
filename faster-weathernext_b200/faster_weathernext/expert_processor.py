"""A mesh-transformer processor whose MLPs are mixtures of experts and whose blocks end in normed, gated branches.

    x = s x + dropout(gate norm(attention(q, k, v of h) w_out)),                 h = norm(x)
    x = s x + dropout(gate norm(sum over a node's experts of weight * expert(h))),  h = norm(x) of the next block

The block of later transformers, beside rms_processor.RmsProcessor's (src/faster_weathernext/patch.py:229-293; no counterpart
of this form in the reference), of the same configurations (ProcessorConfig) and with the same attention kernels: every norm
after a block, its gate, dropout, the residual's addition and the norm before the next block are one pass
(branch.branch_norm), every node goes to `top_k` of `experts` MLPs (experts.route, dispatch, linear_grouped, combine). The
gates are learned per channel, and with a conditioning vector per sample: gate = blk.gate + cond w_gate. Weights are stored
as the processor's, [in, out] (of each expert) float32.

Training: model(x, tiles, cond, seed=step's seed). Forecasts: plan = model.forecast_plan() once per set of weights, then
model.forecast(x, tiles, plan, cond): no dropout, weights laid out for the kernels, and (eight_bit) the q / k / v projections'
operands in 8 bits with scales.
"""

import dataclasses

import torch

from faster_weathernext import branch
from faster_weathernext import experts as moe
from faster_weathernext import patch
from faster_weathernext import projection
from faster_weathernext import tiled_attn
from faster_weathernext.processor import ProcessorConfig, _glorot

_BF16, _F32 = torch.bfloat16, torch.float32


@dataclasses.dataclass
class ExpertPlan:
  """The weights of a forecast, laid out once: bf16 tensors with rows along the summed dimension, q / k / v optionally as
  (e4m3 values, scales); norms, biases and gates float32. Holds copies: build it again after the weights change. Rows are as
  long as their dimension: those off multiples of 8 (an odd mlp_hidden) are laid out again by every product."""
  eight_bit: bool
  blocks: list
  norm_first: torch.Tensor


class ExpertProcessor(torch.nn.Module):
  """Random-init processor of `experts` MLPs a block, `top_k` for each node; parameters float32, products in bf16."""

  def __init__(self, cfg: ProcessorConfig = ProcessorConfig(), experts: int = 8, top_k: int = 2, dropout: float = 0.0,
               residual_scale: float = 1.0, seed: int = 0, device=None, eps: float = 1e-6):
    super().__init__()
    if not 1 <= top_k <= experts:
      raise ValueError(f"top_k is {top_k}, expected 1 to {experts} (the number of experts)")
    self.cfg, self.experts, self.top_k, self.dropout, self.residual_scale, self.eps = cfg, experts, top_k, dropout, residual_scale, eps
    dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    d, hd, hidden = cfg.d_model, cfg.heads * cfg.head_dim, cfg.mlp_hidden
    ones = lambda: torch.nn.Parameter(torch.ones(d, device=dev))  # noqa: E731
    stack = lambda i, o: torch.nn.Parameter(torch.stack([_glorot(gen, i, o, dev).detach() for _ in range(experts)]))  # noqa: E731
    zeros = lambda *s: torch.nn.Parameter(torch.zeros(*s, device=dev))  # noqa: E731
    self.norm_first = ones()
    self.blocks = torch.nn.ModuleList()
    for _ in range(cfg.layers):
      blk = torch.nn.Module()
      blk.w_qkv = _glorot(gen, d, 3 * hd, dev)      # columns [head, (q, k, v), head_dim], as Processor's
      blk.w_out = _glorot(gen, hd, d, dev)
      blk.post1, blk.gate1, blk.w_gate1, blk.norm1 = ones(), ones(), zeros(cfg.cond_dim, d), ones()
      blk.w_router = _glorot(gen, d, experts, dev)
      blk.w1, blk.b1 = stack(d, hidden), zeros(experts, hidden)
      blk.w2, blk.b2 = stack(hidden, d), zeros(experts, d)
      blk.post2, blk.gate2, blk.w_gate2, blk.norm2 = ones(), ones(), zeros(cfg.cond_dim, d), ones()
      self.blocks.append(blk)

  def _check(self, x, cond):
    if x.dim() != 3 or x.shape[2] != self.cfg.d_model or x.dtype != _F32:
      raise ValueError(f"x has shape {tuple(x.shape)} and dtype {x.dtype}, expected float32 [B, n, {self.cfg.d_model}]")
    if cond is not None and (cond.shape != (x.shape[0], self.cfg.cond_dim) or cond.dtype != _F32):
      raise ValueError(f"cond has shape {tuple(cond.shape)} and dtype {cond.dtype}, expected float32 ({x.shape[0]}, {self.cfg.cond_dim})")

  def _attend(self, qkv, tiles, b, n):
    cfg = self.cfg
    out = tiled_attn.attention_qkv(qkv.view(b, n, cfg.heads, 3, cfg.head_dim), tiles, scale=cfg.head_dim ** -0.5,
                                   strict_fp32=patch.OPTIONS.strict_fp32)
    return out.reshape(b * n, cfg.heads * cfg.head_dim)

  def _mix(self, h, w_router, w1, b1, w2, b2):
    """The experts' MLPs on rows h, weights as [out, in] views."""
    r = moe.route(projection.linear(h, w_router, out_dtype=_F32), self.top_k)
    y = moe.linear_grouped(moe.dispatch(h, r), w1, r.offsets, b1, activation="gelu")
    return moe.combine(moe.linear_grouped(y, w2, r.offsets, b2), r)

  def forward(self, x: torch.Tensor, tiles: "tiled_attn.AttentionTiles", cond: torch.Tensor = None, seed=None) -> torch.Tensor:
    """x [B, n, d_model] float32 -> [B, n, d_model] float32, differentiable. cond [B, cond_dim] float32 or None; seed: of
    the step's dropout (branch.dropout's: an int or an int64 tensor on the device), read in training mode with dropout > 0;
    block l drops at sites 2 l and 2 l + 1."""
    self._check(x, cond)
    b, n, d = x.shape
    p = self.dropout if self.training else 0.0
    if p > 0 and seed is None:
      raise ValueError("dropout in training needs the step's seed")
    gate_of = lambda gate, w: gate if cond is None else gate + cond @ w  # noqa: E731
    end = lambda y, post, gate, weight, site, out: branch.branch_norm(  # noqa: E731
        x, y.view(b, n, d), post, weight, gate=gate, residual_scale=self.residual_scale, p=p, seed=seed, site=site, eps=self.eps,
        out_dtype=out)
    turned = lambda w: w.to(_BF16).transpose(-1, -2)  # noqa: E731
    h = projection.rms_norm(x, self.norm_first, eps=self.eps, out_dtype=_BF16 if self.blocks else _F32)
    for i, blk in enumerate(self.blocks):
      qkv = projection.linear(h.view(b * n, d), turned(blk.w_qkv))
      a = projection.linear(self._attend(qkv, tiles, b, n), turned(blk.w_out))
      h, x = end(a, blk.post1, gate_of(blk.gate1, blk.w_gate1), blk.norm1, 2 * i, _BF16)
      m = self._mix(h.view(b * n, d), turned(blk.w_router), turned(blk.w1), blk.b1, turned(blk.w2), blk.b2)
      h, x = end(m, blk.post2, gate_of(blk.gate2, blk.w_gate2), blk.norm2, 2 * i + 1,
                 _F32 if i + 1 == len(self.blocks) else _BF16)
    return h

  @torch.no_grad()
  def forecast_plan(self, eight_bit: bool = True) -> ExpertPlan:
    """The weights as a forecast reads them (rows along the summed dimension), q / k / v in 8 bits."""
    turned = lambda w: w.detach().transpose(-1, -2).to(_BF16).contiguous()  # noqa: E731
    fed = lambda w: projection.quantize_fp8(w.detach().t().contiguous()) if eight_bit else turned(w)  # noqa: E731
    blocks = []
    for blk in self.blocks:
      kept = {k: v.detach().clone() for k, v in blk.named_parameters() if not k.startswith("w")}
      blocks.append({**kept, "w_gate1": blk.w_gate1.detach().clone(), "w_gate2": blk.w_gate2.detach().clone(),
                     "w_qkv": fed(blk.w_qkv), **{k: turned(getattr(blk, k)) for k in ("w_out", "w_router", "w1", "w2")}})
    return ExpertPlan(eight_bit, blocks, self.norm_first.detach().clone())

  @torch.no_grad()
  def forecast(self, x: torch.Tensor, tiles: "tiled_attn.AttentionTiles", plan: ExpertPlan, cond: torch.Tensor = None) -> torch.Tensor:
    """forward without gradients and dropout on a plan's weights; x [B, n, d_model] float32 (B = 1, n = 1 included)."""
    self._check(x, cond)
    b, n, d = x.shape
    if not plan.blocks:
      return projection.rms_norm(x, plan.norm_first, eps=self.eps, out_dtype=_F32)
    gate_of = lambda blk, i: blk[f"gate{i}"] if cond is None else blk[f"gate{i}"] + cond @ blk[f"w_gate{i}"]  # noqa: E731
    kw = {"residual_scale": self.residual_scale, "eps": self.eps}
    h = (projection.rms_norm_fp8 if plan.eight_bit else projection.rms_norm)(x, plan.norm_first, eps=self.eps)
    for i, blk in enumerate(plan.blocks):
      if plan.eight_bit:
        qkv = projection.linear_fp8(h[0].view(b * n, d), h[1].view(b * n), *blk["w_qkv"])
      else:
        qkv = projection.linear(h.view(b * n, d), blk["w_qkv"])
      a = projection.linear(self._attend(qkv, tiles, b, n), blk["w_out"])
      h, x = branch.branch_norm(x, a.view(b, n, d), blk["post1"], blk["norm1"], gate=gate_of(blk, 1), **kw)
      m = self._mix(h.view(b * n, d), *[blk[k] for k in ("w_router", "w1", "b1", "w2", "b2")]).view(b, n, d)
      ends = x, m, blk["post2"], blk["norm2"]
      if i + 1 == len(plan.blocks):
        return branch.branch_norm(*ends, gate=gate_of(blk, 2), out_dtype=_F32, **kw)[0]
      if plan.eight_bit:
        values, scale, x = branch.branch_norm_fp8(*ends, gate=gate_of(blk, 2), **kw)
        h = values, scale
      else:
        h, x = branch.branch_norm(*ends, gate=gate_of(blk, 2), **kw)
