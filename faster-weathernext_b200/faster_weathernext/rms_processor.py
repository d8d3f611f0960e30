"""A mesh-transformer processor of RMS-norm blocks on the pre-norm projections (faster_weathernext.projection).

    x = x + attention(q, k, v of rms_norm(x)) w_out
    x = x + GELU(rms_norm(x) w1 + b1) w2 + b2

The block of later transformers, beside processor.Processor's conditioned LayerNorm blocks (src/faster_weathernext/patch.py:
229-293; no counterpart of this form in the reference), of the same configurations (ProcessorConfig) and with the same
attention kernels. Weights are stored as the processor's, [in, out] float32.

Training: model(x, tiles). Every product, norm and residual runs on fwn_linear and fwn_rms_norm with their gradients: the
output projection adds the residual stream in its epilogue, the MLP's output (bf16) is added by the next norm.

Forecasts: plan = model.forecast_plan(eight_bit=True) once per set of weights, then model.forecast(x, tiles, plan): the
norms write 8-bit rows with scales and the q / k / v and up-projections, 58 % of the products' work at widths of 512 and
2,048, multiply them with 8-bit weights; without eight_bit the plan holds bf16 weights. 24 layers on 40,962 nodes, one
B200: forecast 10.4 ms, with 8-bit rows 9.2, forward and gradients 39.8.
"""

import dataclasses

import torch

from faster_weathernext import patch
from faster_weathernext import projection
from faster_weathernext import tiled_attn
from faster_weathernext.processor import ProcessorConfig, _glorot

_BF16, _F32 = torch.bfloat16, torch.float32


@dataclasses.dataclass
class ForecastPlan:
  """The weights of a forecast, laid out once: per block bf16 tensors [out, in], q / k / v and up-projection optionally as
  (e4m3 values, scales); biases and norm weights float32. Holds copies: build it again after the weights change."""
  eight_bit: bool
  blocks: list
  norm_final: torch.Tensor


class RmsProcessor(torch.nn.Module):
  """Random-init RMS-norm processor; parameters float32, products in bf16 (or 8 bits in a forecast)."""

  def __init__(self, cfg: ProcessorConfig = ProcessorConfig(), seed: int = 0, device=None, eps: float = 1e-6):
    super().__init__()
    self.cfg, self.eps = cfg, eps
    dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    d, hd = cfg.d_model, cfg.heads * cfg.head_dim
    self.blocks = torch.nn.ModuleList()
    for _ in range(cfg.layers):
      blk = torch.nn.Module()
      blk.norm1 = torch.nn.Parameter(torch.ones(d, device=dev))
      blk.norm2 = torch.nn.Parameter(torch.ones(d, device=dev))
      blk.w_qkv = _glorot(gen, d, 3 * hd, dev)      # columns [head, (q, k, v), head_dim], as Processor's
      blk.w_out = _glorot(gen, hd, d, dev)
      blk.w1 = _glorot(gen, d, cfg.mlp_hidden, dev)
      blk.b1 = torch.nn.Parameter(torch.zeros(cfg.mlp_hidden, device=dev))
      blk.w2 = _glorot(gen, cfg.mlp_hidden, d, dev)
      blk.b2 = torch.nn.Parameter(torch.zeros(d, device=dev))
      self.blocks.append(blk)
    self.norm_final = torch.nn.Parameter(torch.ones(d, device=dev))

  def _check(self, x):
    if x.dim() != 3 or x.shape[2] != self.cfg.d_model or x.dtype != _F32:
      raise ValueError(f"x has shape {tuple(x.shape)} and dtype {x.dtype}, expected float32 [B, n, {self.cfg.d_model}]")

  def _attend(self, qkv, tiles, b, n):
    cfg = self.cfg
    out = tiled_attn.attention_qkv(qkv.view(b, n, cfg.heads, 3, cfg.head_dim), tiles, scale=cfg.head_dim ** -0.5,
                                   strict_fp32=patch.OPTIONS.strict_fp32)
    return out.reshape(b * n, cfg.heads * cfg.head_dim)

  def forward(self, x: torch.Tensor, tiles: "tiled_attn.AttentionTiles") -> torch.Tensor:
    """x [B, n, d_model] float32 -> [B, n, d_model] float32, differentiable."""
    self._check(x)
    b, n, d = x.shape
    rows, pending = x.reshape(b * n, d), None
    norm = lambda w: projection.rms_norm(rows, w, pending, eps=self.eps)  # noqa: E731
    for blk in self.blocks:
      if pending is None:
        h = norm(blk.norm1)
      else:
        h, rows = norm(blk.norm1)
      qkv = projection.linear(h, blk.w_qkv.to(_BF16).t())
      rows = projection.linear(self._attend(qkv, tiles, b, n), blk.w_out.to(_BF16).t(), None, rows, out_dtype=_F32)
      h = projection.rms_norm(rows, blk.norm2, eps=self.eps)
      h = projection.linear(h, blk.w1.to(_BF16).t(), blk.b1, activation="gelu")
      pending = projection.linear(h, blk.w2.to(_BF16).t(), blk.b2)
    if pending is None:
      return projection.rms_norm(rows, self.norm_final, eps=self.eps, out_dtype=_F32).view(b, n, d)
    return projection.rms_norm(rows, self.norm_final, pending, eps=self.eps, out_dtype=_F32)[0].view(b, n, d)

  @torch.no_grad()
  def forecast_plan(self, eight_bit: bool = True) -> ForecastPlan:
    """The weights as a forecast reads them (rows along the summed dimension), 8-bit where the norms feed them."""
    turned = lambda w: w.detach().t().to(_BF16).contiguous()  # noqa: E731
    fed = lambda w: projection.quantize_fp8(w.detach().t().contiguous()) if eight_bit else turned(w)  # noqa: E731
    blocks = [{"norm1": blk.norm1.detach().clone(), "norm2": blk.norm2.detach().clone(), "w_qkv": fed(blk.w_qkv),
               "w_out": turned(blk.w_out), "w1": fed(blk.w1), "b1": blk.b1.detach().clone(), "w2": turned(blk.w2),
               "b2": blk.b2.detach().clone()} for blk in self.blocks]
    return ForecastPlan(eight_bit, blocks, self.norm_final.detach().clone())

  @torch.no_grad()
  def forecast(self, x: torch.Tensor, tiles: "tiled_attn.AttentionTiles", plan: ForecastPlan) -> torch.Tensor:
    """forward without gradients on a plan's weights; x [B, n, d_model] float32 (B = 1, n = 1 included)."""
    self._check(x)
    b, n, d = x.shape
    rows, pending = x.reshape(b * n, d), None

    def fed(weight, w, bias=None, activation=None):
      """The norm of the stream (with what is pending added into it) through a product; the stream after the norm."""
      if plan.eight_bit:
        got = projection.rms_norm_fp8(rows, weight, pending, eps=self.eps)
        y = projection.linear_fp8(got[0], got[1], w[0], w[1], bias, activation=activation)
        return y, rows if pending is None else got[2]
      got = projection.rms_norm(rows, weight, pending, eps=self.eps)
      h, stream = (got, rows) if pending is None else got
      return projection.linear(h, w, bias, activation=activation), stream

    for blk in plan.blocks:
      qkv, rows = fed(blk["norm1"], blk["w_qkv"])
      rows = projection.linear(self._attend(qkv, tiles, b, n), blk["w_out"], None, rows, out_dtype=_F32)
      pending = None
      h, _ = fed(blk["norm2"], blk["w1"], blk["b1"], "gelu")
      pending = projection.linear(h, blk["w2"], blk["b2"])
    got = projection.rms_norm(rows, plan.norm_final, pending, eps=self.eps, out_dtype=_F32)
    return (got if pending is None else got[0]).view(b, n, d)
