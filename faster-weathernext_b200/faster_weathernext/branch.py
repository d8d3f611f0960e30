"""Residual branches: dropout from a counter-based generator, and the norms after and before a block in one pass with the
block's gate, dropout and residual scale.

    y = dropout(x, 0.1, seed, site=layer)                     # differentiable; the mask is never stored
    h, x = branch_norm(x, y, post_weight, weight, gate=gate, residual_scale=1.0, p=0.1, seed=seed, site=layer)
                                                              # x = residual_scale x + dropout(gate norm(y)), h = norm(x)
    values, scale, x = branch_norm_fp8(x, y, post_weight, weight, gate=gate)   # h in e4m3 with one scale per row

No counterpart in the reference, whose blocks add their output into the stream as it is (src/faster_weathernext/patch.py:
238-252): this is the sub-block's end in the form of later transformers, beside projection.rms_norm, which adds a residual
and norms the sum. The kernels are csrc/branch.cu and csrc/branch_bwd.cuh (C ABI in include/fwn_attn.h, fwn_dropout and
fwn_branch_norm*). Every call runs on the current stream of its tensors' device and takes its workspace from torch's
allocator.
"""

import ctypes

import torch

from faster_weathernext import _lib
from faster_weathernext.projection import (_BF16, _CODE, _E4M3, _F32, _check, _constant, _first_order, _no_tangent,
                                           _on_device, _rows)


# ---- dropout --------------------------------------------------------------------------------------------------------

def _drop_check(like, p, seed, site):
  """The threshold of 65,536 that p stands for."""
  if not 0.0 <= p <= 1.0:
    raise ValueError(f"p must lie between 0 and 1 (got {p})")
  if not 0 <= site < 2 ** 32:
    raise ValueError(f"site must be a 32-bit number, not negative (got {site})")
  if isinstance(seed, torch.Tensor):
    _check("seed", seed, like, (torch.int64,))
    if seed.numel() != 1:
      raise ValueError(f"seed has shape {tuple(seed.shape)}, expected one number")
  elif not isinstance(seed, int) or isinstance(seed, bool):
    raise TypeError(f"seed is {seed!r}, expected an int or an int64 tensor of one number")
  elif not 0 <= seed < 2 ** 64:
    raise ValueError(f"seed must be a 64-bit number, not negative (got {seed})")
  return int(round(65536 * p))


def _drop_desc(threshold, seed, site):
  if isinstance(seed, torch.Tensor):
    return _lib.DropoutDesc(0, seed.data_ptr(), site, threshold)
  return _lib.DropoutDesc(seed or 0, None, site, threshold)


def _dropout_launch(stream, x, threshold, seed, site):
  out = torch.empty_like(x, memory_format=torch.contiguous_format)
  status = _lib.lib().fwn_dropout(_drop_desc(threshold, seed, site), x.data_ptr(), out.data_ptr(), x.numel(), _CODE[x.dtype],
                                  stream)
  if status:
    _lib.check(status)
  return out


class _Dropout(torch.autograd.Function):
  """dropout; its gradient is the same function of the output's gradient (and so on). A seed on the device is saved, so that
  changing it between forward and backward raises torch's error for a tensor modified in place."""

  @staticmethod
  def forward(ctx, x, threshold, seed, site):
    ctx.threshold, ctx.site = threshold, site
    ctx.seed = None if isinstance(seed, torch.Tensor) else seed
    if ctx.seed is None:
      ctx.save_for_backward(seed)
    return _on_device(x, _dropout_launch, x.contiguous(), threshold, seed, site)

  @staticmethod
  def backward(ctx, dy):
    seed = ctx.saved_tensors[0] if ctx.seed is None else ctx.seed
    _no_tangent("dropout's gradient", dy)
    if torch.is_grad_enabled():  # a graph of the gradient is kept
      return _Dropout.apply(dy, ctx.threshold, seed, ctx.site), None, None, None
    return _on_device(dy, _dropout_launch, dy.contiguous(), ctx.threshold, seed, ctx.site), None, None, None


def dropout(x, p, seed, *, site=0):
  """x [...] float32 or bf16, each value 0 with probability p and multiplied by 1 / (1 - p) otherwise; a dropped value is 0
  whatever it was. The mask is a function of the seed, the site and the value's place in x (Philox4x32-10, 16 bits a value:
  p counts as the nearest multiple of 2^-16, and its factor with it), the same on every device and for every layout.

  seed: an int of 64 bits, or an int64 tensor of one number on x's device, read when the kernel runs: change it between
  steps (seed.add_(1)), also between a captured graph's replays, but not between a forward and its backward. site tells
  apart the masks of one step (the layer's number, say). Differentiable in x, any number of times (backward; forward mode
  raises NotImplementedError)."""
  _check("x", x, x, (_BF16, _F32))
  threshold = _drop_check(x, p, seed, site)
  _no_tangent("dropout", x)
  if torch.is_grad_enabled() and x.requires_grad:
    return _Dropout.apply(x, threshold, seed, site)
  return _on_device(x, _dropout_launch, x.contiguous(), threshold, seed, site)


# ---- the norms around a branch --------------------------------------------------------------------------------------

def _gate_rows(gate, x):
  """(gate as rows [gates, d], rows of x for each): gate [d], of x's shape, or with one row for all of x's last rows."""
  shape, xs = gate.shape, x.shape
  if shape == xs[-1:]:
    return gate, x.numel() // xs[-1]
  if shape == xs:
    return gate, 1
  if len(xs) >= 2 and (shape == xs[:-2] + xs[-1:] or shape == xs[:-2] + (1,) + xs[-1:]):
    return gate, xs[-2]
  raise ValueError(f"gate has shape {tuple(shape)}, expected ({xs[-1]},), x's {tuple(xs)} or one row for each {tuple(xs[:-2])}")


def _starts(t):
  """Whether t starts where 8 of its values are one access."""
  return t.data_ptr() % (8 * t.element_size()) == 0


def _plain(t):
  """t, or a copy: contiguous from an address where 8 values are one access."""
  if t is None or (t.is_contiguous() and _starts(t)):
    return t
  return t.clone(memory_format=torch.contiguous_format)


def _wide_or_plain(d, x, y):
  """(x, its row stride, y, its row stride): as they are where they are contiguous, or where every row of both allows wide
  accesses; else contiguous copies."""
  if x.is_contiguous() and y.is_contiguous() and _starts(x) and _starts(y):
    return x, d, y, d
  x2, y2 = _rows(x), _rows(y)
  if d % 8 == 0 and all(_starts(t) and (t.stride(0) % 8 == 0 or t.shape[0] == 1) for t in (x2, y2)):
    return x2, max(x2.stride(0), d), y2, max(y2.stride(0), d)
  return _plain(x2), d, _plain(y2), d


# Descriptors by their fields, of calls without dropout: a call's own time counts for single rows, and filling one takes 4 us.
_DESCS = {}


def _branch_desc(x, xs, y, ys, pw, w, gate, span, out_dtype, eps, scale, threshold, seed, site):
  d = x.shape[-1]
  fields = (x.numel() // d, xs, ys, span, d, _CODE[x.dtype], _CODE[y.dtype], 0 if pw is None else _CODE[pw.dtype],
            0 if w is None else _CODE[w.dtype], 0 if gate is None else _CODE[gate.dtype], _CODE[out_dtype], eps, scale, 0)
  if threshold:
    return _lib.BranchDesc(*fields, _drop_desc(threshold, seed, site))
  desc = _DESCS.get(fields)
  if desc is None:
    if len(_DESCS) >= 4096:
      _DESCS.clear()
    desc = _DESCS[fields] = _lib.BranchDesc(*fields)
  return desc


def _ptr(t):
  return None if t is None else t.data_ptr()


def _branch_launch(stream, x, xs, y, ys, pw, w, gate, span, out_dtype, eps, scale, threshold, seed, site, keep_rstd, shape):
  """(h, its scales or None, s, both roots of each row or None, the call's descriptor), h and s of x's shape."""
  s = x.new_empty(shape)
  h = x.new_empty(shape, dtype=out_dtype)
  h_scale = x.new_empty(shape[:-1], dtype=_F32) if out_dtype is _E4M3 else None
  rstd = x.new_empty((*shape[:-1], 2), dtype=_F32) if keep_rstd else None
  desc = _branch_desc(x, xs, y, ys, pw, w, gate, span, out_dtype, eps, scale, threshold, seed, site)
  status = _lib.lib().fwn_branch_norm(desc, x.data_ptr(), y.data_ptr(), _ptr(pw), _ptr(w), _ptr(gate), s.data_ptr(),
                                      h.data_ptr(), _ptr(h_scale), _ptr(rstd), stream)
  if status:
    _lib.check(status)
  return h, h_scale, s, rstd, desc


def _branch_forward(x, y, pw, w, gate, span, out_dtype, eps, scale, threshold=0, seed=None, site=0, keep_rstd=False):
  return _on_device(x, _branch_launch, *_wide_or_plain(x.shape[-1], x, y), _plain(pw), _plain(w), _plain(gate), span, out_dtype,
                    eps, scale, threshold, seed, site, keep_rstd, x.shape)


_BWD_BYTES = {}  # workspaces' sizes, which go by the shape alone


def _bwd_bytes(x, desc):
  key = (x.get_device(), desc.rows, desc.d, desc.gate_span)
  size = _BWD_BYTES.get(key)
  if size is None:
    need = ctypes.c_size_t(0)
    _lib.check(_lib.lib().fwn_branch_norm_bwd_workspace_size(desc, need))
    if len(_BWD_BYTES) >= 4096:
      _BWD_BYTES.clear()
    size = _BWD_BYTES[key] = need.value
  return size


class _BranchNorm(torch.autograd.Function):
  """branch_norm with gradients for x, y, the weights and the gate. The backward reads the inputs again (not the written,
  rounded stream) and the two reciprocal roots of each row, and makes the mask again."""

  @staticmethod
  def forward(ctx, x, y, pw, w, gate, seed, args):
    span, out_dtype, eps, scale, threshold, site = ctx.args = args
    ctx.seed = None if isinstance(seed, torch.Tensor) else seed
    h, _, s, rstd, ctx.desc = _branch_forward(x, y, pw, w, gate, span, out_dtype, eps, scale, threshold, seed, site, True)
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(x, y, pw, w, gate, rstd, seed if isinstance(seed, torch.Tensor) else None)
    return h, s

  @staticmethod
  def backward(ctx, dh, ds):
    x, y, pw, w, gate, rstd, seed = ctx.saved_tensors
    _no_tangent("branch_norm's gradient", x, y, pw, w, gate, dh, ds)
    if dh is None and ds is None:
      return (None,) * 7
    _first_order("branch_norm")
    grads = _on_device(x, _BranchNorm._launch, ctx, x, y, pw, w, gate, rstd, ctx.seed if seed is None else seed, dh, ds)
    return (*grads, None, None)

  @staticmethod
  def _launch(stream, ctx, x, y, pw, w, gate, rstd, seed, dh, ds):
    span, out_dtype, eps, scale, threshold, site = ctx.args
    need = ctx.needs_input_grad
    d = x.shape[-1]
    x2, xs, y2, ys = _wide_or_plain(d, x, y)
    pw2, w2, gate2, rstd, dh, ds = _plain(pw), _plain(w), _plain(gate), _plain(rstd), _plain(dh), _plain(ds)
    dx, dy, dpw, dw, dgate = [t.new_empty(t.shape) if wanted else None for t, wanted in zip((x, y, pw, w, gate), need)]
    if need[4] and x.numel() == 0:
      dgate.zero_()
    desc = ctx.desc  # the forward's, but where saved tensors came back in other places (hooks may move them)
    if isinstance(seed, torch.Tensor) or (desc.x_stride, desc.y_stride) != (xs, ys):
      desc = _branch_desc(x2, xs, y2, ys, pw, w, gate, span, out_dtype, eps, scale, threshold, seed, site)
    lib = _lib.lib()
    size = _bwd_bytes(x, desc)
    ws = x.new_empty((size,), dtype=torch.uint8) if size else None
    status = lib.fwn_branch_norm_bwd(desc, x2.data_ptr(), y2.data_ptr(), _ptr(pw2), _ptr(w2), _ptr(gate2), rstd.data_ptr(),
                                     _ptr(dh), _ptr(ds), _ptr(dx), _ptr(dy), _ptr(dpw), _ptr(dw), _ptr(dgate), _ptr(ws), size,
                                     stream)
    if status:
      _lib.check(status)
    return dx, dy, dpw, dw, dgate


def _branch_check(x, y, pw, w, gate, residual_scale, eps):
  if x.dim() < 1 or x.shape[-1] < 1:
    raise ValueError(f"x has shape {tuple(x.shape)}, expected [..., d] with d >= 1")
  if not eps >= 0:
    raise ValueError(f"eps must not be negative (got {eps})")
  _check("x", x, x, (_BF16, _F32))
  _check("y", y, x, (_BF16, _F32))
  if y.shape != x.shape:
    raise ValueError(f"y has shape {tuple(y.shape)}, expected {tuple(x.shape)}")
  for name, t in (("post_weight", pw), ("weight", w)):
    if t is not None:
      _check(name, t, x, (_BF16, _F32))
      if t.shape != x.shape[-1:]:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected ({x.shape[-1]},)")
  if not isinstance(residual_scale, (int, float)):
    raise TypeError(f"residual_scale is {residual_scale!r}, expected a number")
  rows = x.numel() // x.shape[-1]
  if gate is None:
    return None, max(rows, 1)
  _check("gate", gate, x, (_BF16, _F32))
  gate, span = _gate_rows(gate, x)
  return gate, max(span, 1)


def branch_norm(x, y, post_weight=None, weight=None, *, gate=None, residual_scale=1.0, p=0.0, seed=None, site=0, eps=1e-6,
                out_dtype=_BF16):
  """The end of one block and the beginning of the next: with norm(v) = v / sqrt(mean(v^2) + eps) over the last dimension,

      s = residual_scale x + dropout(gate norm(y) post_weight),   h = norm(s) weight.

  x, the residual stream, and y, the block's output, [..., d] float32 or bf16 (d <= 8,192, widths off multiples of 8 <=
  8,185); post_weight and weight [d] or None (ones); any strides. gate: None (ones), [d], one row for all of a sample's rows
  ([B, d] or [B, 1, d] for x [B, n, d]), or of x's shape. residual_scale is a number; p, seed and site are dropout's (seed
  is needed where p > 0). Sums are float32 and h is the norm of the unrounded s. Returns (h in out_dtype, bf16 or float32;
  s in x's dtype). Differentiable in x, y, the weights and the gate (backward, gradients in their dtypes; forward mode and
  second derivatives raise NotImplementedError)."""
  gate, span = _branch_check(x, y, post_weight, weight, gate, residual_scale, eps)
  if out_dtype is not _BF16 and out_dtype is not _F32:
    raise ValueError(f"out_dtype {out_dtype}: expected torch.bfloat16 or torch.float32")
  threshold = 0
  if p != 0:
    threshold = _drop_check(x, p, seed, site)
  if threshold == 0:
    seed = None
  _no_tangent("branch_norm", x, y, post_weight, weight, gate)
  if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, y, post_weight, weight, gate)):
    return _BranchNorm.apply(x, y, post_weight, weight, gate, seed, (span, out_dtype, eps, residual_scale, threshold, site))
  h, _, s, _, _ = _branch_forward(x, y, post_weight, weight, gate, span, out_dtype, eps, residual_scale, threshold, seed, site)
  return h, s


def branch_norm_fp8(x, y, post_weight=None, weight=None, *, gate=None, residual_scale=1.0, eps=1e-6):
  """branch_norm with h in 8 bits, the left operand of projection.linear_fp8: returns (values e4m3 [..., d], scale float32
  [...], s). scale = max |h| / 448 over the row, h = scale * values. Rows whose max |h| is below 2^-100 get scale 0 and
  values 0. No dropout and no gradient (forecasts): inputs that require one raise NotImplementedError."""
  gate, span = _branch_check(x, y, post_weight, weight, gate, residual_scale, eps)
  _constant("branch_norm_fp8", x, y, post_weight, weight, gate)
  return _branch_forward(x, y, post_weight, weight, gate, span, _E4M3, eps, residual_scale)[:3]
