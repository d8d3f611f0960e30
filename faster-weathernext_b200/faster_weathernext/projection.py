"""Pre-norm projections: the root-mean-square norm with the residual's addition and the projection with bias, activation
and residual in its epilogue, in bf16 with gradients and in 8 bits for forecasts.

    h, x = rms_norm(x, weight, residual=a)                 # x += a, h = rms norm of the sum (differentiable)
    y = linear(h, w, bias, activation="gelu")              # GELU(h w^T + bias) (differentiable)
    x = linear(y, w2, bias2, residual=x, out_dtype=x.dtype)

    values, scale, x = rms_norm_fp8(x, weight, residual=a) # h in e4m3 with one scale per row
    y = linear_fp8(values, scale, w8, w8_scale, bias, activation="gelu")   # w8, w8_scale = quantize_fp8(w), kept

No counterpart in the reference, whose blocks use LayerNorm and plain projections (src/faster_weathernext/patch.py:
165-177, 238-252): this is the same sub-block in the form of later transformers. The kernels are csrc/rms.cu and
csrc/linear.cu (C ABI in include/fwn_attn.h, fwn_rms_norm* and fwn_linear*). Every call runs on the current stream of
its tensors' device and takes its workspace from torch's allocator.
"""

import ctypes

import torch
from torch.autograd import forward_ad

from faster_weathernext import _lib

_BF16, _F32, _E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
_CODE = {_BF16: _lib.DTYPE_BF16, _F32: _lib.DTYPE_F32, _E4M3: _lib.DTYPE_E4M3}
_ACT = {None: _lib.ACT_NONE, "gelu": _lib.ACT_GELU_TANH, "swish": _lib.ACT_SWISH}


# The current device and its current stream's handle, without the Python objects around them (a call's own time counts
# for single rows).
_device_now = torch._C._cuda_getDevice
_stream_of = torch._C._cuda_getCurrentRawStream


def _check(name, t, like, dtypes):
  if t.dtype in dtypes and t.is_cuda and t.get_device() == like.get_device():
    return
  if t.dtype not in dtypes:
    raise TypeError(f"{name} has dtype {t.dtype}, expected one of {[str(d) for d in dtypes]}")
  if not t.is_cuda or t.device != like.device:
    raise ValueError(f"{name} is on {t.device}, expected the CUDA device of the first argument ({like.device})")


def _constant(name, *tensors):
  """Refuses inputs of a function without gradients that ask for one: its result would be cut off from them unnoticed."""
  if torch.is_grad_enabled():
    for t in tensors:
      if t is not None and t.requires_grad:
        raise NotImplementedError(f"{name} has no gradient (forecasts): call it under torch.no_grad() or on detached tensors")
  _no_tangent(name, *tensors)


def _no_tangent(name, *tensors):
  """Refuses inputs with a forward-mode tangent, which the kernels would lose (they have backward gradients only)."""
  if forward_ad._current_level < 0:  # outside every dual_level, as unpack_dual looks it up, without its call for each
    return
  for t in tensors:
    if t is not None and forward_ad.unpack_dual(t).tangent is not None:
      raise NotImplementedError(f"{name} has no forward-mode derivative")


def _first_order(name):
  """Refuses a backward that keeps a graph (create_graph=True): the kernels' gradients would be constants in it, and second
  derivatives would lack their terms unnoticed. (A node that raises when it is differentiated would not do: autograd.grad
  skips nodes that lead to none of its inputs.)"""
  if torch.is_grad_enabled():
    raise NotImplementedError(f"{name} has no second derivative: take its gradient without create_graph=True")


def _rows(t):
  """t as [rows, d] with d contiguous and rows that do not overlap: a view where the strides allow it, else a copy."""
  if t.is_contiguous():
    if t.dim() == 2:
      return t
  d = t.shape[-1]
  if t.dim() != 2:
    t = t.reshape(t.numel() // d, d)
  if (t.stride(1) != 1 and d > 1) or (t.stride(0) < d and t.shape[0] > 1):
    t = t.contiguous()
  return t


def _on_device(t, call, *args):
  """call(stream handle, *args) with t's device current: launches and allocations go there."""
  i = t.get_device()
  if i == _device_now():
    return call(_stream_of(i), *args)
  with torch.cuda.device(i):
    return call(_stream_of(i), *args)


# ---- rms_norm -------------------------------------------------------------------------------------------------------

def _rms_check(x, weight, residual, eps):
  if x.dim() < 1 or x.shape[-1] < 1:
    raise ValueError(f"x has shape {tuple(x.shape)}, expected [..., d] with d >= 1")
  if not eps >= 0:
    raise ValueError(f"eps must not be negative (got {eps})")
  _check("x", x, x, (_BF16, _F32))
  if residual is not None:
    _check("residual", residual, x, (_BF16, _F32))
    if residual.shape != x.shape:
      raise ValueError(f"residual has shape {tuple(residual.shape)}, expected {tuple(x.shape)}")
  if weight is not None:
    _check("weight", weight, x, (_BF16, _F32))
    if weight.shape != x.shape[-1:]:
      raise ValueError(f"weight has shape {tuple(weight.shape)}, expected ({x.shape[-1]},)")


def _rms_launch(stream, x, weight, residual, eps, out_dtype, flags):
  rows, d = x.shape
  out = x.new_empty((rows, d), dtype=out_dtype)
  scale = x.new_empty((rows,), dtype=_F32) if out_dtype is _E4M3 else None
  x_new = None if residual is None else x.new_empty((rows, d))
  desc = _lib.RmsDesc(rows, d, _CODE[x.dtype], 0 if residual is None else _CODE[residual.dtype],
                      0 if weight is None else _CODE[weight.dtype], _CODE[out_dtype], flags, eps, 0, x.stride(0),
                      0 if residual is None else residual.stride(0))
  status = _lib.lib().fwn_rms_norm(desc, x.data_ptr(), None if residual is None else residual.data_ptr(),
                                   None if weight is None else weight.data_ptr(),
                                   None if x_new is None else x_new.data_ptr(), out.data_ptr(),
                                   None if scale is None else scale.data_ptr(), stream)
  if status:
    _lib.check(status)
  return out, scale, x_new


def _rms_forward(x, weight, residual, eps, out_dtype, flags=0):
  """(h, scale or None, x_new or None) in x's shape."""
  x2 = _rows(x)
  if weight is not None and not weight.is_contiguous():
    weight = weight.contiguous()
  h, scale, x_new = _on_device(x, _rms_launch, x2, weight, None if residual is None else _rows(residual), eps, out_dtype,
                               flags)
  if x.dim() != 2:
    h = h.view(x.shape)
    scale = None if scale is None else scale.view(x.shape[:-1])
    x_new = None if x_new is None else x_new.view(x.shape)
  return h, scale, x_new


class _RmsNorm(torch.autograd.Function):
  """rms_norm with gradients for x, weight and residual. What the backward normalises again: the float32 sum, which the
  forward wrote, or a bf16 stream's own inputs (its written sum is rounded, and the gradients are of the unrounded)."""

  @staticmethod
  def forward(ctx, x, weight, residual, eps, out_dtype):
    h, _, x_new = _rms_forward(x, weight, residual, eps, out_dtype)
    ctx.eps = eps
    ctx.residual_dtype = None if residual is None else residual.dtype
    ctx.set_materialize_grads(False)
    if residual is None:
      ctx.save_for_backward(x, weight, None)
      return h
    if x.dtype is _F32:
      ctx.save_for_backward(x_new, weight, None)
    else:
      ctx.save_for_backward(x, weight, residual)
    return h, x_new

  @staticmethod
  def backward(ctx, dh, ds=None):
    x, w, r = ctx.saved_tensors
    _no_tangent("rms_norm's gradient", x, w, r, dh, ds)
    need_x, need_w, need_r = ctx.needs_input_grad[:3]
    if dh is None:
      # Only the stored sum was used: its gradient passes through.
      if ds is None:
        return None, None, None, None, None
      return (ds if need_x else None, torch.zeros_like(w) if need_w else None,
              ds.to(ctx.residual_dtype) if need_r else None, None, None)
    _first_order("rms_norm")
    dx, dw, dr = _on_device(x, _RmsNorm._launch, ctx, x, w, r, dh, ds, need_x, need_w, need_r)
    return dx, dw, dr, None, None

  @staticmethod
  def _launch(stream, ctx, x, w, r, dh, ds, need_x, need_w, need_r):
    shape = x.shape
    x = _rows(x)
    r = None if r is None else _rows(r)
    w = None if w is None else w.contiguous()
    rows, d = x.shape
    dh = dh.contiguous()
    ds = None if ds is None else ds.contiguous()
    dx = x.new_empty(shape) if need_x else None
    dr = x.new_empty(shape, dtype=ctx.residual_dtype) if need_r else None
    dw = torch.empty_like(w) if need_w else None
    desc = _lib.RmsDesc(rows, d, _CODE[x.dtype], 0 if ctx.residual_dtype is None else _CODE[ctx.residual_dtype],
                        0 if w is None else _CODE[w.dtype], _CODE[dh.dtype], 0, ctx.eps, 0, x.stride(0),
                        0 if r is None else r.stride(0))
    lib = _lib.lib()
    ws, size = _workspace(x, desc, lib.fwn_rms_norm_bwd_workspace_size) if need_w else (None, 0)
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    _lib.check(lib.fwn_rms_norm_bwd(desc, x.data_ptr(), ptr(r), ptr(w), dh.data_ptr(), ptr(ds), ptr(dx), ptr(dr), ptr(dw),
                                    ptr(ws), size, stream))
    return dx, dw, dr


def rms_norm(x, weight=None, residual=None, *, eps=1e-6, out_dtype=_BF16):
  """h = s / sqrt(mean(s^2) + eps) * weight over the last dimension, s = x + residual (or x).

  x [..., d] float32 or bf16 (d <= 16,384), residual of x's shape, weight [d], each float32 or bf16; any strides. Sums
  are float32. Returns h in out_dtype (bf16 or float32), or, with a residual, (h, s) with s in x's dtype: the residual
  stream after the addition. Differentiable in x, weight and residual (backward, gradients in their dtypes; forward mode
  and second derivatives raise NotImplementedError)."""
  _rms_check(x, weight, residual, eps)
  _no_tangent("rms_norm", x, weight, residual)
  if out_dtype is not _BF16 and out_dtype is not _F32:
    raise ValueError(f"out_dtype {out_dtype}: expected torch.bfloat16 or torch.float32")
  if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or
                                  (residual is not None and residual.requires_grad)):
    return _RmsNorm.apply(x, weight, residual, eps, out_dtype)
  h, _, x_new = _rms_forward(x, weight, residual, eps, out_dtype)
  return h if residual is None else (h, x_new)


def rms_norm_fp8(x, weight=None, residual=None, *, eps=1e-6):
  """rms_norm with h in 8 bits, the left operand of linear_fp8: returns (values e4m3 [..., d], scale float32 [...]), or,
  with a residual, (values, scale, s). scale = max |h| / 448 over the row, h = scale * values. Rows whose max |h| is
  below 2^-100 get scale 0 and values 0. No gradient (forecasts): inputs that require one raise NotImplementedError."""
  _rms_check(x, weight, residual, eps)
  _constant("rms_norm_fp8", x, weight, residual)
  h, scale, x_new = _rms_forward(x, weight, residual, eps, _E4M3)
  return (h, scale) if residual is None else (h, scale, x_new)


def quantize_fp8(t):
  """Rows of t [..., k] (float32 or bf16) in 8 bits: (values e4m3 [..., k], scale float32 [...]) as rms_norm_fp8's. The
  form linear_fp8 takes a weight [n, k] in; computed once and kept, a constant whatever t requires."""
  _rms_check(t, None, None, 0.0)
  return _rms_forward(t, None, None, 0.0, _E4M3, _lib.RMS_SCALE_ONLY)[:2]


# ---- linear ---------------------------------------------------------------------------------------------------------

def _orient(t):
  """(tensor, row stride, transposed): t [r, c] with c contiguous, or with r contiguous (a transposed view); a copy of a
  tensor with neither."""
  r, c = t.shape
  s0, s1 = t.stride()
  if (s1 == 1 or c == 1) and (s0 >= c or r == 1):
    return t, max(s0, c), False
  if (s0 == 1 or r == 1) and (s1 >= r or c == 1):
    return t, max(s1, r), True
  return t.contiguous(), c, False


def _padded(t):
  """t, or a copy of t [r, c] in its own order with rows of whole 16 bytes, which TMA can address: an operand of three
  products (odd widths) is laid out once instead of by each."""
  src, ld, turned = _orient(t)
  rows, cols = (src.shape[1], src.shape[0]) if turned else src.shape
  if (ld % 8 == 0 and src.data_ptr() % 16 == 0) or rows <= 8:
    return t
  out = src.new_empty((rows, -(-cols // 8) * 8))
  _lib.check(_on_device(src, _pack_launch, src, ld, out, rows, cols))
  out = out[:, :cols]
  return out.t() if turned else out


def _pack_launch(stream, src, ld, out, rows, cols):
  return _lib.lib().fwn_linear_pack(src.data_ptr(), ld, out.data_ptr(), out.shape[1], rows, cols, _lib.DTYPE_BF16, stream)


# Workspace bytes by a call's device (its number of SMs counts), shape, types, strides and the alignment of its operands
# (asked once for each).
_WORKSPACE = {}


def _workspace(like, desc, size_of, *ptrs):
  """(tensor or None, bytes) that `size_of` wants for a call with these operands."""
  key = (like.get_device(), bytes(desc), *[p & 15 for p in ptrs])
  size = _WORKSPACE.get(key)
  if size is None:
    need = ctypes.c_size_t(0)
    _lib.check(size_of(desc, *ptrs, need))
    if len(_WORKSPACE) >= 4096:
      _WORKSPACE.clear()
    size = _WORKSPACE[key] = need.value
  return like.new_empty((size,), dtype=torch.uint8) if size else None, size


def _forward_launch(stream, a, b, bias, x, act, out_dtype, a_scale=None, b_scale=None):
  """act(a b^T + bias) + x for 2D a [m, k], b [n, k] in either orientation."""
  m, k = a.shape
  n = b.shape[0]
  dtype = a.dtype
  a, lda, a_t = _orient(a)
  b, ldb, b_t = _orient(b)
  if dtype is _E4M3:
    if a_t:
      a, lda, a_t = a.contiguous(), k, False
    if b_t:
      b, ldb, b_t = b.contiguous(), k, False
  out = a.new_empty((m, n), dtype=out_dtype)
  flags = (_lib.LINEAR_A_M_CONTIGUOUS if a_t else 0) | (_lib.LINEAR_B_N_CONTIGUOUS if b_t else 0)
  ap, bp = a.data_ptr(), b.data_ptr()
  desc = _lib.LinearDesc(m, n, k, _CODE[dtype], _CODE[out_dtype], 0 if bias is None else _CODE[bias.dtype],
                         0 if x is None else _CODE[x.dtype], act, flags, lda, ldb,
                         0 if x is None else max(x.stride(0), n), n)
  lib = _lib.lib()
  ws, size = _workspace(a, desc, lib.fwn_linear_workspace_size, ap, bp)
  status = lib.fwn_linear(desc, ap, None if a_scale is None else a_scale.data_ptr(), bp,
                          None if b_scale is None else b_scale.data_ptr(), None if bias is None else bias.data_ptr(),
                          None if x is None else x.data_ptr(), out.data_ptr(), None,
                          None if ws is None else ws.data_ptr(), size, stream)
  if status:
    _lib.check(status)
  return out


class _Linear(torch.autograd.Function):
  """linear with gradients. The backward (fwn_linear_bwd) recomputes the pre-activation inside the product that turns dy
  into its gradient (x act'(a w^T + bias), with the bias gradient's column sums), then takes d_a = d_pre w and
  d_weight = d_pre^T a on the same kernel; the residual's gradient is dy."""

  @staticmethod
  def forward(ctx, a, weight, bias, residual, act, out_dtype):
    ctx.act, ctx.shape = act, a.shape
    a2, w2 = _padded(_rows(a)), _padded(weight)
    if bias is not None and not bias.is_contiguous():
      bias = bias.contiguous()
    ctx.save_for_backward(a2, w2, bias)
    y = _on_device(a2, _forward_launch, a2, w2, bias, None if residual is None else _rows(residual), act, out_dtype)
    return y if a.dim() == 2 else y.view(*a.shape[:-1], weight.shape[0])

  @staticmethod
  def backward(ctx, dy):
    a, weight, bias = ctx.saved_tensors
    _no_tangent("linear's gradient", a, weight, bias, dy)
    need_a, need_w, need_b, need_r = ctx.needs_input_grad[:4]
    d_a = d_w = d_b = None
    if a.shape[0] == 0:
      d_a = a.new_zeros(ctx.shape) if need_a else None
      d_w = torch.zeros_like(weight) if need_w else None
      d_b = torch.zeros_like(bias) if need_b else None
    elif need_a or need_w or need_b:
      _first_order("linear")
      d_a, d_w, d_b = _on_device(a, _Linear._launch, a, weight, bias, ctx.act,
                                 _rows(dy if dy.dim() == 2 else dy.reshape(a.shape[0], -1)), need_a, need_w, need_b)
      if need_a and len(ctx.shape) != 2:
        d_a = d_a.view(ctx.shape)
    return d_a, d_w, d_b, dy if need_r else None, None, None

  @staticmethod
  def _launch(stream, a, weight, bias, act, dy, need_a, need_w, need_b):
    m, k = a.shape
    n = weight.shape[0]
    a, lda, a_t = _orient(a)
    b, ldb, b_t = _orient(weight)
    d_a = a.new_empty((m, k)) if need_a else None
    d_w = a.new_empty((k, n) if b_t else (n, k)) if need_w else None
    d_b = torch.empty_like(bias) if need_b else None
    flags = (_lib.LINEAR_A_M_CONTIGUOUS if a_t else 0) | (_lib.LINEAR_B_N_CONTIGUOUS if b_t else 0)
    ap, bp, dp = a.data_ptr(), b.data_ptr(), dy.data_ptr()
    desc = _lib.LinearDesc(m, n, k, _lib.DTYPE_BF16, _CODE[dy.dtype], 0 if bias is None else _CODE[bias.dtype],
                           _CODE[dy.dtype], act, flags, lda, ldb, max(dy.stride(0), n), n)
    lib = _lib.lib()
    ws, size = _workspace(a, desc, lib.fwn_linear_bwd_workspace_size, ap, bp, dp)
    status = lib.fwn_linear_bwd(desc, ap, bp, None if bias is None else bias.data_ptr(), dp,
                                None if d_a is None else d_a.data_ptr(), None if d_w is None else d_w.data_ptr(),
                                None if d_b is None else d_b.data_ptr(), None if ws is None else ws.data_ptr(), size, stream)
    if status:
      _lib.check(status)
    return d_a, d_w.t() if b_t and need_w else d_w, d_b


def _linear_forward(a, weight, bias, residual, act, out_dtype, a_scale=None, b_scale=None):
  if bias is not None and not bias.is_contiguous():
    bias = bias.contiguous()
  out = _on_device(a, _forward_launch, _rows(a), weight, bias, None if residual is None else _rows(residual), act, out_dtype,
                   a_scale, b_scale)
  return out if a.dim() == 2 else out.view(*a.shape[:-1], weight.shape[0])


def _linear_check(a, weight, bias, residual, activation, out_dtype, dtype):
  if a.dim() < 1 or weight.dim() != 2 or a.shape[-1] != weight.shape[1] or weight.shape[0] < 1 or weight.shape[1] < 1:
    raise ValueError(f"a has shape {tuple(a.shape)} and weight {tuple(weight.shape)}, expected [..., k] and [n, k], "
                     "n, k >= 1")
  n = weight.shape[0]
  _check("a", a, a, (dtype,))
  _check("weight", weight, a, (dtype,))
  if activation not in _ACT:
    raise ValueError(f"activation {activation!r}: expected None, 'gelu' or 'swish'")
  if out_dtype is not _BF16 and out_dtype is not _F32:
    raise ValueError(f"out_dtype {out_dtype}: expected torch.bfloat16 or torch.float32")
  if bias is not None:
    _check("bias", bias, a, (_BF16, _F32))
    if bias.dim() != 1 or bias.shape[0] != n:
      raise ValueError(f"bias has shape {tuple(bias.shape)}, expected ({n},)")
  if residual is not None:
    _check("residual", residual, a, (out_dtype,))
    if residual.dim() != a.dim() or residual.shape[-1] != n or residual.shape[:-1] != a.shape[:-1]:
      raise ValueError(f"residual has shape {tuple(residual.shape)}, expected {tuple(a.shape[:-1]) + (n,)}")


def linear(a, weight, bias=None, residual=None, *, activation=None, out_dtype=_BF16):
  """act(a weight^T + bias) + residual in one kernel: a [..., k] and weight [n, k] bf16, bias [n] bf16 or float32,
  residual [..., n] in out_dtype (bf16 or float32), activation None, "gelu" (tanh form) or "swish"; float32
  accumulation, rounded once (in the backward so is the gradient of the pre-activation, to bf16: the operand of the
  products for a's and weight's). weight may be the transposed view of a [k, n] tensor (either orientation is read in
  place); rows of any stride. Differentiable in a, weight, bias and residual (backward, gradients in their dtypes;
  forward mode and second derivatives raise NotImplementedError)."""
  _linear_check(a, weight, bias, residual, activation, out_dtype, _BF16)
  _no_tangent("linear", a, weight, bias, residual)
  act = _ACT[activation]
  if torch.is_grad_enabled() and (a.requires_grad or weight.requires_grad or
                                  (bias is not None and bias.requires_grad) or
                                  (residual is not None and residual.requires_grad)):
    return _Linear.apply(a, weight, bias, residual, act, out_dtype)
  return _linear_forward(a, weight, bias, residual, act, out_dtype)


def linear_fp8(a, a_scale, weight, weight_scale, bias=None, residual=None, *, activation=None, out_dtype=_BF16):
  """linear on 8-bit operands: act((a weight^T) a_scale weight_scale + bias) + residual, a [..., k] and weight [n, k]
  e4m3 with float32 scales per row (a_scale [...], weight_scale [n]), as rms_norm_fp8 and quantize_fp8 give them. No
  gradient (forecasts): inputs that require one raise NotImplementedError."""
  _linear_check(a, weight, bias, residual, activation, out_dtype, _E4M3)
  _check("a_scale", a_scale, a, (_F32,))
  _check("weight_scale", weight_scale, a, (_F32,))
  if a_scale.shape != a.shape[:-1]:
    raise ValueError(f"a_scale has shape {tuple(a_scale.shape)}, expected {tuple(a.shape[:-1])}")
  if weight_scale.shape != weight.shape[:1]:
    raise ValueError(f"weight_scale has shape {tuple(weight_scale.shape)}, expected ({weight.shape[0]},)")
  _constant("linear_fp8", a, a_scale, weight, weight_scale, bias, residual)
  return _linear_forward(a, weight, bias, residual, _ACT[activation], out_dtype, a_scale.contiguous(),
                         weight_scale.contiguous())
