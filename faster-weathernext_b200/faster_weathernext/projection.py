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

from faster_weathernext import _lib

_BF16, _F32, _E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
_CODE = {_BF16: _lib.DTYPE_BF16, _F32: _lib.DTYPE_F32, _E4M3: _lib.DTYPE_E4M3}
_ACT = {None: _lib.ACT_NONE, "gelu": _lib.ACT_GELU_TANH, "swish": _lib.ACT_SWISH}


def _ptr(t):
  return None if t is None else t.data_ptr()


def _need(ok, message):
  if not ok:
    raise ValueError(message)


def _check(name, t, like, dtypes):
  if t.dtype not in dtypes:
    raise TypeError(f"{name} has dtype {t.dtype}, expected one of {[str(d) for d in dtypes]}")
  if not t.is_cuda or t.device != like.device:
    raise ValueError(f"{name} is on {t.device}, expected the CUDA device of the first argument ({like.device})")


def _rows(t):
  """t as [rows, d] with d contiguous and rows that do not overlap: a view where the strides allow it, else a copy."""
  d = t.shape[-1]
  if t.dim() != 2:
    t = t.reshape(t.numel() // d, d)
  if (t.stride(1) != 1 and d > 1) or (t.stride(0) < d and t.shape[0] > 1):
    t = t.contiguous()
  return t


class _Device:
  """Makes the tensors' device current for the duration of a call (the launches and the allocations go there)."""

  def __init__(self, t):
    self.guard = None if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)

  def __enter__(self):
    if self.guard is not None:
      self.guard.__enter__()
    return torch.cuda.current_stream().cuda_stream

  def __exit__(self, *exc):
    if self.guard is not None:
      self.guard.__exit__(*exc)


# ---- rms_norm -------------------------------------------------------------------------------------------------------

def _rms_desc(x, residual, weight, out_dtype, eps, flags=0):
  rows, d = x.shape
  return _lib.RmsDesc(rows, d, _CODE[x.dtype], _CODE[residual.dtype] if residual is not None else 0,
                      _CODE[weight.dtype] if weight is not None else 0, _CODE[out_dtype], flags, eps, 0,
                      x.stride(0), residual.stride(0) if residual is not None else 0)


def _rms_check(x, weight, residual, eps):
  _need(x.dim() >= 1 and x.shape[-1] >= 1, f"x has shape {tuple(x.shape)}, expected [..., d] with d >= 1")
  _need(eps >= 0, f"eps must not be negative (got {eps})")
  _check("x", x, x, (_BF16, _F32))
  if residual is not None:
    _check("residual", residual, x, (_BF16, _F32))
    _need(residual.shape == x.shape, f"residual has shape {tuple(residual.shape)}, expected {tuple(x.shape)}")
  if weight is not None:
    _check("weight", weight, x, (_BF16, _F32))
    _need(weight.shape == x.shape[-1:], f"weight has shape {tuple(weight.shape)}, expected ({x.shape[-1]},)")


def _rms_forward(x, weight, residual, eps, out_dtype, flags=0):
  """(h, scale or None, x_new or None) over 2D rows."""
  with _Device(x) as stream:
    out = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    scale = torch.empty(x.shape[0], dtype=_F32, device=x.device) if out_dtype == _E4M3 else None
    x_new = torch.empty(x.shape, dtype=x.dtype, device=x.device) if residual is not None else None
    desc = _rms_desc(x, residual, weight, out_dtype, eps, flags)
    _lib.check(_lib.lib().fwn_rms_norm(ctypes.byref(desc), x.data_ptr(), _ptr(residual), _ptr(weight), _ptr(x_new),
                                       out.data_ptr(), _ptr(scale), stream))
  return out, scale, x_new


class _RmsNorm(torch.autograd.Function):
  """rms_norm with gradients for x, weight and residual. What the backward normalises again: the float32 sum, which the
  forward wrote, or a bf16 stream's own inputs (its written sum is rounded, and the gradients are of the unrounded)."""

  @staticmethod
  def forward(ctx, x, weight, residual, eps, out_dtype):
    x2 = _rows(x)
    r2 = None if residual is None else _rows(residual)
    w = None if weight is None else weight.contiguous()
    h, _, x_new = _rms_forward(x2, w, r2, eps, out_dtype)
    ctx.eps, ctx.shape = eps, x.shape
    ctx.residual_dtype = None if residual is None else residual.dtype
    ctx.set_materialize_grads(False)
    if residual is None:
      ctx.save_for_backward(x2, w, None)
      return h.view(x.shape)
    if x.dtype == _F32:
      ctx.save_for_backward(x_new, w, None)
    else:
      ctx.save_for_backward(x2, w, r2)
    return h.view(x.shape), x_new.view(x.shape)

  @staticmethod
  def backward(ctx, dh, ds=None):
    x, w, r = ctx.saved_tensors
    rows, d = x.shape
    need_x, need_w, need_r = ctx.needs_input_grad[:3]
    if dh is None:
      # Only the stored sum was used: its gradient passes through.
      if ds is None:
        return None, None, None, None, None
      return (ds if need_x else None, torch.zeros_like(w) if need_w else None,
              ds.to(ctx.residual_dtype) if need_r else None, None, None)
    with _Device(x) as stream:
      dh = dh.reshape(rows, d).contiguous()
      ds = None if ds is None else ds.reshape(rows, d).contiguous()
      dx = torch.empty(rows, d, dtype=x.dtype, device=x.device) if need_x else None
      dr = torch.empty(rows, d, dtype=ctx.residual_dtype, device=x.device) if need_r else None
      dw = torch.empty_like(w) if need_w else None
      desc = _rms_desc(x, r, w, dh.dtype, ctx.eps)
      if ctx.residual_dtype is not None:
        desc.residual_dtype = _CODE[ctx.residual_dtype]
      lib, ws, size = _lib.lib(), None, ctypes.c_size_t(0)
      if need_w:
        _lib.check(lib.fwn_rms_norm_bwd_workspace_size(ctypes.byref(desc), ctypes.byref(size)))
        ws = torch.empty(size.value, dtype=torch.uint8, device=x.device)
      _lib.check(lib.fwn_rms_norm_bwd(ctypes.byref(desc), x.data_ptr(), _ptr(r), _ptr(w), dh.data_ptr(), _ptr(ds),
                                      _ptr(dx), _ptr(dr), _ptr(dw), _ptr(ws), size.value, stream))
    return (None if dx is None else dx.view(ctx.shape), dw, None if dr is None else dr.view(ctx.shape), None, None)


def rms_norm(x, weight=None, residual=None, *, eps=1e-6, out_dtype=_BF16):
  """h = s / sqrt(mean(s^2) + eps) * weight over the last dimension, s = x + residual (or x).

  x [..., d] float32 or bf16 (d <= 16,384), residual of x's shape, weight [d], each float32 or bf16; any strides. Sums
  are float32. Returns h in out_dtype (bf16 or float32), or, with a residual, (h, s) with s in x's dtype: the residual
  stream after the addition. Differentiable in x, weight and residual (gradients in their dtypes)."""
  _rms_check(x, weight, residual, eps)
  _need(out_dtype in (_BF16, _F32), f"out_dtype {out_dtype}: expected torch.bfloat16 or torch.float32")
  if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or
                                  (residual is not None and residual.requires_grad)):
    return _RmsNorm.apply(x, weight, residual, eps, out_dtype)
  h, _, x_new = _rms_forward(_rows(x), None if weight is None else weight.contiguous(),
                             None if residual is None else _rows(residual), eps, out_dtype)
  return h.view(x.shape) if residual is None else (h.view(x.shape), x_new.view(x.shape))


def rms_norm_fp8(x, weight=None, residual=None, *, eps=1e-6):
  """rms_norm with h in 8 bits, the left operand of linear_fp8: returns (values e4m3 [..., d], scale float32 [...]), or,
  with a residual, (values, scale, s). scale = max |h| / 448 over the row, h = scale * values. Rows whose max |h| is
  below 2^-100 get scale 0 and values 0. Not differentiable (forecasts)."""
  _rms_check(x, weight, residual, eps)
  h, scale, x_new = _rms_forward(_rows(x), None if weight is None else weight.contiguous(),
                                 None if residual is None else _rows(residual), eps, _E4M3)
  out = (h.view(x.shape), scale.view(x.shape[:-1]))
  return out if residual is None else out + (x_new.view(x.shape),)


def quantize_fp8(t):
  """Rows of t [..., k] (float32 or bf16) in 8 bits: (values e4m3 [..., k], scale float32 [...]) as rms_norm_fp8's. The
  form linear_fp8 takes a weight [n, k] in; computed once and kept."""
  _rms_check(t, None, None, 0.0)
  h, scale, _ = _rms_forward(_rows(t), None, None, 0.0, _E4M3, _lib.RMS_SCALE_ONLY)
  return h.view(t.shape), scale.view(t.shape[:-1])


# ---- linear ---------------------------------------------------------------------------------------------------------

def _orient(t):
  """(tensor, row stride, transposed): t [r, c] with c contiguous, or with r contiguous (a transposed view); a copy of a
  tensor with neither."""
  r, c = t.shape
  if (t.stride(1) == 1 or c == 1) and (t.stride(0) >= c or r == 1):
    return t, max(t.stride(0), c), False
  if (t.stride(0) == 1 or r == 1) and (t.stride(1) >= r or c == 1):
    return t, max(t.stride(1), r), True
  t = t.contiguous()
  return t, c, False


def _product(a, b, bias, x, act, out_dtype, *, a_scale=None, b_scale=None, pre_grad=False, d_bias=None, pad=False):
  """act(a b^T + bias) + x for 2D a [m, k], b [n, k] in either orientation; pre_grad: x act'(a b^T + bias) with d_bias's
  column sums. pad: the output's row stride is rounded up to 16 bytes (an operand of the next product)."""
  m, k = a.shape
  n = b.shape[0]
  with _Device(a) as stream:
    a, lda, a_t = _orient(a)
    b, ldb, b_t = _orient(b)
    if a.dtype == _E4M3:
      if a_t:
        a, lda, a_t = a.contiguous(), k, False
      if b_t:
        b, ldb, b_t = b.contiguous(), k, False
    if x is not None:
      x = _rows(x)
    if pad and n % 8:
      out = torch.empty(m, -(-n // 8) * 8, dtype=out_dtype, device=a.device)[:, :n]
    else:
      out = torch.empty(m, n, dtype=out_dtype, device=a.device)
    flags = ((_lib.LINEAR_A_M_CONTIGUOUS if a_t else 0) | (_lib.LINEAR_B_N_CONTIGUOUS if b_t else 0) |
             (_lib.LINEAR_PRE_GRAD if pre_grad else 0))
    desc = _lib.LinearDesc(m, n, k, _CODE[a.dtype], _CODE[out_dtype], _CODE[bias.dtype] if bias is not None else 0,
                           _CODE[x.dtype] if x is not None else 0, act, flags, lda, ldb,
                           max(x.stride(0), n) if x is not None else 0, max(out.stride(0), n))
    lib, size = _lib.lib(), ctypes.c_size_t(0)
    ref = ctypes.byref(desc)
    _lib.check(lib.fwn_linear_workspace_size(ref, a.data_ptr(), b.data_ptr(), ctypes.byref(size)))
    ws = torch.empty(size.value, dtype=torch.uint8, device=a.device) if size.value else None
    _lib.check(lib.fwn_linear(ref, a.data_ptr(), _ptr(a_scale), b.data_ptr(), _ptr(b_scale), _ptr(bias), _ptr(x),
                              out.data_ptr(), _ptr(d_bias), _ptr(ws), size.value, stream))
  return out


def _pre_gradient(a, weight, bias, act, dy, need_bias):
  """(gradient of the pre-activation in bf16, gradient of the bias or None) for dy [m, n]."""
  m, n = dy.shape
  d_bias = torch.empty_like(bias) if need_bias else None
  if act != _lib.ACT_NONE:
    return _product(a, weight, bias, dy, act, _BF16, pre_grad=True, d_bias=d_bias, pad=True), d_bias
  dy = _rows(dy)
  cast = None
  if dy.dtype != _BF16:
    cast = torch.empty(m, -(-n // 8) * 8, dtype=_BF16, device=dy.device)[:, :n]
  if cast is not None or need_bias:
    with _Device(dy) as stream:
      lib, size = _lib.lib(), ctypes.c_size_t(0)
      _lib.check(lib.fwn_linear_grad_cast_workspace_size(m, n, ctypes.byref(size)))
      ws = torch.empty(max(size.value, 16), dtype=torch.uint8, device=dy.device) if need_bias else None
      _lib.check(lib.fwn_linear_grad_cast(dy.data_ptr(), _CODE[dy.dtype], max(dy.stride(0), n), m, n, _ptr(cast),
                                          cast.stride(0) if cast is not None else 0, _ptr(d_bias),
                                          _CODE[bias.dtype] if bias is not None else 0, _ptr(ws), size.value, stream))
  return dy if cast is None else cast, d_bias


class _Linear(torch.autograd.Function):
  """linear with gradients. The backward recomputes the pre-activation inside the product that turns dy into its
  gradient (x act'(a w^T + bias), with the bias gradient's column sums), then takes d_a = d_pre w and
  d_weight = d_pre^T a on the same kernel; the residual's gradient is dy."""

  @staticmethod
  def forward(ctx, a, weight, bias, residual, act, out_dtype):
    a2 = _rows(a)
    r2 = None if residual is None else _rows(residual)
    b1 = None if bias is None else bias.contiguous()
    ctx.act, ctx.shape = act, a.shape
    ctx.save_for_backward(a2, weight, b1)
    return _product(a2, weight, b1, r2, act, out_dtype).view(*a.shape[:-1], weight.shape[0])

  @staticmethod
  def backward(ctx, dy):
    a, weight, bias = ctx.saved_tensors
    need_a, need_w, need_b, need_r = ctx.needs_input_grad[:4]
    n, k = weight.shape
    d_a = d_w = d_b = None
    if a.shape[0] == 0:
      d_a = torch.zeros(ctx.shape, dtype=_BF16, device=a.device) if need_a else None
      d_w = torch.zeros_like(weight) if need_w else None
      d_b = torch.zeros_like(bias) if need_b else None
    elif need_a or need_w or need_b:
      d_pre, d_b = _pre_gradient(a, weight, bias, ctx.act, dy.reshape(-1, n), need_b)
      if need_a:
        d_a = _product(d_pre, weight.t(), None, None, _lib.ACT_NONE, _BF16).view(ctx.shape)
      if need_w:
        # In the weight's own orientation, so that the gradient's rows are written as they lie.
        if weight.stride(0) == 1 and weight.stride(1) != 1:
          d_w = _product(a.t(), d_pre.t(), None, None, _lib.ACT_NONE, _BF16).t()
        else:
          d_w = _product(d_pre.t(), a.t(), None, None, _lib.ACT_NONE, _BF16)
    return d_a, d_w, d_b, dy if need_r else None, None, None


def _linear_check(a, weight, bias, residual, activation, out_dtype, dtype):
  _need(a.dim() >= 1 and weight.dim() == 2 and a.shape[-1] == weight.shape[1],
        f"a has shape {tuple(a.shape)} and weight {tuple(weight.shape)}, expected [..., k] and [n, k]")
  n, k = weight.shape
  _need(n >= 1 and k >= 1, f"weight has shape {tuple(weight.shape)}, expected n, k >= 1")
  _check("a", a, a, (dtype,))
  _check("weight", weight, a, (dtype,))
  _need(activation in _ACT, f"activation {activation!r}: expected None, 'gelu' or 'swish'")
  _need(out_dtype in (_BF16, _F32), f"out_dtype {out_dtype}: expected torch.bfloat16 or torch.float32")
  if bias is not None:
    _check("bias", bias, a, (_BF16, _F32))
    _need(bias.shape == (n,), f"bias has shape {tuple(bias.shape)}, expected ({n},)")
  if residual is not None:
    _check("residual", residual, a, (out_dtype,))
    _need(residual.shape == a.shape[:-1] + (n,),
          f"residual has shape {tuple(residual.shape)}, expected {tuple(a.shape[:-1]) + (n,)}")


def linear(a, weight, bias=None, residual=None, *, activation=None, out_dtype=_BF16):
  """act(a weight^T + bias) + residual in one kernel: a [..., k] and weight [n, k] bf16, bias [n] bf16 or float32,
  residual [..., n] in out_dtype (bf16 or float32), activation None, "gelu" (tanh form) or "swish"; float32
  accumulation, rounded once. weight may be the transposed view of a [k, n] tensor (either orientation is read in
  place); rows of any stride. Differentiable in a, weight, bias and residual (gradients in their dtypes)."""
  _linear_check(a, weight, bias, residual, activation, out_dtype, _BF16)
  act = _ACT[activation]
  if torch.is_grad_enabled() and (a.requires_grad or weight.requires_grad or
                                  (bias is not None and bias.requires_grad) or
                                  (residual is not None and residual.requires_grad)):
    return _Linear.apply(a, weight, bias, residual, act, out_dtype)
  out = _product(_rows(a), weight, None if bias is None else bias.contiguous(),
                 None if residual is None else _rows(residual), act, out_dtype)
  return out.view(*a.shape[:-1], weight.shape[0])


def linear_fp8(a, a_scale, weight, weight_scale, bias=None, residual=None, *, activation=None, out_dtype=_BF16):
  """linear on 8-bit operands: act((a weight^T) a_scale weight_scale + bias) + residual, a [..., k] and weight [n, k]
  e4m3 with float32 scales per row (a_scale [...], weight_scale [n]), as rms_norm_fp8 and quantize_fp8 give them. Not
  differentiable (forecasts)."""
  _linear_check(a, weight, bias, residual, activation, out_dtype, _E4M3)
  _check("a_scale", a_scale, a, (_F32,))
  _check("weight_scale", weight_scale, a, (_F32,))
  _need(a_scale.shape == a.shape[:-1], f"a_scale has shape {tuple(a_scale.shape)}, expected {tuple(a.shape[:-1])}")
  _need(weight_scale.shape == weight.shape[:1],
        f"weight_scale has shape {tuple(weight_scale.shape)}, expected ({weight.shape[0]},)")
  out = _product(_rows(a), weight, None if bias is None else bias.contiguous(),
                 None if residual is None else _rows(residual), _ACT[activation], out_dtype,
                 a_scale=a_scale.contiguous(), b_scale=weight_scale.contiguous())
  return out.view(*a.shape[:-1], weight.shape[0])
