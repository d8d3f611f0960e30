"""Mixtures of experts: matrix products grouped by expert with ragged sizes, and the routing of rows to experts and back.

    r = route(x @ w_router, top_k=2)                     # a row's experts and their weights, rows in the experts' order
    rows = dispatch(x, r)                                # [rows * top_k, d], sorted by expert
    y = linear_grouped(rows, w1, r.offsets, b1, activation="gelu")   # rows of expert e times w1[e]
    y = linear_grouped(y, w2, r.offsets, b2)
    x = combine(y, r)                                    # the experts' rows, weighted, added back

Everything is differentiable, and nothing waits for the device: the experts' sizes stay there. No counterpart in the
reference, whose MLPs are dense (src/faster_weathernext/patch.py:250-252); beside projection.linear, whose kernel
linear_grouped walks over the experts. The kernels are csrc/grouped*.cu, csrc/linear_tile.cuh and csrc/routing.cu (C ABI in
include/fwn_attn.h, fwn_linear_grouped* and fwn_route*). Every call runs on the current stream of its tensors' device and
takes its workspace from torch's allocator.
"""

import typing

import torch

from faster_weathernext import _lib
from faster_weathernext.projection import (_ACT, _BF16, _CODE, _F32, _check, _first_order, _no_tangent, _on_device, _rows,
                                           _workspace)


# ---- products grouped by expert --------------------------------------------------------------------------------------

def _orient3(w):
  """(tensor, row stride, expert stride, transposed): w [e, n, k] with k contiguous, or with n contiguous (a transposed
  view); a copy of a tensor with neither."""
  e, n, k = w.shape
  s0, s1, s2 = w.stride()
  if (s2 == 1 or k == 1) and (s1 >= k or n == 1) and (s0 >= k or e == 1):
    ld = max(s1, k)
    return w, ld, s0 if e > 1 else n * ld, False
  if (s1 == 1 or n == 1) and (s2 >= n or k == 1) and (s0 >= n or e == 1):
    ld = max(s2, n)
    return w, ld, s0 if e > 1 else k * ld, True
  w = w.contiguous()
  return w, k, n * k, False


def _pack(src, rows, cols, ld):
  """A copy of `rows` rows of `cols` values, ld apart, in rows of whole 16 bytes."""
  out = src.new_empty((rows, -(-cols // 8) * 8))
  status = _on_device(src, lambda stream: _lib.lib().fwn_linear_pack(src.data_ptr(), ld, out.data_ptr(), out.shape[1], rows,
                                                                     cols, _lib.DTYPE_BF16, stream))
  if status:
    _lib.check(status)
  return out


def _laid_out(w):
  """w [e, n, k], or a copy in its own orientation, with rows that TMA can address."""
  src, ld, stride, turned = _orient3(w)
  if ld % 8 == 0 and stride % 8 == 0 and src.data_ptr() % 16 == 0:
    return src
  e, n, k = src.shape
  outer, inner = (k, n) if turned else (n, k)
  if e > 1 and stride != outer * ld:
    src = src.transpose(1, 2).contiguous() if turned else src.contiguous()
    ld = inner
  out = _pack(src, e * outer, inner, ld).view(e, outer, -1)[:, :, :inner]
  return out.transpose(1, 2) if turned else out


def _laid_rows(a):
  """Rows a [m, k], or a copy that TMA can address."""
  m, k = a.shape
  ld = a.stride(0) if m > 1 else k
  if (ld % 8 == 0 or m == 1) and a.data_ptr() % 16 == 0:
    return a
  return _pack(a, m, k, max(ld, k))[:, :k] if m else a


def _grouped_desc(a, weight, bias, out_dtype, x_dtype, act, ldx):
  """(descriptor, transposed) of a product whose operands are laid out."""
  m, k = a.shape
  e, n, _ = weight.shape
  _, ldb, stride, turned = _orient3(weight)
  return _lib.GroupedDesc(m, e, n, k, _CODE[out_dtype], 0 if bias is None else _CODE[bias.dtype], _CODE[x_dtype], act,
                          _lib.LINEAR_B_N_CONTIGUOUS if turned else 0, max(a.stride(0), k), ldb, stride, ldx), turned


def _ptr(t):
  return None if t is None else t.data_ptr()


def _grouped_launch(stream, a, weight, offsets, bias, act, out_dtype):
  m, n = a.shape[0], weight.shape[1]
  out = a.new_empty((m, n), dtype=out_dtype)
  if m == 0:
    return out
  desc, _ = _grouped_desc(a, weight, bias, out_dtype, out_dtype, act, n)
  lib = _lib.lib()
  ws, size = _workspace(a, desc, lib.fwn_linear_grouped_workspace_size)
  status = lib.fwn_linear_grouped(desc, a.data_ptr(), weight.data_ptr(), _ptr(bias), offsets.data_ptr(), out.data_ptr(),
                                  _ptr(ws), size, stream)
  if status:
    _lib.check(status)
  return out


class _LinearGrouped(torch.autograd.Function):
  """linear_grouped with gradients, as projection._Linear's for each expert (fwn_linear_grouped_bwd). Saved tensors may come
  back in other places (hooks may move them): the operands are laid out again where they did."""

  @staticmethod
  def forward(ctx, a, weight, offsets, bias, act, out_dtype):
    ctx.act = act
    a2, w2 = _laid_rows(_rows(a)), _laid_out(weight)
    ctx.save_for_backward(a2, w2, offsets, bias)
    return _on_device(a2, _grouped_launch, a2, w2, offsets, bias, act, out_dtype)

  @staticmethod
  def backward(ctx, dy):
    a, weight, offsets, bias = ctx.saved_tensors
    _no_tangent("linear_grouped's gradient", a, weight, bias, dy)
    need_a, need_w, _, need_b = ctx.needs_input_grad[:4]
    _first_order("linear_grouped")
    a, weight = _laid_rows(_rows(a)), _laid_out(weight)
    d_a, d_w, d_b = _on_device(a, _LinearGrouped._launch, a, weight, offsets.contiguous(),
                               None if bias is None else bias.contiguous(), ctx.act, _rows(dy), need_a, need_w, need_b)
    return d_a, d_w, None, d_b, None, None

  @staticmethod
  def _launch(stream, a, weight, offsets, bias, act, dy, need_a, need_w, need_b):
    m, k = a.shape
    e, n, _ = weight.shape
    desc, turned = _grouped_desc(a, weight, bias, dy.dtype, dy.dtype, act, max(dy.stride(0), n) if m else n)
    d_a = a.new_empty((m, k)) if need_a else None
    d_w = a.new_empty((e, k, n) if turned else (e, n, k)) if need_w else None
    d_b = bias.new_empty((e, n)) if need_b else None
    lib = _lib.lib()
    dp = dy.data_ptr()
    ws, size = _workspace(a, desc, lib.fwn_linear_grouped_bwd_workspace_size, dp) if m else (None, 0)
    status = lib.fwn_linear_grouped_bwd(desc, a.data_ptr(), weight.data_ptr(), _ptr(bias), offsets.data_ptr(), dp, _ptr(d_a),
                                        _ptr(d_w), _ptr(d_b), _ptr(ws), size, stream)
    if status:
      _lib.check(status)
    return d_a, d_w.transpose(1, 2) if turned and need_w else d_w, d_b


def linear_grouped(a, weight, offsets, bias=None, *, activation=None, out_dtype=_BF16):
  """out[i] = act(a[i] weight[e]^T + bias[e]) for offsets[e] <= i < offsets[e + 1], 0 in rows of no expert: a [m, k] and
  weight [e, n, k] bf16, offsets int32 [e + 1] on the device (not decreasing, within [0, m]; read there alone, so that no
  call waits for them), bias [e, n] bf16 or float32, activation None, "gelu" (tanh form) or "swish"; float32 accumulation,
  rounded once to out_dtype (bf16 or float32). weight may be the transposed view of an [e, k, n] tensor; either orientation
  is read in place where rows and experts lie multiples of 16 bytes apart, else every call copies it (all experts; for up to
  eight rows without a gradient it is read as it lies). Up to 1,023 experts; rows of any stride. Rows of no expert, which a
  buffer of fixed size may have, are not read.

  Differentiable in a, weight and bias as projection.linear (backward, gradients in their dtypes, 0 for rows of no expert and
  experts of no row; forward mode and second derivatives raise NotImplementedError). The gradient of the pre-activation is
  rounded to bf16, the operand of the products for a's and weight's, and so is a float32 dy without an activation: these
  gradients are off by 2.3e-3 where their own rounding alone is 1.7e-3. bias's is summed from float32."""
  if a.dim() != 2 or weight.dim() != 3 or a.shape[1] != weight.shape[2] or min(weight.shape) < 1:
    raise ValueError(f"a has shape {tuple(a.shape)} and weight {tuple(weight.shape)}, expected [m, k] and [e, n, k], "
                     "e, n, k >= 1")
  _check("a", a, a, (_BF16,))
  _check("weight", weight, a, (_BF16,))
  _check("offsets", offsets, a, (torch.int32,))
  if offsets.dim() != 1 or offsets.shape[0] != weight.shape[0] + 1:
    raise ValueError(f"offsets has shape {tuple(offsets.shape)}, expected ({weight.shape[0] + 1},)")
  if activation not in _ACT:
    raise ValueError(f"activation {activation!r}: expected None, 'gelu' or 'swish'")
  if out_dtype is not _BF16 and out_dtype is not _F32:
    raise ValueError(f"out_dtype {out_dtype}: expected torch.bfloat16 or torch.float32")
  if bias is not None:
    _check("bias", bias, a, (_BF16, _F32))
    if bias.shape != weight.shape[:2]:
      raise ValueError(f"bias has shape {tuple(bias.shape)}, expected {tuple(weight.shape[:2])}")
    if not bias.is_contiguous():
      bias = bias.contiguous()
  _no_tangent("linear_grouped", a, weight, bias)
  if not offsets.is_contiguous():
    offsets = offsets.contiguous()
  act = _ACT[activation]
  if torch.is_grad_enabled() and (a.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
    return _LinearGrouped.apply(a, weight, offsets, bias, act, out_dtype)
  a = _rows(a)
  if a.shape[0] > 8 or _orient3(weight)[3]:
    a, weight = _laid_rows(a), _laid_out(weight)
  else:
    weight = _orient3(weight)[0]
  return _on_device(a, _grouped_launch, a, weight, offsets, bias, act, out_dtype)


# ---- routing ---------------------------------------------------------------------------------------------------------

class Routing(typing.NamedTuple):
  """Where rows go: experts [rows, top_k] int32 (largest logit first) and weights [rows, top_k] float32 (differentiable);
  position [rows, top_k] int32, the place of each pair (row, choice) in the experts' order; order [rows * top_k] int32, the
  pair (row * top_k + choice) in each place; offsets [experts + 1] int32, the first place of each expert."""
  experts: torch.Tensor
  weights: torch.Tensor
  position: torch.Tensor
  order: torch.Tensor
  offsets: torch.Tensor


def _route_launch(stream, logits, top_k):
  rows, e = logits.shape
  chosen, position, order = logits.new_empty((3, rows, top_k), dtype=torch.int32).unbind()
  order = order.view(rows * top_k)
  weights, offsets = logits.new_empty((rows, top_k), dtype=_F32), logits.new_empty((e + 1,), dtype=torch.int32)
  desc = _lib.RouteDesc(rows, e, top_k, _CODE[logits.dtype], 0)
  lib = _lib.lib()
  ws, size = _workspace(logits, desc, lib.fwn_route_workspace_size)
  status = lib.fwn_route(desc, logits.data_ptr(), max(logits.stride(0), e), chosen.data_ptr(), weights.data_ptr(),
                         order.data_ptr(), position.data_ptr(), offsets.data_ptr(), _ptr(ws), size, stream)
  if status:
    _lib.check(status)
  return chosen, weights, position, order, offsets


class _Route(torch.autograd.Function):
  """route with the weights' gradient; the choice itself has none."""

  @staticmethod
  def forward(ctx, logits, top_k):
    chosen, weights, position, order, offsets = _on_device(logits, _route_launch, _rows(logits), top_k)
    ctx.mark_non_differentiable(chosen, position, order, offsets)
    ctx.set_materialize_grads(False)  # zeros for each of them, otherwise
    ctx.shape, ctx.dtype = logits.shape, logits.dtype
    ctx.save_for_backward(chosen, weights)
    return chosen, weights, position, order, offsets

  @staticmethod
  def backward(ctx, _chosen, d_weights, *_rest):
    if d_weights is None:
      return None, None
    chosen, weights = ctx.saved_tensors
    _no_tangent("route's gradient", weights, d_weights)
    _first_order("route")
    return _on_device(weights, _Route._launch, ctx, chosen.contiguous(), weights.contiguous(), d_weights.contiguous()), None

  @staticmethod
  def _launch(stream, ctx, chosen, weights, d_weights):
    d_logits = weights.new_empty(ctx.shape, dtype=ctx.dtype)
    desc = _lib.RouteDesc(chosen.shape[0], ctx.shape[1], chosen.shape[1], _CODE[ctx.dtype], 0)
    status = _lib.lib().fwn_route_bwd(desc, weights.data_ptr(), chosen.data_ptr(), d_weights.data_ptr(), d_logits.data_ptr(),
                                      stream)
    if status:
      _lib.check(status)
    return d_logits


def route(logits, top_k):
  """The top_k largest of each row's logits [rows, e] (float32 or bf16, any strides; e <= 1,023, top_k <= 16) and their
  softmax, and the rows in the experts' order: a Routing. Equal logits go to the lower expert, a NaN counts as the largest
  (and gives its row NaN weights), -infinity has weight 0 (a row of nothing else: every weight 0). The sort is stable and
  deterministic. Differentiable in the logits through the weights (backward; forward mode and second derivatives raise
  NotImplementedError)."""
  if logits.dim() != 2 or logits.shape[1] < 1:
    raise ValueError(f"logits has shape {tuple(logits.shape)}, expected [rows, e] with e >= 1")
  _check("logits", logits, logits, (_BF16, _F32))
  if not isinstance(top_k, int) or not 1 <= top_k <= logits.shape[1]:
    raise ValueError(f"top_k is {top_k!r}, expected a whole number of 1 to {logits.shape[1]}")
  _no_tangent("route", logits)
  if torch.is_grad_enabled() and logits.requires_grad:
    return Routing(*_Route.apply(logits, top_k))
  return Routing(*_on_device(logits, _route_launch, _rows(logits), top_k))


_MOVES = {}  # descriptors of the rows' ways


def _move_desc(t, position):
  key = (position.shape, t.dtype)
  desc = _MOVES.get(key)
  if desc is None:
    if len(_MOVES) >= 4096:
      _MOVES.clear()
    rows, top_k = position.shape
    desc = _MOVES[key] = _lib.RouteDesc(rows, top_k, top_k, _CODE[t.dtype], 0)  # the number of experts does not matter here
  return desc


def _spread_launch(stream, x, position, weights, y, wanted):
  """(weights[r, j] x[r] in the experts' order or None, dots with y or None)."""
  rows, top_k = position.shape
  d = x.shape[1]
  out = x.new_empty((rows * top_k, d)) if wanted else None
  dots = x.new_empty((rows, top_k), dtype=_F32) if y is not None else None
  status = _lib.lib().fwn_route_spread(_move_desc(x, position), d, x.data_ptr(), max(x.stride(0), d), position.data_ptr(),
                                       _ptr(weights), _ptr(y), _ptr(out), _ptr(dots), stream)
  if status:
    _lib.check(status)
  return out, dots


def _gather_launch(stream, y, position, weights):
  out = y.new_empty((position.shape[0], y.shape[1]))
  status = _lib.lib().fwn_route_gather(_move_desc(y, position), y.shape[1], y.data_ptr(), position.data_ptr(), _ptr(weights),
                                       out.data_ptr(), stream)
  if status:
    _lib.check(status)
  return out


class _Dispatch(torch.autograd.Function):

  @staticmethod
  def forward(ctx, x, position):
    ctx.save_for_backward(position)
    return _on_device(x, _spread_launch, _rows(x), position, None, None, True)[0]

  @staticmethod
  def backward(ctx, d_rows):
    position, = ctx.saved_tensors
    _no_tangent("dispatch's gradient", d_rows)
    _first_order("dispatch")
    return _on_device(d_rows, _gather_launch, d_rows.contiguous(), position.contiguous(), None), None


class _Combine(torch.autograd.Function):

  @staticmethod
  def forward(ctx, y, weights, position):
    y2 = y.contiguous()
    ctx.save_for_backward(y2, weights, position)
    return _on_device(y2, _gather_launch, y2, position, weights)

  @staticmethod
  def backward(ctx, d_out):
    y, weights, position = ctx.saved_tensors
    _no_tangent("combine's gradient", y, weights, d_out)
    _first_order("combine")
    d_y, d_weights = _on_device(d_out, _spread_launch, _rows(d_out), position.contiguous(), weights.contiguous(),
                                y.contiguous() if ctx.needs_input_grad[1] else None, ctx.needs_input_grad[0])
    return d_y, d_weights, None


def _routed_check(name, t, routing, each):
  """t [rows * each, d] belongs to a routing of `rows` rows."""
  _check(name, t, t, (_BF16, _F32))
  _check("routing.position", routing.position, t, (torch.int32,))
  _check("routing.weights", routing.weights, t, (_F32,))
  if (routing.position.dim() != 2 or routing.weights.shape != routing.position.shape or not routing.position.is_contiguous()
      or not routing.weights.is_contiguous()):
    raise ValueError("routing's position and weights are not contiguous [rows, top_k] as route returns them")
  rows = routing.position.shape[0] * each
  if t.dim() != 2 or t.shape[0] != rows or t.shape[1] < 1:
    raise ValueError(f"{name} has shape {tuple(t.shape)}, expected ({rows}, d) with d >= 1")
  _no_tangent(name, t, routing.weights)


def dispatch(x, routing):
  """The rows of x [rows, d] (float32 or bf16, any strides) in the experts' order: [rows * top_k, d], linear_grouped's left
  operand with routing.offsets. Differentiable in x: the gradient of a row is the sum of its places', in float32, rounded
  once (backward; forward mode and second derivatives raise NotImplementedError)."""
  _routed_check("x", x, routing, 1)
  if torch.is_grad_enabled() and x.requires_grad:
    return _Dispatch.apply(x, routing.position)
  return _on_device(x, _spread_launch, _rows(x), routing.position, None, None, True)[0]


def combine(y, routing):
  """The experts' rows y [rows * top_k, d] (float32 or bf16), in the experts' order, added back: out[r] = sum over a row's
  choices of weight * y's row, in float32, rounded once to y's type. Differentiable in y and in the routing's weights
  (backward; forward mode and second derivatives raise NotImplementedError)."""
  _routed_check("y", y, routing, routing.position.shape[-1])
  if torch.is_grad_enabled() and (y.requires_grad or routing.weights.requires_grad):
    return _Combine.apply(y, routing.weights, routing.position)
  return _on_device(y, _gather_launch, y.contiguous(), routing.position, routing.weights)
