"""Cases of the pre-norm projections: the root-mean-square norm with the residual's addition (rms_norm, rms_norm_fp8)
and the matrix product with bias, activation and residual in its epilogue (linear, linear_fp8).

Rows are mesh nodes times ensemble members: 40,962 nodes (a level-6 icosphere) for the configurations the benchmark
times, 12 to 10,242 for the coarser levels, 1 for a single node or token. Widths are the processor's (512, MLP 2,048)
and odd ones. Each case runs in its plain form (`own` false: elementary torch operations in float32, rounded once) or
through faster_weathernext.projection (`own` true).

  rms_norm      s = x + residual,  h = s / sqrt(mean(s^2) + eps) * weight;  outputs h and, with a residual, s
  rms_norm_fp8  the same h as e4m3 values with one float32 scale per row, scale = max |h| / 448
  linear        act(a weight^T + bias) + residual, bf16 operands, optionally with all its gradients
  linear_fp8    act((a weight^T) a_scale weight_scale + bias) + residual, e4m3 operands with a scale per row of each
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-6
_DT = {"bf16": torch.bfloat16, "f32": torch.float32}
_NODES = 40962          # level-6 icosphere


# ---- cases ----------------------------------------------------------------------------------------------------------

def _rms(name, rows, d, stream="f32", residual="bf16", weight="f32", out="bf16", train=False):
  return {"name": name, "op": "rms_norm", "rows": rows, "d": d, "stream": stream, "residual": residual,
          "weight": weight, "out": out, "train": train}


def _lin(name, m, k, n, kind="bf16", act="none", bias="f32", residual="none", out="bf16", layout="nk", train=False):
  return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "kind": kind, "act": act, "bias": bias,
          "residual": residual, "out": out, "layout": layout, "train": train}


def listed():
  return [
      # A block's norm in a forecast of four members: the sub-block's bf16 output is added into the float32 stream.
      _rms("norm residual", 4 * _NODES, 512),
      # The same norm before an 8-bit projection.
      _rms("norm residual fp8", 4 * _NODES, 512, out="fp8"),
      # One node (or token) into an 8-bit projection: a call's own cost.
      _rms("norm one row fp8", 1, 2048, stream="bf16", residual="none", weight="bf16", out="fp8"),
      # Fine-tuning: forward and every gradient at four members.
      _rms("norm train", 4 * _NODES, 512, train=True),
      # A level-5 mesh with an odd width and a bf16 stream, forward and every gradient.
      _rms("norm train odd", 10242, 1001, stream="bf16", weight="f32", train=True),
      # The MLP's up-projection of a forecast of four members.
      _lin("up gelu", 4 * _NODES, 512, 2048, act="gelu"),
      # The same with 8-bit operands.
      _lin("up gelu fp8", 4 * _NODES, 512, 2048, kind="fp8", act="gelu"),
      # The down-projection, adding into the float32 residual stream in its epilogue.
      _lin("down residual", 4 * _NODES, 2048, 512, residual="f32", out="f32"),
      # One node (or token) through the down-projection: the weights' bytes and the call's latency.
      _lin("down one row", 1, 2048, 512, residual="f32", out="f32"),
      # A level-1 mesh (42 nodes) through the 8-bit up-projection.
      _lin("up small fp8", 42, 512, 2048, kind="fp8", act="swish"),
      # Fine-tuning: the up-projection with the processor's [k, n] weights, forward and every gradient, two members.
      _lin("up train", 2 * _NODES, 512, 2048, act="gelu", layout="kn", train=True),
      # A level-4 mesh with odd widths, forward and every gradient.
      _lin("odd train", 2562, 1001, 515, act="swish", residual="bf16", train=True),
  ]


_MOST_FLOPS = 6.0 * 2 * _NODES * 512 * 2048     # the largest listed case ("up train")
_MOST_VALUES = 4 * _NODES * 512                 # values of the norm's largest listed case
_MOST_OUT = 4 * _NODES * 2048                   # and of the projection's largest output


def _spread(rng, lo, hi):
  v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
  return min(max(v, lo), hi)


def _width(rng, lo, hi):
  """Half of the widths are multiples of 64, the others are left as drawn."""
  while True:
    v = _spread(rng, lo, hi)
    if rng.random() < 0.5:
      v = max(64, (v + 32) // 64 * 64)
    if v != 3 * 1024:
      return v


def draw(rng):
  if rng.random() < 0.45:
    while True:
      c = _rms("", _spread(rng, 1, 4 * _NODES), _width(rng, 64, 4096), stream=rng.choice(["f32", "bf16"]),
               residual=rng.choice(["none", "bf16", "bf16", "f32"]), weight=rng.choice(["none", "bf16", "f32", "f32"]),
               out=rng.choice(["bf16", "bf16", "fp8", "f32"]))
      c["train"] = c["out"] != "fp8" and rng.random() < 0.5
      if c["rows"] * c["d"] <= _MOST_VALUES:
        break
  else:
    while True:
      out = rng.choice(["bf16", "bf16", "f32"])
      c = _lin("", _spread(rng, 1, 4 * _NODES), _width(rng, 64, 4096), _width(rng, 64, 4096),
               kind=rng.choice(["bf16", "bf16", "fp8"]), act=rng.choice(["none", "gelu", "swish"]),
               bias=rng.choice(["none", "bf16", "f32"]), residual=rng.choice(["none", out]), out=out)
      if c["kind"] == "bf16":
        c["layout"] = rng.choice(["nk", "kn"])
        c["train"] = rng.random() < 0.4
      flops = 2.0 * c["m"] * c["k"] * c["n"] * (3 if c["train"] else 1)
      if flops <= _MOST_FLOPS and c["m"] * max(c["k"], c["n"]) <= _MOST_OUT // (2 if c["train"] else 1):
        break
  del c["name"]
  return c


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _gen(seed):
  return torch.Generator(device="cuda").manual_seed(int(seed))


def _prepare_rms(c, seed):
  g = _gen(seed)
  rows, d = c["rows"], c["d"]
  rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
  # A residual stream: channels of different sizes, a few of them large, as after some blocks.
  channel = torch.exp(0.5 * rand(d))
  channel[:: max(1, d // 8)] *= 6.0
  s = {"case": c, "x": (rand(rows, d) * channel).to(_DT[c["stream"]])}
  s["residual"] = (0.3 * rand(rows, d)).to(_DT[c["residual"]]) if c["residual"] != "none" else None
  s["weight"] = (1.0 + 0.1 * rand(d)).to(_DT[c["weight"]]) if c["weight"] != "none" else None
  if c["train"]:
    s["dh"] = (0.01 * rand(rows, d)).to(_DT[c["out"]])
    s["dx"] = (0.01 * rand(rows, d)).to(_DT[c["stream"]]) if s["residual"] is not None else None
    for key in ("x", "residual", "weight"):
      if s[key] is not None:
        s[key].requires_grad_()
  return s


def _quantized(t):
  """e4m3 values and one scale per row, as a checkpoint in 8 bits holds a weight."""
  scale = t.abs().amax(1) / 448.0
  return (t / scale[:, None]).to(torch.float8_e4m3fn), scale


def _prepare_lin(c, seed):
  g = _gen(seed)
  m, k, n = c["m"], c["k"], c["n"]
  rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
  s = {"case": c}
  a, w = rand(m, k), rand(n, k) * k ** -0.5
  if c["kind"] == "fp8":
    s["a"], s["a_scale"] = _quantized(a)
    s["weight"], s["weight_scale"] = _quantized(w)
  else:
    s["a"] = a.to(torch.bfloat16)
    # "kn": the processor keeps its weights as [k, n]; the call gets the transposed view.
    s["weight"] = w.to(torch.bfloat16) if c["layout"] == "nk" else w.t().contiguous().to(torch.bfloat16).t()
  s["bias"] = (0.2 * rand(n)).to(_DT[c["bias"]]) if c["bias"] != "none" else None
  s["residual"] = rand(m, n).to(_DT[c["residual"]]) if c["residual"] != "none" else None
  if c["train"]:
    s["dy"] = (0.01 * rand(m, n)).to(_DT[c["out"]])
    for key in ("a", "weight", "bias", "residual"):
      if s[key] is not None:
        s[key].requires_grad_()
  return s


def prepare(case, seed):
  return _prepare_rms(case, seed) if case["op"] == "rms_norm" else _prepare_lin(case, seed)


# ---- plain forms ----------------------------------------------------------------------------------------------------

def _plain_rms(s):
  c = s["case"]
  x = s["x"].float()
  total = x if s["residual"] is None else x + s["residual"].float()
  rstd = 1.0 / torch.sqrt(torch.mean(total * total, 1, keepdim=True) + EPS)
  xhat = total * rstd
  w = None if s["weight"] is None else s["weight"].float()
  h = xhat if w is None else xhat * w
  out = {}
  if s["residual"] is not None:
    out["x"] = total.to(s["x"].dtype)
  if c["out"] == "fp8":
    scale = torch.amax(torch.abs(h), 1) / 448.0
    out["values"] = torch.clamp(h / scale[:, None], -448.0, 448.0).to(torch.float8_e4m3fn)
    out["scale"] = scale
    return out
  out["h"] = h.to(_DT[c["out"]])
  if c["train"]:
    dh = s["dh"].float()
    gr = dh if w is None else dh * w
    dx = (gr - xhat * torch.mean(gr * xhat, 1, keepdim=True)) * rstd
    if s["residual"] is not None:
      dx = dx + s["dx"].float()
      out["d_residual"] = dx.to(s["residual"].dtype)
    out["d_x"] = dx.to(s["x"].dtype)
    if w is not None:
      out["d_weight"] = torch.sum(dh * xhat, 0).to(s["weight"].dtype)
  return out


_C0, _C1 = math.sqrt(2.0 / math.pi), 0.044715


def _plain_act(x, act):
  if act == "gelu":
    return 0.5 * x * (1.0 + torch.tanh(_C0 * (x + _C1 * x * x * x)))
  if act == "swish":
    return x / (1.0 + torch.exp(-x))
  return x


def _plain_act_grad(x, act):
  if act == "gelu":
    t = torch.tanh(_C0 * (x + _C1 * x * x * x))
    return 0.5 * (1.0 + t) + 0.5 * x * (1.0 - t * t) * _C0 * (1.0 + 3.0 * _C1 * x * x)
  if act == "swish":
    p = 1.0 / (1.0 + torch.exp(-x))
    return p * (1.0 + x * (1.0 - p))
  return None


def _plain_lin(s):
  c = s["case"]
  a, w = s["a"].float(), s["weight"].float()
  if c["kind"] == "fp8":
    a, w = a * s["a_scale"][:, None], w * s["weight_scale"][:, None]
  pre = torch.matmul(a, w.t())
  if s["bias"] is not None:
    pre = pre + s["bias"].float()
  y = _plain_act(pre, c["act"])
  if s["residual"] is not None:
    y = y + s["residual"].float()
  out = {"y": y.to(_DT[c["out"]])}
  if c["train"]:
    del y
    dy = s["dy"].float()
    slope = _plain_act_grad(pre, c["act"])
    d_pre = dy if slope is None else dy * slope
    out["d_a"] = torch.matmul(d_pre, w).to(s["a"].dtype)
    out["d_weight"] = torch.matmul(d_pre.t(), a).to(s["weight"].dtype)
    if s["bias"] is not None:
      out["d_bias"] = torch.sum(d_pre, 0).to(s["bias"].dtype)
    if s["residual"] is not None:
      out["d_residual"] = dy.to(s["residual"].dtype)
  return out


# ---- the framework's calls ------------------------------------------------------------------------------------------

def _projection():
  path = os.path.join(os.getcwd(), "faster-weathernext_b200")
  if path not in sys.path:
    sys.path.insert(0, path)
  from faster_weathernext import projection
  return projection


def _own_rms(s):
  c, pr = s["case"], _projection()
  if c["out"] == "fp8":
    got = pr.rms_norm_fp8(s["x"], s["weight"], s["residual"], eps=EPS)
    out = {"values": got[0], "scale": got[1]}
    if s["residual"] is not None:
      out["x"] = got[2]
    return out
  got = pr.rms_norm(s["x"], s["weight"], s["residual"], eps=EPS, out_dtype=_DT[c["out"]])
  outs = got if s["residual"] is not None else (got,)
  out = {"h": outs[0].detach()}
  if s["residual"] is not None:
    out["x"] = outs[1].detach()
  if c["train"]:
    keys = [k for k in ("x", "residual", "weight") if s[k] is not None]
    grads = torch.autograd.grad(outs, [s[k] for k in keys], (s["dh"],) if s["residual"] is None else (s["dh"], s["dx"]))
    out.update({"d_" + k: v for k, v in zip(keys, grads)})
  return out


def _own_lin(s):
  c, pr = s["case"], _projection()
  act, dt = None if c["act"] == "none" else c["act"], _DT[c["out"]]
  if c["kind"] == "fp8":
    return {"y": pr.linear_fp8(s["a"], s["a_scale"], s["weight"], s["weight_scale"], s["bias"], s["residual"],
                               activation=act, out_dtype=dt)}
  y = pr.linear(s["a"], s["weight"], s["bias"], s["residual"], activation=act, out_dtype=dt)
  out = {"y": y.detach()}
  if c["train"]:
    keys = [k for k in ("a", "weight", "bias", "residual") if s[k] is not None]
    out.update({"d_" + k: v for k, v in zip(keys, torch.autograd.grad(y, [s[k] for k in keys], s["dy"]))})
  return out


def run(state):
  rms = state["case"]["op"] == "rms_norm"
  if own:
    return _own_rms(state) if rms else _own_lin(state)
  with torch.no_grad():
    return _plain_rms(state) if rms else _plain_lin(state)


# ---- work and exact values ------------------------------------------------------------------------------------------

def _size(name):
  return {"none": 0, "fp8": 1, "bf16": 2, "f32": 4}[name]


def work(case):
  c = case
  if c["op"] == "rms_norm":
    r, d = c["rows"], c["d"]
    st, re, ou, we = (_size(c[k]) for k in ("stream", "residual", "out", "weight"))
    nbytes = r * d * (st + re + ou + (st if re else 0)) + d * we + (4 * r if c["out"] == "fp8" else 0)
    flops = 5.0 * r * d
    if c["train"]:
      # The gradients' read (and the stream's again, from what the forward wrote or read), the inputs' gradients.
      nbytes += r * d * (ou + (st if re else 0) + st + st + re) + d * we
      flops += 10.0 * r * d
    return {"bytes": nbytes, "flops": flops}
  m, k, n = c["m"], c["k"], c["n"]
  es = 1 if c["kind"] == "fp8" else 2
  ou, re, bi = _size(c["out"]), _size(c["residual"]), _size(c["bias"])
  nbytes = es * (m * k + n * k) + m * n * (ou + re) + n * bi + (4 * (m + n) if c["kind"] == "fp8" else 0)
  flops = 2.0 * m * n * k
  if c["train"]:
    nbytes += m * n * (ou + re) + 2 * (m * k + n * k) * 2 + n * bi
    flops *= 3
  return {"bytes": nbytes, "flops": flops}


def _leaf(t):
  return None if t is None else t.detach().double().requires_grad_()


def _exact_rms(c, s):
  with torch.enable_grad():
    x, r, w = _leaf(s["x"]), _leaf(s["residual"]), _leaf(s["weight"])
    total = x if r is None else torch.add(x, r)
    h = total * torch.rsqrt(total.pow(2).sum(-1).div(c["d"]).add(EPS)).unsqueeze(-1)
    if w is not None:
      h = torch.mul(h, w)
    out = {}
    if r is not None:
      out["x"] = total.detach()
    if c["out"] == "fp8":
      scale = h.detach().abs().max(-1).values.div(448.0)
      out["values"], out["scale"] = h.detach().div(scale.unsqueeze(-1)), scale
      return out
    out["h"] = h.detach()
    if c["train"]:
      keys = [k for k, v in (("x", x), ("residual", r), ("weight", w)) if v is not None]
      heads, seeds = ([h], [s["dh"].double()]) if r is None else ([h, total], [s["dh"].double(), s["dx"].double()])
      grads = torch.autograd.grad(heads, [{"x": x, "residual": r, "weight": w}[k] for k in keys], seeds)
      out.update({"d_" + k: v for k, v in zip(keys, grads)})
  return out


def _exact_lin(c, s):
  with torch.enable_grad():
    a, w, b, r = _leaf(s["a"]), _leaf(s["weight"]), _leaf(s["bias"]), _leaf(s["residual"])
    y = torch.einsum("mk,nk->mn", a, w)
    if c["kind"] == "fp8":
      y = y * torch.outer(s["a_scale"].double(), s["weight_scale"].double())
    if b is not None:
      y = torch.add(y, b)
    if c["act"] == "gelu":
      # x sigmoid(2 u): the tanh form written through the logistic function.
      y = y * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y.pow(3)))
    elif c["act"] == "swish":
      y = y * torch.sigmoid(y)
    if r is not None:
      y = torch.add(y, r)
    out = {"y": y.detach()}
    if c["train"]:
      keys = [k for k, v in (("a", a), ("weight", w), ("bias", b), ("residual", r)) if v is not None]
      grads = torch.autograd.grad(y, [{"a": a, "weight": w, "bias": b, "residual": r}[k] for k in keys], s["dy"].double())
      out.update({"d_" + k: v for k, v in zip(keys, grads)})
  return out


def exact(case, seed):
  s = prepare(case, seed)
  return _exact_rms(case, s) if case["op"] == "rms_norm" else _exact_lin(case, s)
