"""Cases of a mixture-of-experts block's operators: dropout from a counter-based generator (dropout), the norms after and
before a block with its gate, its residual scale and dropout in one pass (branch_norm, branch_norm_fp8), matrix products
grouped by expert with ragged sizes (linear_grouped), and the routing of rows to experts and back (route, dispatch,
combine).

Rows are mesh nodes times ensemble members: 40,962 nodes (a level-6 icosphere) for the configurations the benchmark
times, 12 to 10,242 for the coarser levels, 1 for a single node or token; a row that goes to k experts makes k rows of
their products. Widths are the processor's (512, MLP 2,048) and odd ones. Each case runs in its plain form (`own` false:
elementary torch operations in float32, rounded once) or through faster_weathernext.branch and
faster_weathernext.experts (`own` true).

  dropout         y = x m,  m = 0 with probability T / 65536, else 65536 / (65536 - T), T = round(65536 p); the mask comes
                  from Philox4x32-10 (Salmon, Moraes, Dror, Shaw, SC 2011): eight 16-bit numbers from the words of the
                  counter (i / 8, site, 0) under the key `seed`, value i of the tensor taking number i % 8, dropped below T
  branch_norm     z = y / sqrt(mean(y^2) + eps) post_weight,  s = residual_scale x + gate z m,
                  h = s / sqrt(mean(s^2) + eps) weight;  outputs h and s, optionally all gradients
  branch_norm_fp8 the same h as e4m3 values with one float32 scale per row, scale = max |h| / 448
  linear_grouped  rows offsets[e] to offsets[e + 1] of act(a weight[e]^T + bias[e]), 0 in rows of no expert
  route, ...      the top_k largest logits of a row (ties: the lower index) and their softmax; rows ordered by expert; rows
                  copied into that order, and the experts' results weighted and added back
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

EPS = 1e-6
_DT = {"bf16": torch.bfloat16, "f32": torch.float32}
_NODES = 40962          # level-6 icosphere


# ---- cases ----------------------------------------------------------------------------------------------------------

def _drop(name, rows, d, p, kind="bf16"):
  return {"name": name, "op": "dropout", "rows": rows, "d": d, "p": p, "kind": kind}


def _branch(name, samples, nodes, d, stream="f32", branch="bf16", gate="sample", weight="f32", out="bf16", scale=1.0,
            p=0.0, train=False):
  return {"name": name, "op": "branch", "samples": samples, "nodes": nodes, "d": d, "stream": stream, "branch": branch,
          "gate": gate, "weight": weight, "out": out, "scale": scale, "p": p, "train": train}


def _grouped(name, rows, experts, k, n, act="none", bias="f32", out="bf16", layout="nk", tail=0, train=False):
  return {"name": name, "op": "grouped", "rows": rows, "experts": experts, "k": k, "n": n, "act": act, "bias": bias,
          "out": out, "layout": layout, "tail": tail, "train": train}


def _mix(name, rows, experts, top_k, d, kind="bf16", train=False):
  return {"name": name, "op": "mix", "rows": rows, "experts": experts, "top_k": top_k, "d": d, "kind": kind,
          "train": train}


def listed():
  return [
      # Fine-tuning of four members: a sub-block's output dropped, and its gradient through the same mask.
      _drop("dropout train", 4 * _NODES, 512, 0.1),
      # A level-5 mesh with an odd width in float32.
      _drop("dropout odd", 10242, 1001, 0.25, kind="f32"),
      # A forecast of four members, each with its own gate (conditioning): the sub-block's bf16 output is normed, gated and
      # added into the float32 stream, and the next sub-block's input is the norm of the sum.
      _branch("branch gate", 4, _NODES, 512),
      # One node (or token) into an 8-bit projection: a call's own cost.
      _branch("branch one row fp8", 1, 1, 2048, stream="bf16", gate="channel", weight="bf16", out="fp8", scale=0.5),
      # Fine-tuning of four members with dropout: forward and every gradient.
      _branch("branch train", 4, _NODES, 512, p=0.1, train=True),
      # A level-5 mesh with an odd width and a bf16 stream, one gate for all rows.
      _branch("branch train odd", 1, 10242, 1001, stream="bf16", gate="channel", scale=1.25, train=True),
      # The experts' up-projection in a forecast of two members, each node to two of eight experts.
      _grouped("grouped up gelu", 4 * _NODES, 8, 512, 2048, act="gelu"),
      # One node (or token) to two of eight experts: the weights' bytes and the call's latency.
      _grouped("grouped two rows", 2, 8, 2048, 512),
      # Fine-tuning: the up-projection with weights kept as [experts, k, n], one member, forward and every gradient.
      _grouped("grouped train", 2 * _NODES, 8, 512, 2048, act="gelu", layout="kn", train=True),
      # A level-4 mesh with odd widths and rows of no expert behind the last (a buffer of fixed size).
      _grouped("grouped train odd", 2 * 2562, 6, 1001, 515, act="swish", tail=60, train=True),
      # Fine-tuning of two members: the routing of each node to two of eight experts, there and back, with gradients.
      _mix("mix train", 2 * _NODES, 8, 2, 512, train=True),
      # One token to four of 64 experts.
      _mix("mix one row", 1, 64, 4, 2048),
  ]


_MOST_VALUES = 4 * _NODES * 512                 # values of the largest listed norm
_MOST_FLOPS = 6.0 * 2 * _NODES * 512 * 2048     # of the largest listed product with its gradients
_MOST_ROUTED = 2 * _NODES * 2 * 512             # values of the largest listed dispatch


def _spread(rng, lo, hi):
  v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
  return min(max(v, lo), hi)


def _width(rng, lo, hi):
  """Half of the widths are multiples of 64, the others are left as drawn."""
  v = _spread(rng, lo, hi)
  if rng.random() < 0.5:
    v = max(64, (v + 32) // 64 * 64)
  return v


def draw(rng):
  kind = rng.random()
  while True:
    if kind < 0.15:
      c = _drop("", _spread(rng, 1, 4 * _NODES), _width(rng, 64, 4096), rng.choice([0.05, 0.1, 0.25, 0.5]),
                kind=rng.choice(["bf16", "f32"]))
      fits = c["rows"] * c["d"] <= _MOST_VALUES
    elif kind < 0.5:
      out = rng.choice(["bf16", "bf16", "f32", "fp8"])
      train = out != "fp8" and rng.random() < 0.6
      c = _branch("", rng.choice([1, 1, 2, 4, 7]), _spread(rng, 1, _NODES), _width(rng, 64, 4096),
                  stream=rng.choice(["f32", "bf16"]), branch=rng.choice(["bf16", "bf16", "f32"]),
                  gate=rng.choice(["none", "channel", "sample", "sample", "value"]), weight=rng.choice(["none", "bf16", "f32", "f32"]),
                  out=out, scale=rng.choice([1.0, 1.0, 0.5, 1.25]), p=rng.choice([0.0, 0.1, 0.25]) if train else 0.0, train=train)
      fits = c["samples"] * c["nodes"] * c["d"] <= _MOST_VALUES // (2 if c["gate"] == "value" else 1)
    elif kind < 0.8:
      c = _grouped("", _spread(rng, 1, 4 * _NODES), _spread(rng, 1, 64), _width(rng, 64, 4096), _width(rng, 64, 4096),
                   act=rng.choice(["none", "gelu", "swish"]), bias=rng.choice(["none", "bf16", "f32"]),
                   out=rng.choice(["bf16", "bf16", "f32"]), layout=rng.choice(["nk", "kn"]),
                   tail=rng.choice([0, 0, 13, 200]), train=rng.random() < 0.4)
      flops = 2.0 * c["rows"] * c["k"] * c["n"] * (3 if c["train"] else 1)
      fits = (flops <= _MOST_FLOPS and c["experts"] * c["k"] * c["n"] <= 64 * 512 * 2048
              and c["rows"] * max(c["k"], c["n"]) <= 4 * _NODES * 2048 // (2 if c["train"] else 1))
    else:
      experts = _spread(rng, 2, 64)
      c = _mix("", _spread(rng, 1, 2 * _NODES), experts, rng.choice([k for k in (1, 2, 2, 3, 4, 8) if k <= experts]),
               _width(rng, 64, 2048), kind=rng.choice(["bf16", "bf16", "f32"]), train=rng.random() < 0.6)
      fits = c["rows"] * c["top_k"] * c["d"] * (2 if c["kind"] == "f32" else 1) <= _MOST_ROUTED
    if fits:
      del c["name"]
      return c


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _randn(seed):
  g = torch.Generator(device="cuda").manual_seed(int(seed))
  return lambda *s: torch.randn(*s, device="cuda", generator=g)


def _seed_tensor(seed):
  """The generator's seed as a training loop keeps it: one 64-bit number on the device."""
  return torch.tensor([random.Random(int(seed)).getrandbits(63)], dtype=torch.int64, device="cuda")


def _prepare_drop(c, seed):
  rand = _randn(seed)
  return {"case": c, "x": rand(c["rows"], c["d"]).to(_DT[c["kind"]]).requires_grad_(),
          "dy": (0.01 * rand(c["rows"], c["d"])).to(_DT[c["kind"]]), "seed": _seed_tensor(seed)}


def _prepare_branch(c, seed):
  rand = _randn(seed)
  b, n, d = c["samples"], c["nodes"], c["d"]
  # A residual stream: channels of different sizes, a few of them large, as after some blocks.
  channel = torch.exp(0.5 * rand(d))
  channel[:: max(1, d // 8)] *= 6.0
  s = {"case": c, "x": (rand(b, n, d) * channel).to(_DT[c["stream"]]), "y": (0.5 * rand(b, n, d)).to(_DT[c["branch"]])}
  w = c["weight"]
  for key in ("post_weight", "weight"):
    s[key] = (1.0 + 0.1 * rand(d)).to(_DT[w]) if w != "none" else None
  shape = {"none": None, "channel": (d,), "sample": (b, d), "value": (b, n, d)}[c["gate"]]
  s["gate"] = None if shape is None else (0.5 + 0.2 * rand(*shape)).to(_DT[c["branch"] if c["gate"] == "value" else "f32"])
  s["seed"] = _seed_tensor(seed)
  if c["train"]:
    s["dh"] = (0.01 * rand(b, n, d)).to(_DT[c["out"]])
    s["ds"] = (0.01 * rand(b, n, d)).to(_DT[c["stream"]])
    for key in _BRANCH_LEAVES:
      if s[key] is not None:
        s[key].requires_grad_()
  return s


_BRANCH_LEAVES = ("x", "y", "post_weight", "weight", "gate")


def _prepare_grouped(c, seed):
  rand = _randn(seed)
  rng = random.Random(int(seed))
  m, e, k, n = c["rows"], c["experts"], c["k"], c["n"]
  # Experts' shares of the rows: uneven, as a router leaves them; about one expert in eight gets no row.
  share = [0.0 if e > 1 and rng.random() < 0.125 else math.exp(rng.gauss(0.0, 0.5)) for _ in range(e)]
  share[rng.randrange(e)] += 0.5
  ends = [0]
  for i in range(e):
    ends.append(int(round(m * sum(share[:i + 1]) / sum(share))))
  s = {"case": c, "sizes": [b - a for a, b in zip(ends, ends[1:])],
       "offsets": torch.tensor(ends, dtype=torch.int32, device="cuda")}
  s["a"] = rand(m + c["tail"], k).to(torch.bfloat16)
  w = (rand(e, n, k) * k ** -0.5).to(torch.bfloat16)
  # "kn": the processor keeps its weights as [k, n]; the call gets the transposed view.
  s["weight"] = w if c["layout"] == "nk" else w.transpose(1, 2).contiguous().transpose(1, 2)
  s["bias"] = (0.2 * rand(e, n)).to(_DT[c["bias"]]) if c["bias"] != "none" else None
  if c["train"]:
    s["dy"] = (0.01 * rand(m + c["tail"], n)).to(_DT[c["out"]])
    for key in ("a", "weight", "bias"):
      if s[key] is not None:
        s[key].requires_grad_()
  return s


def _prepare_mix(c, seed):
  rand = _randn(seed)
  rows, e, k, d, dt = c["rows"], c["experts"], c["top_k"], c["d"], _DT[c["kind"]]
  s = {"case": c, "logits": rand(rows, e) + 0.5 * rand(e), "x": rand(rows, d).to(dt),
       "y": rand(rows * k, d).to(dt)}          # y: the experts' results, in the order of their rows
  if c["train"]:
    s["d_rows"] = (0.01 * rand(rows * k, d)).to(dt)
    s["d_out"] = (0.01 * rand(rows, d)).to(dt)
    for key in ("logits", "x", "y"):
      s[key].requires_grad_()
  return s


def prepare(case, seed):
  return {"dropout": _prepare_drop, "branch": _prepare_branch, "grouped": _prepare_grouped,
          "mix": _prepare_mix}[case["op"]](case, seed)


# ---- plain forms ----------------------------------------------------------------------------------------------------

_LOW = 0xFFFFFFFF


def _mul32(a, b):
  """High and low 32 bits of a b in 64-bit integers (the product wraps, its bits are right)."""
  t = a * b
  return (t >> 32) & _LOW, t & _LOW


def _keep(shape, seed, site, threshold):
  """True where the generator keeps a value, in the tensor's order."""
  n = math.prod(shape)
  i = torch.arange((n + 7) // 8, dtype=torch.int64, device=seed.device)
  c0, c1, c2, c3 = i & _LOW, i >> 32, torch.full_like(i, site), torch.zeros_like(i)
  k0, k1 = seed & _LOW, (seed >> 32) & _LOW
  for _ in range(10):  # the generator's rounds
    h0, l0 = _mul32(c0, 0xD2511F53)
    h1, l1 = _mul32(c2, 0xCD9E8D57)
    c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
    k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
  words = torch.stack((c0, c1, c2, c3), 1)
  numbers = torch.stack((words & 0xFFFF, words >> 16), 2).reshape(-1)[:n]
  return (numbers >= threshold).reshape(shape)


def _threshold(p):
  return int(round(65536 * p))


def _drop_values(x, keep, p):
  return torch.where(keep, x * (65536.0 / (65536 - _threshold(p))), torch.zeros_like(x))


def _plain_drop(s):
  c = s["case"]
  keep = _keep(s["x"].shape, s["seed"], 3, _threshold(c["p"]))
  return {"y": _drop_values(s["x"].float(), keep, c["p"]).to(s["x"].dtype),
          "d_x": _drop_values(s["dy"].float(), keep, c["p"]).to(s["x"].dtype)}


def _plain_branch(s):
  c = s["case"]
  d = c["d"]
  f = {key: None if s[key] is None else s[key].float() for key in _BRANCH_LEAVES}
  x, y, alpha = f["x"], f["y"], c["scale"]
  gate = None if f["gate"] is None else f["gate"][:, None, :] if c["gate"] == "sample" else f["gate"]
  r1 = 1.0 / torch.sqrt(torch.mean(y * y, -1, keepdim=True) + EPS)
  yhat = y * r1
  z = yhat if f["post_weight"] is None else yhat * f["post_weight"]
  b = z if gate is None else z * gate
  keep = None
  if c["p"] > 0:
    keep = _keep(x.shape, s["seed"], 3, _threshold(c["p"]))
    b = _drop_values(b, keep, c["p"])
  total = alpha * x + b
  r2 = 1.0 / torch.sqrt(torch.mean(total * total, -1, keepdim=True) + EPS)
  shat = total * r2
  h = shat if f["weight"] is None else shat * f["weight"]
  out = {"s": total.to(s["x"].dtype)}
  if c["out"] == "fp8":
    scale = torch.amax(torch.abs(h), -1) / 448.0
    out["values"] = torch.clamp(h / scale[..., None], -448.0, 448.0).to(torch.float8_e4m3fn)
    out["scale"] = scale
    return out
  out["h"] = h.to(_DT[c["out"]])
  if c["train"]:
    dh, ds = s["dh"].float(), s["ds"].float()
    g = dh if f["weight"] is None else dh * f["weight"]
    dt = (g - shat * torch.mean(g * shat, -1, keepdim=True)) * r2 + ds
    out["d_x"] = (alpha * dt).to(s["x"].dtype)
    db = dt if keep is None else _drop_values(dt, keep, c["p"])
    if gate is not None:
      dg = db * z
      dg = dg.sum(1) if c["gate"] == "sample" else dg.sum((0, 1)) if c["gate"] == "channel" else dg
      out["d_gate"] = dg.to(s["gate"].dtype)
      db = db * gate
    if f["weight"] is not None:
      out["d_weight"] = torch.sum((dh * shat).reshape(-1, d), 0).to(s["weight"].dtype)
      out["d_post_weight"] = torch.sum((db * yhat).reshape(-1, d), 0).to(s["post_weight"].dtype)
      db = db * f["post_weight"]
    out["d_y"] = ((db - yhat * torch.mean(db * yhat, -1, keepdim=True)) * r1).to(s["y"].dtype)
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
  p = 1.0 / (1.0 + torch.exp(-x))
  return p * (1.0 + x * (1.0 - p))


def _plain_grouped(s):
  c = s["case"]
  a, w = s["a"], s["weight"]
  y = torch.zeros((a.shape[0], c["n"]), dtype=_DT[c["out"]], device=a.device)
  out = {"y": y}
  if c["train"]:
    out["d_a"], out["d_weight"] = torch.zeros_like(a), torch.zeros_like(w)
    if s["bias"] is not None:
      out["d_bias"] = torch.zeros_like(s["bias"])
  at = 0
  for e, size in enumerate(s["sizes"]):  # one product an expert, as many as their sizes, which differ, make
    if size == 0:
      continue
    rows = slice(at, at + size)
    at += size
    ae, we = a[rows].float(), w[e].float()
    pre = torch.matmul(ae, we.t())
    if s["bias"] is not None:
      pre = pre + s["bias"][e].float()
    y[rows] = _plain_act(pre, c["act"]).to(y.dtype)
    if c["train"]:
      d_pre = s["dy"][rows].float()
      if c["act"] != "none":
        d_pre = d_pre * _plain_act_grad(pre, c["act"])
      out["d_a"][rows] = torch.matmul(d_pre, we).to(a.dtype)
      out["d_weight"][e] = torch.matmul(d_pre.t(), ae).to(w.dtype)
      if s["bias"] is not None:
        out["d_bias"][e] = torch.sum(d_pre, 0).to(s["bias"].dtype)
  return out


def _plain_mix(s):
  c = s["case"]
  e, k, d = c["experts"], c["top_k"], c["d"]
  top, idx = (t[:, :k] for t in torch.sort(s["logits"].float(), dim=1, descending=True, stable=True))
  p = torch.exp(top - top[:, :1])
  w = p / torch.sum(p, 1, keepdim=True)
  flat = idx.reshape(-1)
  order = torch.sort(flat, stable=True)[1]
  position = torch.empty_like(order)
  position[order] = torch.arange(order.numel(), device=order.device)
  counts = torch.sum(flat[None, :] == torch.arange(e, device=flat.device)[:, None], 1)
  offsets = torch.cat((torch.zeros_like(counts[:1]), torch.cumsum(counts, 0)))
  back = s["y"][position].reshape(-1, k, d).float()
  out = {"experts": idx.to(torch.int32), "weights": w, "order": order.to(torch.int32),
         "offsets": offsets.to(torch.int32), "rows": s["x"][order // k], "out": torch.sum(back * w[:, :, None], 1).to(s["x"].dtype)}
  if c["train"]:
    d_out = s["d_out"].float()
    out["d_x"] = torch.sum(s["d_rows"][position].reshape(-1, k, d).float(), 1).to(s["x"].dtype)
    out["d_y"] = (w[:, :, None] * d_out[:, None, :]).reshape(-1, d)[order].to(s["y"].dtype)
    dw = torch.sum(back * d_out[:, None, :], 2)
    d_top = w * (dw - torch.sum(w * dw, 1, keepdim=True))
    out["d_logits"] = torch.zeros_like(s["logits"]).scatter_(1, idx, d_top.to(s["logits"].dtype))
  return out


# ---- the framework's calls ------------------------------------------------------------------------------------------

def _package():
  path = os.path.join(os.getcwd(), "faster-weathernext_b200")
  if path not in sys.path:
    sys.path.insert(0, path)
  from faster_weathernext import branch, experts
  return branch, experts


def _own_drop(s):
  branch, _ = _package()
  y = branch.dropout(s["x"], s["case"]["p"], s["seed"], site=3)
  return {"y": y.detach(), "d_x": torch.autograd.grad(y, s["x"], s["dy"])[0]}


def _own_branch(s):
  c, (branch, _) = s["case"], _package()
  args = s["x"], s["y"], s["post_weight"], s["weight"]
  if c["out"] == "fp8":
    values, scale, total = branch.branch_norm_fp8(*args, gate=s["gate"], residual_scale=c["scale"], eps=EPS)
    return {"s": total, "values": values, "scale": scale}
  h, total = branch.branch_norm(*args, gate=s["gate"], residual_scale=c["scale"], p=c["p"],
                                seed=s["seed"] if c["p"] > 0 else None, site=3, eps=EPS, out_dtype=_DT[c["out"]])
  out = {"s": total.detach(), "h": h.detach()}
  if c["train"]:
    keys = [key for key in _BRANCH_LEAVES if s[key] is not None]
    grads = dict(zip(keys, torch.autograd.grad((h, total), [s[key] for key in keys], (s["dh"], s["ds"]))))
    # In the plain form's order.
    out.update({"d_" + key: grads[key] for key in ("x", "gate", "weight", "post_weight", "y") if key in grads})
  return out


def _own_grouped(s):
  c, (_, experts) = s["case"], _package()
  y = experts.linear_grouped(s["a"], s["weight"], s["offsets"], s["bias"],
                             activation=None if c["act"] == "none" else c["act"], out_dtype=_DT[c["out"]])
  out = {"y": y.detach()}
  if c["train"]:
    keys = [key for key in ("a", "weight", "bias") if s[key] is not None]
    out.update({"d_" + key: v for key, v in zip(keys, torch.autograd.grad(y, [s[key] for key in keys], s["dy"]))})
  return out


def _own_mix(s):
  c, (_, experts) = s["case"], _package()
  routing = experts.route(s["logits"], c["top_k"])
  rows = experts.dispatch(s["x"], routing)
  total = experts.combine(s["y"], routing)
  out = {"experts": routing.experts, "weights": routing.weights.detach(), "order": routing.order,
         "offsets": routing.offsets, "rows": rows.detach(), "out": total.detach()}
  if c["train"]:
    grads = torch.autograd.grad((rows, total), (s["x"], s["y"], s["logits"]), (s["d_rows"], s["d_out"]))
    out.update({"d_x": grads[0], "d_y": grads[1], "d_logits": grads[2]})
  return out


def run(state):
  op = state["case"]["op"]
  if own:
    return {"dropout": _own_drop, "branch": _own_branch, "grouped": _own_grouped, "mix": _own_mix}[op](state)
  with torch.no_grad():
    return {"dropout": _plain_drop, "branch": _plain_branch, "grouped": _plain_grouped, "mix": _plain_mix}[op](state)


# ---- work and exact values ------------------------------------------------------------------------------------------

def _size(name):
  return {"none": 0, "fp8": 1, "bf16": 2, "f32": 4}[name]


def work(case):
  c = case
  if c["op"] == "dropout":
    values = c["rows"] * c["d"]
    return {"bytes": 4 * values * _size(c["kind"]), "flops": 2.0 * values}
  if c["op"] == "branch":
    rows, d = c["samples"] * c["nodes"], c["d"]
    values = rows * d
    st, br, ou = _size(c["stream"]), _size(c["branch"]), _size(c["out"])
    gate = {"none": 0, "channel": 4 * d, "sample": 4 * c["samples"] * d, "value": br * values}[c["gate"]]
    params = gate + 2 * d * _size(c["weight"])
    nbytes = values * (2 * st + br + ou) + params + (4 * rows if c["out"] == "fp8" else 0)
    flops = 12.0 * values
    if c["train"]:
      # What the gradient reads: those of h and s, and the inputs again; and writes: the inputs' gradients.
      nbytes += values * (ou + 3 * st + 2 * br) + 2 * params
      flops += 25.0 * values
    return {"bytes": nbytes, "flops": flops}
  if c["op"] == "grouped":
    m, e, n, k = c["rows"], c["experts"], c["n"], c["k"]
    hit = min(e, m)  # weights of experts that no row goes to are not read
    nbytes = 2 * (m * k + hit * n * k) + (m + c["tail"]) * n * _size(c["out"]) + hit * n * _size(c["bias"])
    flops = 2.0 * m * n * k
    if c["train"]:
      nbytes += m * n * _size(c["out"]) + 2 * 2 * ((m + c["tail"]) * k + e * n * k) + e * n * _size(c["bias"])
      flops *= 3
    return {"bytes": nbytes, "flops": flops}
  rows, e, k, d, es = c["rows"], c["experts"], c["top_k"], c["d"], _size(c["kind"])
  nbytes = 4 * rows * e + 16 * rows * k + rows * d * es * (2 + 2 * k)
  flops = 2.0 * rows * k * d
  if c["train"]:
    nbytes += rows * d * es * (2 + 3 * k) + 4 * rows * e
    flops *= 4
  return {"bytes": nbytes, "flops": flops}


def _philox_keep(n, seed, site, threshold):
  """The generator again, in unsigned NumPy words: keep flags of n values."""
  i = np.arange((n + 7) // 8, dtype=np.uint64)
  mask, s32 = np.uint64(0xFFFFFFFF), np.uint64(32)
  x = [i & mask, i >> s32, np.full_like(i, site), np.zeros_like(i)]
  key = [seed & 0xFFFFFFFF, seed >> 32]
  for r in range(10):
    if r:
      key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    p, q = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
    x = [(q >> s32) ^ x[1] ^ np.uint64(key[0]), q & mask, (p >> s32) ^ x[3] ^ np.uint64(key[1]), p & mask]
  numbers = np.stack(x, 1).astype("<u4").view("<u2").reshape(-1)[:n]
  return numbers >= threshold


def _factor(shape, s, p):
  """The mask with its factor in 64 bits."""
  t = _threshold(p)
  keep = _philox_keep(math.prod(shape), int(s["seed"].item()), 3, t)
  return torch.from_numpy(keep).to("cuda").reshape(shape).double().mul(65536.0).div(65536 - t)


def _leaf(t):
  return None if t is None else t.detach().double().requires_grad_()


def _exact_drop(c, s):
  f = _factor(s["x"].shape, s, c["p"])
  return {"y": torch.mul(f, s["x"].detach().double()), "d_x": torch.mul(f, s["dy"].double())}


def _exact_branch(c, s):
  with torch.enable_grad():
    v = {key: _leaf(s[key]) for key in _BRANCH_LEAVES}
    unit = lambda t: torch.mul(t, torch.rsqrt(t.pow(2).sum(-1).div(c["d"]).add(EPS)).unsqueeze(-1))  # noqa: E731
    add = unit(v["y"])
    if v["post_weight"] is not None:
      add = torch.einsum("bnd,d->bnd", add, v["post_weight"])
    if v["gate"] is not None:
      add = torch.einsum({"channel": "bnd,d->bnd", "sample": "bnd,bd->bnd", "value": "bnd,bnd->bnd"}[c["gate"]], add, v["gate"])
    if c["p"] > 0:
      add = torch.mul(add, _factor(add.shape, s, c["p"]))
    total = torch.add(add, v["x"], alpha=c["scale"])
    h = unit(total)
    if v["weight"] is not None:
      h = torch.einsum("bnd,d->bnd", h, v["weight"])
    out = {"s": total.detach()}
    if c["out"] == "fp8":
      scale = h.detach().abs().max(-1).values.div(448.0)
      out["values"], out["scale"] = h.detach().div(scale.unsqueeze(-1)), scale
      return out
    out["h"] = h.detach()
    if c["train"]:
      keys = [key for key in ("x", "gate", "weight", "post_weight", "y") if v[key] is not None]
      grads = torch.autograd.grad([h, total], [v[key] for key in keys], [s["dh"].double(), s["ds"].double()])
      out.update({"d_" + key: g for key, g in zip(keys, grads)})
  return out


def _exact_grouped(c, s):
  with torch.enable_grad():
    a, w, b = _leaf(s["a"]), _leaf(s["weight"]), _leaf(s["bias"])
    parts = list(torch.split(a[:c["rows"]], s["sizes"]))
    for e, t in enumerate(parts):
      t = torch.einsum("mk,nk->mn", t, w[e])
      if b is not None:
        t = torch.add(t, b[e])
      if c["act"] == "gelu":
        # x sigmoid(2 u): the tanh form written through the logistic function.
        t = t * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (t + 0.044715 * t.pow(3)))
      elif c["act"] == "swish":
        t = t * torch.sigmoid(t)
      parts[e] = t
    parts.append(torch.zeros(c["tail"], c["n"], dtype=torch.float64, device=a.device))
    y = torch.cat(parts)
    out = {"y": y.detach()}
    if c["train"]:
      keys = [key for key, v in (("a", a), ("weight", w), ("bias", b)) if v is not None]
      grads = torch.autograd.grad(y, [{"a": a, "weight": w, "bias": b}[key] for key in keys], s["dy"].double())
      out.update({"d_" + key: g for key, g in zip(keys, grads)})
  return out


def _exact_mix(c, s):
  e, k, d = c["experts"], c["top_k"], c["d"]
  logits = s["logits"].detach().double().cpu().numpy()
  idx = np.argsort(-logits, axis=1, kind="stable")[:, :k]
  order = np.argsort(idx.reshape(-1), kind="stable")
  offsets = np.concatenate(([0], np.cumsum(np.bincount(idx.reshape(-1), minlength=e))))
  dev = s["x"].device
  on = lambda t: torch.from_numpy(np.ascontiguousarray(t)).to(dev)  # noqa: E731
  with torch.enable_grad():
    x, y, lg = _leaf(s["x"]), _leaf(s["y"]), _leaf(s["logits"])
    w = torch.softmax(torch.gather(lg, 1, on(idx)), 1)
    source = on(order // k)
    rows = torch.index_select(x, 0, source)
    pair_weight = torch.index_select(w.reshape(-1), 0, on(order))
    total = torch.zeros(c["rows"], d, dtype=torch.float64, device=dev).index_add(0, source, y * pair_weight.unsqueeze(1))
    out = {"experts": on(idx.astype(np.int32)), "weights": w.detach(), "order": on(order.astype(np.int32)),
           "offsets": on(offsets.astype(np.int32)), "rows": rows.detach(), "out": total.detach()}
    if c["train"]:
      grads = torch.autograd.grad([rows, total], [x, y, lg], [s["d_rows"].double(), s["d_out"].double()])
      out.update({"d_x": grads[0], "d_y": grads[1], "d_logits": grads[2]})
  return out


def exact(case, seed):
  s = prepare(case, seed)
  return {"dropout": _exact_drop, "branch": _exact_branch, "grouped": _exact_grouped, "mix": _exact_mix}[case["op"]](case, s)
