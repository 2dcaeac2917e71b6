"""Operators of a pre-norm feed-forward block, for timing and for comparing one build with another.

The root-mean-square norm with the residual's addition, forward, in training and with its output in
8 bits; the matrix product with bias, activation and residual in its epilogue, forward and in training;
and the same product of 8-bit operands. Where ``own`` is true ``run`` calls the package's entry points,
else it computes the same outputs from elementary torch operations in float32.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"bf16": 2, "f32": 4}
E4M3_MAX = 448.0
SCALE_MIN = 2.0 ** -126


def _norm(name, op, rows, channels, dtype):
  return dict(name=name, op=op, rows=rows, channels=channels, dtype=dtype)


def _linear(name, op, rows, ins, outs, dtype, activation="none", residual=False, pad=0):
  """`pad`: columns of the buffer that x is a slice of, past its own."""
  return dict(name=name, op=op, rows=rows, ins=ins, outs=outs, dtype=dtype, activation=activation, residual=residual,
              pad=pad)


def listed():
  return [
      # One token's residual and norm: the latency of a call.
      _norm("norm_token", "norm", 1, 768, "bf16"),
      # The block's norm in training on the 0.25 degree mesh.
      _norm("norm_mesh_train", "norm_train", 40962, 768, "bf16"),
      # Full precision training on a 1 degree ensemble, an odd number of channels.
      _norm("norm_odd_f32_train", "norm_train", 10242, 1283, "f32"),
      # Serving in 8 bits: a few rows of a wide model, then the whole mesh.
      _norm("norm_q8_rows", "norm_q8", 24, 5120, "bf16"),
      _norm("norm_q8_mesh", "norm_q8", 40962, 768, "bf16"),
      # One token through the feed-forward's first layer: the weight's trip from memory.
      _linear("linear_token", "linear", 1, 768, 3072, "bf16", "gelu_tanh"),
      # A serving batch of tokens through a wide layer with the residual.
      _linear("linear_rows", "linear", 24, 4096, 4096, "bf16", "none", True),
      # The feed-forward's first layer on the 0.25 degree mesh, inference.
      _linear("linear_mesh_up", "linear", 40962, 768, 3072, "bf16", "gelu_tanh"),
      # Its second layer with the residual, a training step.
      _linear("linear_mesh_down_train", "linear_train", 40962, 3072, 768, "bf16", "none", True),
      # A small full precision layer with odd sizes in training, its activation's gradient included.
      _linear("linear_odd_f32_train", "linear_train", 2562, 515, 1027, "f32", "gelu", True),
      # The 8-bit layer for a serving batch and on the mesh.
      _linear("linear_q8_rows", "linear_q8", 24, 5120, 5120, "bf16", "silu"),
      _linear("linear_q8_mesh", "linear_q8", 40962, 768, 3072, "bf16", "gelu_tanh"),
  ]


MOST_NORM = 40962 * 768         # elements of a drawn norm
MOST_LINEAR = 40962 * 768 * 3072  # products of a drawn matrix product


def _spread(rng, lo, hi):
  return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _width(rng, lo, hi):
  """A width spread over the logarithm of the range: most are whole 64s, the others whole 8s or any."""
  c = _spread(rng, lo, hi)
  unit = rng.choice([64, 64, 64, 8, 1])
  return max(unit, c // unit * unit)


def draw(rng):
  op = rng.choice(["norm", "norm_train", "norm_q8", "linear", "linear", "linear_train", "linear_train", "linear_q8"])
  if op.startswith("norm"):
    channels = _width(rng, 64, 8192)
    rows = _spread(rng, 1, min(65536, MOST_NORM // channels))
    return dict(op=op, rows=rows, channels=channels, dtype=rng.choice(["bf16", "bf16", "f32"]))
  dtype = "bf16" if op == "linear_q8" else rng.choice(["bf16", "bf16", "f32"])
  most = MOST_LINEAR // (8 if dtype == "f32" else 1)
  while True:
    rows, ins, outs = _spread(rng, 1, 65536), _width(rng, 64, 8192), _width(rng, 64, 8192)
    if rows * ins * outs <= most and rows * max(ins, outs) <= 1 << 28:
      break
  c = _linear("", op, rows, ins, outs, dtype, rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]),
              rng.random() < 0.5, 0 if op == "linear_q8" else rng.choice([0, 0, 0, 64]))
  del c["name"]
  return c


def prepare(case, seed):
  gen = torch.Generator(device=DEV).manual_seed(seed)
  dtype = DTYPES[case["dtype"]]

  def normal(*shape, std=1.0, mean=0.0, dt=dtype):
    return torch.randn(*shape, generator=gen, device=DEV).mul_(std).add_(mean).to(dt)

  train = case["op"].endswith("_train")
  s = dict(case)
  if case["op"].startswith("norm"):
    rows, c = case["rows"], case["channels"]
    # A residual stream: its channels differ in size, a few are large.
    size = torch.exp(0.5 * torch.randn(c, generator=gen, device=DEV))
    size[:: max(1, c // 8)] *= 10
    s["x"] = (torch.randn(rows, c, generator=gen, device=DEV) * size).to(dtype)
    s["y"] = normal(rows, c)
    s["weight"] = normal(c, std=0.1, mean=1.0)
    if train:
      s["g_sum"], s["g_out"] = normal(rows, c), normal(rows, c)
      for k in ("x", "y", "weight"):
        s[k].requires_grad_()
    return s
  rows, ins, outs = case["rows"], case["ins"], case["outs"]
  x = normal(rows, ins + case["pad"])[:, :ins]
  weight = normal(outs, ins, std=ins ** -0.5)
  s["bias"] = normal(outs, std=0.1)
  s["residual"] = normal(rows, outs) if case["residual"] else None
  if case["op"] == "linear_q8":
    s["x"], s["x_scale"] = _quantize(x.float())
    s["weight"], s["weight_scale"] = _quantize(weight.float())
    return s
  s["x"], s["weight"] = x, weight
  if train:
    s["g"] = normal(rows, outs)
    for k in ("x", "weight", "bias", "residual"):
      if s[k] is not None:
        s[k].requires_grad_()
  return s


# ---- the plain forms


def _quantize(v):
  """(e4m3 values, scale) of each row of float32 v."""
  scale = torch.clamp(v.abs().amax(-1) / E4M3_MAX, min=SCALE_MIN)
  return torch.clamp(v / scale[:, None], -E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


def _act(z, activation):
  if activation == "relu":
    return torch.clamp(z, min=0)
  if activation == "gelu":
    return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
  if activation == "gelu_tanh":
    return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
  if activation == "silu":
    return z * torch.sigmoid(z)
  return z


def _act_gradient(z, activation):
  if activation == "relu":
    return (z > 0).to(z.dtype)
  if activation == "gelu":
    return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
  if activation == "gelu_tanh":
    t = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z))
    return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
  if activation == "silu":
    g = torch.sigmoid(z)
    return g * (1 + z * (1 - g))
  return torch.ones_like(z)


def _plain_norm(s):
  dtype = s["x"].dtype
  total = (s["x"].float() + s["y"].float()).to(dtype)  # the norm is of the sum as it is stored
  t, w = total.float(), s["weight"].float()
  r = torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS)
  v = t * r * w
  if s["op"] == "norm_q8":
    return (total, *_quantize(v))
  if s["op"] == "norm":
    return total, v.to(dtype)
  g = s["g_out"].float()
  h = g * w
  gx = (s["g_sum"].float() + r * h - t * (r ** 3 * (h * t).mean(-1, keepdim=True))).to(dtype)
  return total, v.to(dtype), gx, gx, (g * t * r).sum(0).to(dtype)


def _plain_linear(s):
  x, w = s["x"].float(), s["weight"].float()
  z = x @ w.t()
  if s["op"] == "linear_q8":
    z = z * s["x_scale"][:, None] * s["weight_scale"]
  z = z + s["bias"].float()
  out = _act(z, s["activation"])
  if s["residual"] is not None:
    out = out + s["residual"].float()
  dtype = DTYPES[s["dtype"]]
  out = out.to(dtype)
  if s["op"] != "linear_train":
    return out
  dz = s["g"].float() * _act_gradient(z, s["activation"])
  grads = [dz @ w, dz.t() @ x, dz.sum(0)] + ([s["g"]] if s["residual"] is not None else [])
  return (out, *(t.to(dtype) for t in grads))


# ---- the package's calls


def _package():
  path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "faster-weathernext_amd")
  if path not in sys.path:
    sys.path.insert(0, path)
  import faster_weathernext_amd
  return faster_weathernext_amd


def _own_norm(s):
  fwn = _package()
  if s["op"] == "norm_q8":
    return fwn.add_rms_norm_q8(s["x"], s["y"], s["weight"], eps=EPS)
  total, out = fwn.add_rms_norm(s["x"], s["y"], s["weight"], eps=EPS)
  if s["op"] == "norm":
    return total, out
  grads = torch.autograd.grad((total, out), (s["x"], s["y"], s["weight"]), (s["g_sum"], s["g_out"]))
  return (total, out, *grads)


def _own_linear(s):
  fwn = _package()
  activation = None if s["activation"] == "none" else s["activation"]
  if s["op"] == "linear_q8":
    return fwn.linear_act_q8(s["x"], s["x_scale"], s["weight"], s["weight_scale"], s["bias"], activation=activation,
                             residual=s["residual"], dtype=DTYPES[s["dtype"]])
  out = fwn.linear_act(s["x"], s["weight"], s["bias"], activation=activation, residual=s["residual"])
  if s["op"] == "linear":
    return out
  leaves = [s[k] for k in ("x", "weight", "bias", "residual") if s[k] is not None]
  return (out, *torch.autograd.grad(out, leaves, s["g"]))


def run(state):
  norm = state["op"].startswith("norm")
  if own:
    out = _own_norm(state) if norm else _own_linear(state)
  else:
    with torch.no_grad():
      out = _plain_norm(state) if norm else _plain_linear(state)
  return tuple(t.detach() for t in out) if isinstance(out, tuple) else out.detach()


# ---- what a pass cannot do without


def work(case):
  b = BYTES[case["dtype"]]
  if case["op"].startswith("norm"):
    rows, c = case["rows"], case["channels"]
    n = rows * c
    if case["op"] == "norm":
      return {"bytes": 4 * n * b + c * b, "flops": 6 * n}
    if case["op"] == "norm_q8":
      return {"bytes": 3 * n * b + n + 4 * rows + c * b, "flops": 9 * n}
    # x, y and the two gradients in; the sum, the norm and the rows' gradient out; the weight and its gradient.
    return {"bytes": 7 * n * b + 2 * c * b, "flops": 20 * n}
  m, k, n = case["rows"], case["ins"], case["outs"]
  product, res = 2 * m * k * n, m * n * b if case["residual"] else 0
  if case["op"] == "linear_q8":
    return {"bytes": m * k + n * k + 4 * (m + n) + n * b + m * n * b + res, "flops": product}
  forward = (m * k + n * k + n + m * n) * b + res
  if case["op"] == "linear":
    return {"bytes": forward, "flops": product}
  # The output's gradient in; those of x, the weight and the bias out.
  return {"bytes": forward + (m * n + m * k + n * k + n) * b, "flops": 3 * product}


# ---- the definitions in 64 bits


def exact(case, seed):
  s = prepare(case, seed)
  with torch.no_grad():
    d = {k: v.detach().double() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    if case["op"].startswith("norm"):
      # The sum is stored in the tensors' type and the norm reads it as stored.
      t = (d["x"] + d["y"]).to(DTYPES[case["dtype"]]).double()
      root = ((t ** 2).sum(1) / case["channels"] + EPS).sqrt()[:, None]
      unit = t / root
      v = unit * d["weight"]
      if case["op"] == "norm_q8":
        return d["x"] + d["y"], None, (v.abs().max(1).values / E4M3_MAX).clamp(min=SCALE_MIN)
      if case["op"] == "norm":
        return d["x"] + d["y"], v
      h = d["g_out"] * d["weight"]
      gx = d["g_sum"] + (h - unit * (h * unit).sum(1, keepdim=True) / case["channels"]) / root
      return d["x"] + d["y"], v, gx, gx, (d["g_out"] * unit).sum(0)
    x, w = d["x"], d["weight"]
    if case["op"] == "linear_q8":
      x, w = x * d["x_scale"][:, None], w * d["weight_scale"][:, None]
    z = torch.addmm(d["bias"], x, w.t())
    kind = case["activation"]
    cube = math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    if kind == "relu":
      a, slope = z.relu(), (z > 0).double()
    elif kind == "gelu":
      phi = torch.special.ndtr(z)
      a, slope = z * phi, phi + z * (z ** 2 / -2).exp() / math.sqrt(2 * math.pi)
    elif kind == "gelu_tanh":
      p = (2 * cube).sigmoid()  # (1 + tanh(u)) / 2
      a, slope = z * p, p + z * 2 * p * (1 - p) * math.sqrt(2 / math.pi) * (1 + 0.134145 * z ** 2)
    elif kind == "silu":
      p = z.sigmoid()
      a, slope = z * p, p + z * p * (1 - p)
    else:
      a, slope = z, torch.ones_like(z)
    out = a if d["residual"] is None else a + d["residual"]
    if case["op"] != "linear_train":
      return out
    dz = d["g"] * slope
    grads = (torch.mm(dz, w), torch.mm(dz.t(), x), dz.sum(0))
    return (out, *grads) if d["residual"] is None else (out, *grads, d["g"])
