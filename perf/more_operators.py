"""Operators of a residual block's branch, for timing and for comparing one build with another.

The root-mean-square norms after a block and before the next with the block's gate, the residual's scale and
dropout between them, forward and in training; dropout by itself, with a mask that is generated and not kept; and
linear layers of 4-bit weights with a scale for each group of 32 inputs. Where ``own`` is true ``run`` calls the
package's entry points, else it computes the same outputs from elementary torch operations in float32.
"""
import math
import os
import sys

import numpy
import torch

own = False

DEV = "cuda"
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"bf16": 2, "f32": 4}
GROUP = 32


def _norms(name, op, members, n, channels, dtype, gate, scale=1.0, p=0.0, post_norm=True):
  """Rows [members, n, channels]; `gate`: "none", "channel" [channels], "member" [members, channels] or "full"."""
  return dict(name=name, op=op, members=members, n=n, channels=channels, dtype=dtype, gate=gate, scale=scale, p=p,
              post_norm=post_norm)


def _dropout(name, op, rows, channels, dtype, p, residual):
  return dict(name=name, op=op, rows=rows, channels=channels, dtype=dtype, p=p, residual=residual)


def _linear(name, rows, ins, outs, dtype, activation="none", residual=False):
  return dict(name=name, op="q4", rows=rows, ins=ins, outs=outs, dtype=dtype, activation=activation, residual=residual)


def listed():
  return [
      # One token between two blocks of a serving loop: the latency of a call.
      _norms("norms_token", "norms", 1, 1, 4096, "bf16", "channel"),
      # Inference on the 0.25 degree mesh, the gate from the member's conditioning.
      _norms("norms_mesh", "norms", 1, 40962, 768, "bf16", "member"),
      # Fine-tuning of an ensemble on the 1 degree mesh with dropout, a gate for each member.
      _norms("norms_members_train", "norms_train", 4, 10242, 768, "bf16", "member", p=0.1),
      # Full precision training, an odd number of channels, one learned gate, a scaled residual.
      _norms("norms_odd_f32_train", "norms_train", 1, 2562, 1283, "f32", "channel", scale=1.5),
      # A wide block whose branch is gated element by element, in training.
      _norms("norms_gated_train", "norms_train", 2, 2562, 4096, "bf16", "full"),
      # Dropout of a small batch's branch onto the residual: the latency of a step's calls.
      _dropout("dropout_small_train", "dropout_train", 64, 768, "bf16", 0.1, True),
      # The mesh's branch in training, dropped and added to the residual.
      _dropout("dropout_mesh_train", "dropout_train", 40962, 768, "bf16", 0.1, True),
      # A full precision layer's inputs, rows of an odd length, forward.
      _dropout("dropout_odd_f32", "dropout", 10242, 1283, "f32", 0.25, False),
      # One token through a 4-bit layer: the weight's trip from memory.
      _linear("q4_token", 1, 4096, 4096, "bf16"),
      # A serving batch through a wide layer with its activation.
      _linear("q4_rows", 24, 5120, 8192, "bf16", "silu"),
      # A few rows of full precision through a layer of odd sizes.
      _linear("q4_odd_f32", 5, 1283, 2051, "f32", "gelu"),
      # A prompt's tokens at once, and the residual.
      _linear("q4_prompt", 512, 4096, 8192, "bf16", "gelu_tanh", True),
  ]


MOST_ROWS = 40962 * 768           # elements of a drawn norm or dropout
MOST_LINEAR = 512 * 4096 * 8192   # products of a drawn linear layer


def _spread(rng, lo, hi):
  return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _width(rng, lo, hi):
  """A width spread over the logarithm of the range: most are whole 64s, the others whole 8s or any."""
  c = _spread(rng, lo, hi)
  unit = rng.choice([64, 64, 64, 8, 1])
  return max(unit, c // unit * unit)


def draw(rng):
  op = rng.choice(["norms", "norms_train", "norms_train", "dropout", "dropout_train", "q4", "q4", "q4"])
  dtype = rng.choice(["bf16", "bf16", "f32"])
  if op == "q4":
    while True:
      rows, ins, outs = _spread(rng, 1, 2048), _width(rng, 64, 16384), _width(rng, 64, 16384)
      if rows * ins * outs <= MOST_LINEAR // (8 if dtype == "f32" else 1) and ins * outs <= 1 << 27:
        break
    c = _linear("", rows, ins, outs, dtype, rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]),
                rng.random() < 0.5)
  else:
    channels = _width(rng, 64, 8192)
    rows = _spread(rng, 1, min(65536, MOST_ROWS // channels // (2 if dtype == "f32" else 1)))
    p = rng.choice([0.05, 0.1, 0.25, 0.5])
    if op.startswith("norms"):
      members = min(rows, rng.choice([1, 1, 2, 4, 8]))
      c = _norms("", op, members, rows // members, channels, dtype, rng.choice(["none", "channel", "member", "full"]),
                 rng.choice([1.0, 1.0, 0.5, 1.5]), p if op == "norms_train" and rng.random() < 0.6 else 0.0,
                 rng.random() < 0.8)
    else:
      c = _dropout("", op, rows, channels, dtype, p, rng.random() < 0.5)
  del c["name"]
  return c


def prepare(case, seed):
  gen = torch.Generator(device=DEV).manual_seed(seed)
  dtype = DTYPES[case["dtype"]]

  def normal(*shape, std=1.0, mean=0.0, dt=dtype):
    return torch.randn(*shape, generator=gen, device=DEV).mul_(std).add_(mean).to(dt)

  s = dict(case)
  # The generator's state as a training program keeps it on the GPU: a seed and the call's offset.
  s["rng"] = torch.randint(0, 1 << 62, (2,), generator=gen, device=DEV)
  if case["op"].startswith("norms"):
    members, n, c = case["members"], case["n"], case["channels"]
    # A residual stream: its channels differ in size, a few are large.
    size = torch.exp(0.5 * torch.randn(c, generator=gen, device=DEV))
    size[:: max(1, c // 8)] *= 10
    s["x"] = (torch.randn(members, n, c, generator=gen, device=DEV) * size).to(dtype)
    s["y"] = normal(members, n, c, std=3.0)
    s["post_weight"] = normal(c, std=0.1, mean=1.0) if case["post_norm"] else None
    s["pre_weight"] = normal(c, std=0.1, mean=1.0)
    shape = {"none": None, "channel": (c,), "member": (members, c), "full": (members, n, c)}[case["gate"]]
    # A member's gate comes in float32, as the conditioning of the norms does.
    s["gate"] = None if shape is None else normal(*shape, std=0.3, mean=0.8,
                                                  dt=torch.float32 if case["gate"] == "member" else dtype)
    if case["op"] == "norms_train":
      s["g_sum"], s["g_out"] = normal(members, n, c), normal(members, n, c)
      for k in ("x", "y", "post_weight", "pre_weight", "gate"):
        if s[k] is not None:
          s[k].requires_grad_()
    return s
  if case["op"].startswith("dropout"):
    rows, c = case["rows"], case["channels"]
    s["x"] = normal(rows, c)
    s["residual"] = normal(rows, c, std=3.0) if case["residual"] else None
    if case["op"] == "dropout_train":
      s["g"] = normal(rows, c)
      for k in ("x", "residual"):
        if s[k] is not None:
          s[k].requires_grad_()
    return s
  rows, ins, outs = case["rows"], case["ins"], case["outs"]
  s["x"] = normal(rows, ins)
  s["bias"] = normal(outs, std=0.1)
  s["residual"] = normal(rows, outs) if case["residual"] else None
  s["weight"], s["weight_scale"] = _pack(normal(outs, ins, std=ins ** -0.5, dt=torch.float32))
  return s


def _pack(w):
  """(codes [outs, 16 groups], two a byte, the even input in the low half; exponents + 127 [outs, groups]) of the rows
  of float32 w, padded with zeros to whole groups: the nearest 4-bit floats (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives)
  at the least power of two of which a group's largest magnitude is at most seven."""
  outs, ins = w.shape
  groups = (ins + GROUP - 1) // GROUP
  w = torch.nn.functional.pad(w, (0, groups * GROUP - ins)).view(outs, groups, GROUP)
  mantissa, exponent = torch.frexp(w.abs().amax(-1))  # mantissa in [0.5, 1)
  exponent = torch.where(mantissa > 0.875, exponent - 2, exponent - 3).clamp(min=-127)
  v = torch.ldexp(w, -exponent[..., None])
  borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEV)
  codes = torch.bucketize(v.abs(), borders).to(torch.uint8) | (v < 0).to(torch.uint8) << 3
  codes = codes.view(outs, groups * GROUP)
  return codes[:, 0::2] | codes[:, 1::2] << 4, (exponent + 127).to(torch.uint8)


# ---- the plain forms


MASK = 0xffffffff


def _kept(rng, rows, channels, p):
  """(kept [rows, channels], the multiplier of what is kept): Philox-4x32-10 with the seed as its key and (c / 8, row,
  the offset's halves) as its counter gives 8 numbers of 16 bits for channels c .. c + 7 of a row; those below p are dropped."""
  border = round(p * 65536)
  blocks = (channels + 7) // 8
  k0, k1 = rng[0] & MASK, (rng[0] >> 32) & MASK
  c0 = torch.arange(blocks, device=DEV)[None].expand(rows, blocks)
  c1 = torch.arange(rows, device=DEV)[:, None].expand(rows, blocks)
  c2, c3 = (rng[1] & MASK).expand(rows, blocks), ((rng[1] >> 32) & MASK).expand(rows, blocks)
  for i in range(10):
    a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # 64 bits, the sign's among them
    c0, c1, c2, c3 = (b >> 32 & MASK) ^ c1 ^ k0, b & MASK, (a >> 32 & MASK) ^ c3 ^ k1, a & MASK
    k0, k1 = (k0 + 0x9E3779B9) & MASK, (k1 + 0xBB67AE85) & MASK
  halves = [h for c in (c0, c1, c2, c3) for h in (c & 0xffff, c >> 16)]
  u = torch.stack(halves, -1).view(rows, blocks * 8)[:, :channels]
  return u >= border, 65536 / (65536 - border)


def _plain_norms(s):
  x, y, dtype = s["x"].float(), s["y"].float(), s["x"].dtype
  members, n, c = x.shape
  post, pre, gate = (None if s[k] is None else s[k].float() for k in ("post_weight", "pre_weight", "gate"))
  if gate is None:
    gate = torch.ones((), device=DEV)
  per_member = gate.dim() == 2
  if per_member:
    gate = gate[:, None]
  r1 = torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) if s["post_norm"] else torch.ones((), device=DEV)
  if post is None:
    post = torch.ones((), device=DEV)
  normed = y * r1
  b = gate * normed * post
  if s["p"]:
    kept, k = _kept(s["rng"], members * n, c, s["p"])
    kept = kept.view(x.shape)
    b = torch.where(kept, b * k, torch.zeros_like(b))
  total = (s["scale"] * x + b).to(dtype)  # the norm is of the sum as it is stored
  t = total.float()
  r2 = torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS)
  out = (t * r2 * pre).to(dtype)
  if s["op"] == "norms":
    return total, out
  g = s["g_out"].float()
  a = g * pre
  ds = s["g_sum"].float() + r2 * (a - t * (r2 * r2 * (a * t).mean(-1, keepdim=True)))
  db = torch.where(kept, ds * k, torch.zeros_like(ds)) if s["p"] else ds
  d = db * gate * post
  gy = r1 * (d - y * (r1 * r1 * (d * y).mean(-1, keepdim=True))) if s["post_norm"] else d
  grads = [(s["scale"] * ds).to(dtype), gy.to(dtype)]
  if s["post_norm"]:
    grads.append((db * gate * normed).sum((0, 1)).to(dtype))
  grads.append((g * t * r2).sum((0, 1)).to(dtype))
  if s["gate"] is not None:
    gg = db * normed * post
    if per_member:
      gg = gg.sum(1)
    elif gate.dim() == 1:
      gg = gg.sum((0, 1))
    grads.append(gg.to(s["gate"].dtype))
  return (total, out, *grads)


def _plain_dropout(s):
  x, dtype = s["x"].float(), s["x"].dtype
  kept, k = _kept(s["rng"], *x.shape, s["p"])
  out = torch.where(kept, x * k, torch.zeros_like(x))
  if s["residual"] is not None:
    out = out + s["residual"].float()
  out = out.to(dtype)
  if s["op"] == "dropout":
    return out
  g = s["g"].float()
  gx = torch.where(kept, g * k, torch.zeros_like(g)).to(dtype)
  return (out, gx) if s["residual"] is None else (out, gx, s["g"])


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


def _plain_linear(s):
  x = s["x"].float()
  table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=DEV)
  table = torch.cat((table, -table))
  codes = s["weight"]
  w = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), -1)
  w = torch.ldexp(w.view(*s["weight_scale"].shape, GROUP), s["weight_scale"][..., None].int() - 127)
  out = _act(x @ w.view(w.shape[0], -1)[:, :x.shape[1]].t() + s["bias"].float(), s["activation"])
  if s["residual"] is not None:
    out = out + s["residual"].float()
  return out.to(s["x"].dtype)


# ---- the package's calls


def _package():
  path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "faster-weathernext_amd")
  if path not in sys.path:
    sys.path.insert(0, path)
  import faster_weathernext_amd
  return faster_weathernext_amd


def _own_norms(s):
  fwn = _package()
  out = fwn.sandwich_norm(s["x"], s["y"], s["post_weight"], s["pre_weight"], gate=s["gate"], scale=s["scale"],
                          post_norm=s["post_norm"], p=s["p"], rng=s["rng"] if s["p"] else None, eps=EPS)
  if s["op"] == "norms":
    return out
  leaves = [s[k] for k in ("x", "y", "post_weight", "pre_weight", "gate") if s[k] is not None]
  return (*out, *torch.autograd.grad(out, leaves, (s["g_sum"], s["g_out"])))


def _own_dropout(s):
  fwn = _package()
  out = fwn.dropout(s["x"], s["p"], s["rng"], residual=s["residual"])
  if s["op"] == "dropout":
    return out
  leaves = [s[k] for k in ("x", "residual") if s[k] is not None]
  return (out, *torch.autograd.grad(out, leaves, s["g"]))


def _own_linear(s):
  fwn = _package()
  activation = None if s["activation"] == "none" else s["activation"]
  return fwn.linear_act_q4(s["x"], s["weight"].view(torch.float4_e2m1fn_x2),
                           s["weight_scale"].view(torch.float8_e8m0fnu), s["bias"], activation=activation,
                           residual=s["residual"])


def run(state):
  op = state["op"].split("_")[0]
  if own:
    out = {"norms": _own_norms, "dropout": _own_dropout, "q4": _own_linear}[op](state)
  else:
    with torch.no_grad():
      out = {"norms": _plain_norms, "dropout": _plain_dropout, "q4": _plain_linear}[op](state)
  return tuple(t.detach() for t in out) if isinstance(out, tuple) else out.detach()


# ---- what a pass cannot do without


def work(case):
  b = BYTES[case["dtype"]]
  if case["op"] == "q4":
    m, k, n = case["rows"], case["ins"], case["outs"]
    groups = (k + GROUP - 1) // GROUP
    res = m * n * b if case["residual"] else 0
    return {"bytes": n * groups * (GROUP // 2 + 1) + (m * k + n + m * n) * b + res, "flops": 2 * m * k * n}
  train = case["op"].endswith("_train")
  if case["op"].startswith("dropout"):
    n = case["rows"] * case["channels"]
    # x and the residual in, the output out; the gradient in, x's out (the residual's is the gradient itself).
    return {"bytes": n * b * (2 + case["residual"] + 2 * train) + 16, "flops": n * (2 + train)}
  n, c = case["members"] * case["n"] * case["channels"], case["channels"]
  gate = {"none": 0, "channel": c * b, "member": case["members"] * c * 4, "full": n * b}[case["gate"]]
  weights = (1 + case["post_norm"]) * c * b
  # x and y in, the sum and its norm out; two gradients in, two out.
  return {"bytes": n * b * (8 if train else 4) + (gate + weights) * (1 + train), "flops": n * (45 if train else 12)}


# ---- the definitions in 64 bits


def _exact_kept(rng, rows, channels, p):
  """_kept's truth values on the host, in unsigned 64-bit numbers."""
  seed, offset = (int(v) & (2 ** 64 - 1) for v in rng.tolist())
  blocks = -(-channels // 8)
  low = numpy.uint64(MASK)
  kept = numpy.empty((rows, blocks, 8), bool)
  step = max(1, (1 << 16) // blocks)
  for first in range(0, rows, step):
    last = min(rows, first + step)
    shape = (last - first, blocks)
    c = [numpy.broadcast_to(numpy.arange(blocks, dtype=numpy.uint64)[None], shape),
         numpy.broadcast_to(numpy.arange(first, last, dtype=numpy.uint64)[:, None], shape),
         numpy.uint64(offset % 2 ** 32), numpy.uint64(offset // 2 ** 32)]
    for i in range(10):
      key = [numpy.uint64((seed % 2 ** 32 + i * 0x9E3779B9) % 2 ** 32),
             numpy.uint64((seed // 2 ** 32 + i * 0xBB67AE85) % 2 ** 32)]
      left, right = numpy.multiply(c[0], numpy.uint64(0xD2511F53)), numpy.multiply(c[2], numpy.uint64(0xCD9E8D57))
      c = [right // numpy.uint64(2 ** 32) ^ c[1] ^ key[0], right & low,
           left // numpy.uint64(2 ** 32) ^ c[3] ^ key[1], left & low]
    words = numpy.stack([numpy.broadcast_to(w, shape) for w in c], -1).astype("<u4")
    kept[first:last] = words.view("<u2").reshape(*shape, 8) >= round(p * 2 ** 16)
  return torch.from_numpy(kept.reshape(rows, blocks * 8)[:, :channels].copy()).to(DEV)


def exact(case, seed):
  s = prepare(case, seed)
  with torch.no_grad():
    rng = s.pop("rng")
    d = {k: v.detach().double() if isinstance(v, torch.Tensor) and v.dtype.is_floating_point else v for k, v in s.items()}
    if case["op"] == "q4":
      return _exact_linear(d)
    p = case["p"]
    if case["op"].startswith("dropout"):
      multiplier = _exact_kept(rng, case["rows"], case["channels"], p).double() / (1 - round(p * 2 ** 16) / 2 ** 16)
      out = d["x"] * multiplier
      if d["residual"] is not None:
        out += d["residual"]
      if case["op"] == "dropout":
        return out
      return (out, d["g"] * multiplier) + (() if d["residual"] is None else (d["g"],))
    return _exact_norms(case, d, rng)


def _exact_norms(case, d, rng):
  members, n, c = d["x"].shape
  ones = torch.ones(1, 1, c, dtype=torch.float64, device=DEV)
  post = ones if d["post_weight"] is None else d["post_weight"].view(1, 1, c)
  pre = d["pre_weight"].view(1, 1, c)
  gate = {"none": lambda: ones, "channel": lambda: d["gate"].view(1, 1, c),
          "member": lambda: d["gate"].view(members, 1, c), "full": lambda: d["gate"]}[case["gate"]]()
  root = 1 / ((d["y"] ** 2).sum(-1, keepdim=True) / c + EPS).sqrt() if case["post_norm"] else torch.ones_like(d["y"][..., :1])
  unit = d["y"] * root
  multiplier = 1.0
  if case["p"]:
    multiplier = _exact_kept(rng, members * n, c, case["p"]).view(members, n, c).double()
    multiplier /= 1 - round(case["p"] * 2 ** 16) / 2 ** 16
  sums = case["scale"] * d["x"] + multiplier * gate * post * unit
  # The sum is stored in the tensors' type and the norm reads it as stored.
  stored = sums.to(DTYPES[case["dtype"]]).double()
  root2 = 1 / ((stored ** 2).sum(-1, keepdim=True) / c + EPS).sqrt()
  unit2 = stored * root2
  out = unit2 * pre
  if case["op"] == "norms":
    return sums, out
  h = d["g_out"] * pre
  g = d["g_sum"] + root2 * (h - unit2 * (h * unit2).sum(-1, keepdim=True) / c)
  branch = g * multiplier
  q = branch * gate * post
  gy = root * (q - unit * (q * unit).sum(-1, keepdim=True) / c) if case["post_norm"] else q
  grads = [case["scale"] * g, gy]
  if case["post_norm"]:
    grads.append((branch * gate * unit).view(-1, c).sum(0))
  grads.append((d["g_out"] * unit2).view(-1, c).sum(0))
  if case["gate"] != "none":
    of_gate = branch * post * unit
    grads.append({"channel": lambda: of_gate.view(-1, c).sum(0), "member": lambda: of_gate.sum(1),
                  "full": lambda: of_gate}[case["gate"]]())
  return (sums, out, *grads)


def _exact_linear(d):
  codes, (outs, groups) = d["weight"].long(), d["weight_scale"].shape
  codes = torch.stack([codes % 16, codes // 16], 2).view(outs, groups, GROUP)
  # Sign, two bits of exponent, one of mantissa; without an exponent the mantissa is a half.
  exponent, mantissa = codes // 2 % 4, (codes % 2).double()
  value = torch.where(exponent == 0, mantissa / 2, (1 + mantissa / 2) * 2.0 ** (exponent - 1).double())
  value = value * (1 - 2 * (codes // 8)) * 2.0 ** (d["weight_scale"].double() - 127)[..., None]
  z = torch.addmm(d["bias"], d["x"], value.view(outs, groups * GROUP)[:, :d["x"].shape[1]].t())
  kind = d["activation"]
  if kind == "relu":
    z = z.relu()
  elif kind == "gelu":
    z = z * torch.special.ndtr(z)
  elif kind == "gelu_tanh":
    z = z * (2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)).sigmoid()  # (1 + tanh(u)) / 2
  elif kind == "silu":
    z = z * z.sigmoid()
  return z if d["residual"] is None else z + d["residual"]
