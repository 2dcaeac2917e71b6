"""Linear layers with bias, activation and residual in the epilogue of their matrix product.

    linear_act(x, weight, bias, activation=..., residual=...) = act(x weight^T + bias) + residual

A feed-forward's first layer with its activation, its second with the block's residual, each one product
whose epilogue does the rest, in the kernels of ``csrc/linear_act.hip``. Products accumulate in float32
and the output is rounded once; float32 tensors keep float32's precision. ``linear_act`` is
differentiable in x, weight, bias and residual; ``linear_act_q8`` takes the 8-bit rows of ``rms``, adds in float32
for float32 outputs and on the e4m3 matrix units for bfloat16 ones, and has no derivative.
"""
import ctypes

import torch

from . import _native as nat
from .rms import _Q8, _needs, _no_grad, dense, launch, rows_of
from .rows import _DTYPES, _addr, as_torch


def _check(x, weight, bias, residual, dtype, lead):
  if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
    raise ValueError(f"weight must be [outs, ins] and x [..., ins], got {tuple(weight.shape)} and {tuple(x.shape)}")
  outs, ins = weight.shape
  if not (1 <= outs <= nat.LINEAR_ACT_MAX and 1 <= ins <= nat.LINEAR_ACT_MAX):
    raise ValueError(f"weight's sizes must be 1 to {nat.LINEAR_ACT_MAX}, got {tuple(weight.shape)}")
  if bias is not None:
    _check_like(bias, "bias", (outs,), dtype, x)
  if residual is not None:
    _check_like(residual, "residual", (*lead, outs), dtype, x)


def _check_like(t, name, shape, dtype, x):
  if not isinstance(t, torch.Tensor) or t.get_device() != x.get_device() or t.shape != shape:
    raise ValueError(f"{name} must be a tensor of shape {tuple(shape)} on the device of x")
  if t.dtype != dtype:
    raise TypeError(f"{name} must be {dtype}, got {t.dtype}")


def _rows(t, most=nat.LINEAR_STRIDE_MAX):
  """(t's rows, their stride) as the launches take them: at most `most` elements apart (a residual's LINEAR_ACT_MAX)."""
  if t is None:
    return None, 0
  rows, stride = rows_of(t)
  return (rows, stride) if stride <= most else (rows.contiguous(), rows.shape[-1])


def _activation(name):
  if name not in nat.ACTIVATIONS:
    raise ValueError(f"unknown activation {name!r} ({', '.join(str(a) for a in nat.ACTIVATIONS)})")
  return nat.ACTIVATIONS[name]


def _workspace(query, d, like, *addresses):
  size = ctypes.c_uint64()
  nat.check(query(d, *addresses, ctypes.byref(size)))
  return (torch.empty(size.value, dtype=torch.uint8, device=like.device) if size.value else None), size.value


def _forward(x, weight, bias, residual, activation, keep):
  """(act(x weight^T + bias) + residual, the pre-activation or None), without autograd."""
  lead, (outs, ins) = x.shape[:-1], weight.shape
  xr, xs = _rows(x)
  wr, ws = _rows(weight)
  rr, rs = _rows(residual, nat.LINEAR_ACT_MAX)
  bias = dense(bias)
  L = nat.lib()
  out = x.new_empty((*lead, outs))
  pre = torch.empty_like(out) if keep else None
  d = nat.LinearDesc(x.numel() // ins, xs, ws, rs, ins, outs, _DTYPES[x.dtype], activation)
  xa, wa = _addr(xr), _addr(wr)
  work, size = _workspace(L.fwn_linear_act_workspace_size, d, x, xa, wa)
  launch(x, L.fwn_linear_act_launch, d, xa, wa, _addr(bias), _addr(rr), _addr(out), _addr(pre), _addr(work), size)
  return out, pre


def _slope(z, activation):
  """act'(z) of float32 z, as torch operations."""
  if activation == nat.ACTIVATIONS["relu"]:
    return (z > 0).to(z.dtype)
  if activation == nat.ACTIVATIONS["gelu"]:
    return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (0.5 / torch.pi) ** 0.5
  if activation == nat.ACTIVATIONS["gelu_tanh"]:
    c = (2 / torch.pi) ** 0.5
    t = torch.tanh(c * (z + 0.044715 * z ** 3))
    return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
  if activation == nat.ACTIVATIONS["silu"]:
    s = torch.sigmoid(z)
    return s * (1 + z * (1 - s))
  return torch.ones_like(z)


def _backward_torch(x, weight, bias, g, activation, needs):
  """The gradients of x, weight and bias as torch operations, for backwards under create_graph (which
  differentiate the pre-activation too: it is formed anew) or of batched gradients."""
  dz = g.float()
  if activation:
    z = torch.matmul(x.float(), weight.float().t())
    dz = dz * _slope(z if bias is None else z + bias.float(), activation)
  rows = lambda t: t.reshape(-1, t.shape[-1])
  return (torch.matmul(dz, weight.float()).to(g.dtype) if needs[0] else None,
          torch.mm(rows(dz).t(), rows(x).float()).to(g.dtype) if needs[1] else None,
          rows(dz).sum(0).to(g.dtype) if needs[2] else None)


class _LinearAct(torch.autograd.Function):
  """Without an activation x is kept for the weight's gradient alone and the weight for x's; with one the
  pre-activation is kept beside them."""

  @staticmethod
  def forward(ctx, x, weight, bias, residual, activation):
    need_x, need_w, need_b = ctx.needs_input_grad[:3]
    act = activation != 0 and (need_x or need_w or need_b)
    out, pre = _forward(x, weight, bias, residual, activation, act)
    ctx.save_for_backward(x if need_w or act else None, weight if need_x or act else None, bias if act else None, pre)
    ctx.sizes, ctx.activation = (x.shape, weight.shape), activation
    return out

  @staticmethod
  def backward(ctx, g):
    x, weight, bias, pre = ctx.saved_tensors
    (x_shape, (outs, ins)), act = ctx.sizes, ctx.activation
    needs = need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
    g_res = g if need_r else None
    if not (need_x or need_w or need_b):
      return None, None, None, g_res, None
    if as_torch(g):
      return (*_backward_torch(x, weight, bias, g, act, needs), g_res, None)
    g = dense(g)
    xr, xs = _rows(x) if need_w else (None, 0)
    wr, ws = _rows(weight) if need_x else (None, 0)
    d = nat.LinearDesc(g.numel() // outs, xs, ws, 0, ins, outs, _DTYPES[g.dtype], act)
    L = nat.lib()
    gx = g.new_empty(x_shape) if need_x else None
    gw = g.new_empty((outs, ins)) if need_w else None
    gb = g.new_empty(outs) if need_b else None
    xa, wa, ga, gxa, gwa, gba = _addr(xr), _addr(wr), _addr(g), _addr(gx), _addr(gw), _addr(gb)
    work, size = _workspace(L.fwn_linear_act_bwd_workspace_size, d, g, xa, wa, ga, gxa, gwa, gba)
    launch(g, L.fwn_linear_act_bwd_launch, d, xa, wa, _addr(pre), ga, gxa, gwa, gba, _addr(work), size)
    return gx, gw, gb, g_res, None


def linear_act(x, weight, bias=None, *, activation=None, residual=None):
  """act(x weight^T + bias) + residual for x [..., ins], weight [outs, ins], bias [outs] and residual
  [..., outs], all float32 or all bfloat16: a Linear layer with its activation (None, "relu", "gelu",
  "gelu_tanh" or "silu") and the residual's addition in the product's epilogue. Accumulated in float32 and
  rounded once. Rows of any stride are read where they lie if their channels are contiguous.
  Differentiable in x, weight, bias and residual. With an activation the backward keeps the pre-activation in the
  tensors' dtype and rounds the gradient in front of it to that for its products: bfloat16 gradients are off by 2.4e-3
  (relative) where the formula in float32, rounded once, is by 1.7e-3, as those of separate bfloat16 layers."""
  if not isinstance(x, torch.Tensor) or not x.is_cuda:
    raise ValueError("x must be a CUDA tensor")
  if x.dtype not in _DTYPES:
    raise TypeError(f"x must be float32 or bfloat16, got {x.dtype}")
  if not isinstance(weight, torch.Tensor) or weight.get_device() != x.get_device():
    raise ValueError("weight must be a tensor on the device of x")
  if weight.dtype != x.dtype:
    raise TypeError(f"weight must be {x.dtype}, got {weight.dtype}")
  act = _activation(activation)
  _check(x, weight, bias, residual, x.dtype, x.shape[:-1])
  if not _needs(x, weight, bias, residual):
    return _forward(x, weight, bias, residual, act, False)[0]
  return _LinearAct.apply(x, weight, bias, residual, act)


def linear_act_q8(x, x_scale, weight, weight_scale, bias=None, *, activation=None, residual=None, dtype=torch.bfloat16):
  """linear_act of 8-bit operands: x [..., ins] and weight [outs, ins] are e4m3 values
  (torch.float8_e4m3fn) with float32 scales x_scale [...] a row and weight_scale [outs] a column of the
  output, as ``rms_norm_q8`` and ``quantize_rows`` give them; act((x weight^T) x_scale weight_scale + bias) +
  residual in `dtype`, which bias and residual have. float32 outputs, and those of up to 32 rows, are float32 sums
  of exact products; bfloat16 ones of more rows come from the e4m3 matrix units, which add eight products at a
  time with 13 bits below the largest (1.4e-5 of the rows' norms, a hundredth of a bfloat16 output's
  rounding; at most 2^-10 of the sum of the products' magnitudes). Forward only."""
  if not isinstance(x, torch.Tensor) or not x.is_cuda:
    raise ValueError("x must be a CUDA tensor")
  if not isinstance(weight, torch.Tensor) or weight.get_device() != x.get_device():
    raise ValueError("weight must be a tensor on the device of x")
  if x.dtype != _Q8 or weight.dtype != _Q8:
    raise TypeError(f"x and weight must be {_Q8}, got {x.dtype} and {weight.dtype}")
  if dtype not in _DTYPES:
    raise TypeError(f"dtype must be float32 or bfloat16, got {dtype}")
  act = _activation(activation)
  lead = x.shape[:-1]
  _check(x, weight, bias, residual, dtype, lead)
  _check_like(x_scale, "x_scale", lead, torch.float32, x)
  _check_like(weight_scale, "weight_scale", weight.shape[:1], torch.float32, x)
  _no_grad("linear_act_q8", x, x_scale, weight, weight_scale, bias, residual)
  outs, ins = weight.shape
  xr, xs = _rows(x)
  wr, ws = _rows(weight)
  rr, rs = _rows(residual, nat.LINEAR_ACT_MAX)
  bias = dense(bias)
  x_scale, weight_scale = dense(x_scale), dense(weight_scale)
  L = nat.lib()
  out = torch.empty((*lead, outs), dtype=dtype, device=x.device)
  d = nat.LinearDesc(x.numel() // ins, xs, ws, rs, ins, outs, _DTYPES[dtype], act)
  xa, wa = _addr(xr), _addr(wr)
  work, size = _workspace(L.fwn_linear_act_q8_workspace_size, d, x, xa, wa)
  launch(x, L.fwn_linear_act_q8_launch, d, xa, _addr(x_scale), wa, _addr(weight_scale), _addr(bias), _addr(rr), _addr(out),
         _addr(work), size)
  return out
