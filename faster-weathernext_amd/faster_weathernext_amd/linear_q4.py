"""Linear layers of 4-bit weights with a scale for each group of 32 inputs, beside the 8-bit ones of ``linear_act``.

    weight[o, i] = value(code[o, i]) * 2 ** (scale[o, i // 32] - 127)

The format is the 4-bit one of the OCP microscaling specification: e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
negatives), two a byte with the even input in the low half, and e8m0 scales, 4.25 bits a weight. ``quantize_q4`` makes them of a layer's
weight once; ``linear_act_q4`` is ``linear_act`` with them. Such a weight is exact in bfloat16, so that only x's own type, the
float32 sums and the output's rounding stand between the result and the exact product with the quantised weight. Up to 16 rows of x
are one pass over the codes. More rows of bfloat16 go by an estimate of the time: up to 32 in that pass too, or any number in tiles
that read the codes, with partial sums in a workspace where the sum is split, or over the weight widened into a workspace by the
kernels of ``linear_act``. float32 takes the one pass up to 32 rows and the widened weight beyond. Rows of bfloat16 that are not
whole aligned 16 bytes, and for the tiles scales whose groups are not whole aligned fours, are laid out in the workspace by
each call. No derivative.
"""
import ctypes
import functools

import torch

from . import _native as nat
from .linear_act import _activation, _check_like, _rows
from .rms import _no_grad, dense, launch
from .rows import _DTYPES, _addr

CODES, SCALES = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu


def _groups(ins):
  return -(-ins // nat.Q4_GROUP)


def quantize_q4(weight):
  """(codes [outs, 16 groups] of torch.float4_e2m1fn_x2, scales [outs, groups] of torch.float8_e8m0fnu) of weight [outs, ins],
  float32 or bfloat16 on a GPU, groups = ceil(ins / 32): the nearest codes (middles to even ones) at the least power of two of which
  a group's largest magnitude is at most seven; beyond six it is cut to six. The last group is filled up with zeros; groups with
  NaN or infinities have the scale NaN. Forward only."""
  if not isinstance(weight, torch.Tensor) or not weight.is_cuda:
    raise ValueError("weight must be a CUDA tensor")
  if weight.dtype not in _DTYPES:
    raise TypeError(f"weight must be float32 or bfloat16, got {weight.dtype}")
  if weight.dim() != 2 or not all(1 <= n <= nat.LINEAR_ACT_MAX for n in weight.shape):
    raise ValueError(f"weight must be [outs, ins], each 1 to {nat.LINEAR_ACT_MAX}, got {tuple(weight.shape)}")
  _no_grad("quantize_q4", weight)
  outs, ins = weight.shape
  wr, ws = _rows(weight)
  codes = torch.empty((outs, 16 * _groups(ins)), dtype=torch.uint8, device=weight.device)
  scales = torch.empty((outs, _groups(ins)), dtype=torch.uint8, device=weight.device)
  launch(weight, nat.lib().fwn_quantize_q4_launch, outs, ins, ws, _DTYPES[weight.dtype], _addr(wr), _addr(codes), _addr(scales))
  return codes.view(CODES), scales.view(SCALES)


def _bytes(t, aligned):
  """t's bytes, contiguous and, for the codes, 16-byte aligned."""
  if t.is_contiguous() and not (aligned and t.data_ptr() % 16):
    return t
  t = t.view(torch.uint8)
  return t.clone(memory_format=torch.contiguous_format)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(rows, x_stride, ins, outs, dtype, x_at, scales_at):
  """A call's workspace, a function of its sizes and of how x and the scales lie to 16 bytes (the query takes 2 us of host time)."""
  d, size = nat.LinearDesc(rows, x_stride, 0, 0, ins, outs, dtype, 0), ctypes.c_uint64()
  nat.check(nat.lib().fwn_linear_act_q4_workspace_size(d, 4096 + x_at, 4096 + scales_at, ctypes.byref(size)))
  return size.value


def linear_act_q4(x, weight, weight_scale, bias=None, *, activation=None, residual=None):
  """act(x w^T + bias) + residual with the 4-bit weight w of codes `weight` [outs, 16 groups] (torch.float4_e2m1fn_x2) and
  scales `weight_scale` [outs, groups] (torch.float8_e8m0fnu), as ``quantize_q4`` gives them, groups = ceil(ins / 32). x [..., ins],
  bias [outs] and residual [..., outs] are all float32 or all bfloat16, activation is as in ``linear_act``, and so is the
  precision of the sums: accumulated in float32 and rounded once to x's dtype. Codes past ins are not used; codes that are not
  contiguous or not 16-byte aligned are copied by each call. Forward only."""
  if not isinstance(x, torch.Tensor) or not x.is_cuda:
    raise ValueError("x must be a CUDA tensor")
  if x.dtype not in _DTYPES:
    raise TypeError(f"x must be float32 or bfloat16, got {x.dtype}")
  for t, name, dtype in ((weight, "weight", CODES), (weight_scale, "weight_scale", SCALES)):
    if not isinstance(t, torch.Tensor) or t.get_device() != x.get_device() or t.dim() != 2:
      raise ValueError(f"{name} must be a tensor of two dimensions on the device of x")
    if t.dtype != dtype:
      raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
  if x.dim() < 1 or not 1 <= x.shape[-1] <= nat.LINEAR_ACT_MAX:
    raise ValueError(f"x must be [..., ins] with 1 to {nat.LINEAR_ACT_MAX} ins, got {tuple(x.shape)}")
  ins, outs, lead = x.shape[-1], weight.shape[0], x.shape[:-1]
  groups = _groups(ins)
  if not 1 <= outs <= nat.LINEAR_ACT_MAX or weight.shape[1] != 16 * groups or weight_scale.shape != (outs, groups):
    raise ValueError(f"weight must be [outs, {16 * groups}] and weight_scale [outs, {groups}] for {ins} ins, got "
                     f"{tuple(weight.shape)} and {tuple(weight_scale.shape)}")
  act = _activation(activation)
  if bias is not None:
    _check_like(bias, "bias", (outs,), x.dtype, x)
  if residual is not None:
    _check_like(residual, "residual", (*lead, outs), x.dtype, x)
  _no_grad("linear_act_q4", x, bias, residual)
  xr, xs = _rows(x)
  rr, rs = _rows(residual, nat.LINEAR_ACT_MAX)
  bias, codes, scales = dense(bias), _bytes(weight, True), _bytes(weight_scale, False)
  out = x.new_empty((*lead, outs))
  rows, dtype = x.numel() // ins, _DTYPES[x.dtype]
  d = nat.LinearDesc(rows, xs, 0, rs, ins, outs, dtype, act)
  xa, sa = _addr(xr), _addr(scales)
  size = _workspace_bytes(rows, xs, ins, outs, dtype, xa % 16, sa % 16) if rows else 0
  work = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
  launch(x, nat.lib().fwn_linear_act_q4_launch, d, xa, _addr(codes), sa, _addr(bias), _addr(rr), _addr(out), _addr(work), size)
  return out
