"""Root-mean-square norm of rows with the residual's addition, and 8-bit rows with a scale each.

The layer norms of ``rows`` have these beside them for pre-norm blocks that take the RMS norm:

    s = x + y                                 # in float32, rounded once to x's dtype
    out = s / sqrt(mean(s^2) + eps) * weight  # of the sum as stored; statistics in float32

``rms_norm`` and ``add_rms_norm`` are differentiable in x, y and weight, one HIP pass forward and one
(plus the weight gradient's small reduction) backward. ``rms_norm_q8``, ``add_rms_norm_q8`` and
``quantize_rows`` give the rows as OCP e4m3 values with a float32 scale a row (row = q * scale), the
operands of ``linear_act_q8``; they have no derivative. Tensors are [..., channels], float32 or bfloat16
on a GPU, with any number of rows and 1 to 16,384 channels; rows of any stride are read where they lie
if their channels are contiguous. The weight is [channels] in x's dtype or float32.
"""
import ctypes

import torch
from torch.autograd import forward_ad

from . import _native as nat
from .rows import _DTYPES, _addr, as_torch

_Q8 = torch.float8_e4m3fn


def launch(t, fn, *args):
  """fn(*args, stream) on t's device and its current stream. A call on the current device, as most are,
  spends 0.3 us on that where a device guard and a stream object take 3.5."""
  device = t.get_device()
  if torch._C._cuda_getDevice() == device:
    nat.check(fn(*args, torch._C._cuda_getCurrentRawStream(device)))
    return
  with torch.cuda.device(device):
    nat.check(fn(*args, torch._C._cuda_getCurrentRawStream(device)))


def dense(t):
  return t if t is None or t.is_contiguous() else t.contiguous()


def new_like(t):
  """A contiguous tensor of t's shape, dtype and device."""
  return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def rows_of(t):
  """(t, or its rows [rows, channels] without a copy where its strides allow it; the rows' stride)."""
  c = t.shape[-1]
  if t.is_contiguous():
    return t, c
  if t.numel() == 0:
    return t.reshape(-1, c) if c else t.reshape(0, 0), c
  if t.dim() == 2 and t.stride(1) == 1:
    return t, t.stride(0)
  if t.dim() == 1 and t.stride(0) == 1:
    return t.view(1, c), c
  try:
    v = t.view(-1, c)
  except RuntimeError:
    v = t.contiguous().view(-1, c)
  if v.stride(1) != 1 and c > 1:
    v = v.contiguous()
  return v, v.stride(0)


def _check(x, name, like=None):
  if not isinstance(x, torch.Tensor) or not x.is_cuda:
    raise ValueError(f"{name} must be a CUDA tensor")
  if like is not None:
    if x.shape != like.shape or x.dtype != like.dtype or x.get_device() != like.get_device():
      raise ValueError(f"{name} must be a tensor of x's shape, dtype and device")
    return
  if x.dim() < 1 or not 1 <= x.shape[-1] <= nat.RMS_MAX_CHANNELS:
    raise ValueError(f"{name} must be [..., channels] with 1 to {nat.RMS_MAX_CHANNELS} channels, got shape "
                     f"{tuple(x.shape)}")
  if x.dtype not in _DTYPES:
    raise TypeError(f"{name} must be float32 or bfloat16, got {x.dtype}")


def _check_weight(weight, x):
  if weight is None:
    return
  if not isinstance(weight, torch.Tensor) or weight.get_device() != x.get_device() or weight.shape != x.shape[-1:]:
    raise ValueError(f"weight must be a tensor of shape {tuple(x.shape[-1:])} on the device of x")
  if weight.dtype not in (x.dtype, torch.float32):
    raise TypeError(f"weight must be {x.dtype} or float32, got {weight.dtype}")


def _desc(x, weight, eps, x_stride, y_stride=0):
  c, dtype = x.shape[-1], _DTYPES[x.dtype]
  return nat.RmsDesc(x.numel() // c, x_stride, y_stride, c, dtype, dtype if weight is None else _DTYPES[weight.dtype], eps)


def _forward(x, y, weight, eps, q8):
  """(sum or None, out) or, with q8, (sum or None, q, scale): one HIP pass (no autograd)."""
  xr, xs = rows_of(x)
  yr, ys = rows_of(y) if y is not None else (None, 0)
  weight = dense(weight)
  d = _desc(x, weight, eps, xs, ys)
  s = None if y is None else new_like(x)
  if not q8:
    out = new_like(x)
    launch(x, nat.lib().fwn_rms_norm_launch, d, _addr(xr), _addr(yr), _addr(weight), _addr(s), _addr(out))
    return s, out
  q = x.new_empty(x.shape, dtype=_Q8)
  scale = x.new_empty(x.shape[:-1], dtype=torch.float32)
  launch(x, nat.lib().fwn_rms_norm_q8_launch, d, _addr(xr), _addr(yr), _addr(weight), _addr(s), _addr(q), _addr(scale))
  return s, q, scale


def _dense(t, like):
  return None if t is None else t.to(like.dtype).contiguous()


def _backward(s, weight, eps, g_out, g_sum, need_w):
  """(gradient of the rows, gradient of weight or None): fwn_rms_norm_bwd_launch."""
  s, weight, g_out, g_sum = s.contiguous(), dense(weight), _dense(g_out, s), _dense(g_sum, s)
  d = _desc(s, weight, eps, s.shape[-1])
  L = nat.lib()
  gx = torch.empty_like(s)
  gw = ws = None
  size = ctypes.c_uint64(0)
  if need_w:
    gw = torch.empty_like(weight)
    nat.check(L.fwn_rms_norm_bwd_workspace_size(d, ctypes.byref(size)))
    ws = torch.empty(size.value, dtype=torch.uint8, device=s.device)
  launch(s, L.fwn_rms_norm_bwd_launch, d, _addr(s), _addr(weight), _addr(g_out), _addr(g_sum), _addr(gx), _addr(gw),
         _addr(ws), size.value)
  return gx, gw


def _backward_torch(s, weight, eps, g_out, g_sum):
  """The same gradients as torch operations, for backwards under create_graph or of batched gradients."""
  g, f = g_out.float(), s.float()
  r = torch.rsqrt(f.square().mean(-1, keepdim=True) + eps)
  h = g if weight is None else g * weight.float()
  gx = r * (h - f * r.square() * (h * f).mean(-1, keepdim=True))
  if g_sum is not None:
    gx = gx + g_sum.float()
  gw = None if weight is None else (g * f * r).reshape(-1, s.shape[-1]).sum(0).to(weight.dtype)
  return gx.to(s.dtype), gw


class _RmsNorm(torch.autograd.Function):
  """(x + y, its norm), or the norm alone where y is None. x and weight are kept as they came: of a contiguous copy
  autograd would not know that it is theirs, and a second derivative would miss what comes through it."""

  @staticmethod
  def forward(ctx, x, y, weight, eps):
    s, out = _forward(x, y, weight, eps, False)
    ctx.save_for_backward(x if y is None else s, weight)
    ctx.set_materialize_grads(False)
    ctx.eps = eps
    return out if y is None else (s, out)

  @staticmethod
  def backward(ctx, *grads):
    s, weight = ctx.saved_tensors
    g_sum, g_out = grads if len(grads) == 2 else (None, grads[0])
    need_x, need_y, need_w = ctx.needs_input_grad[:3]
    if g_out is None:
      return (g_sum if need_x else None, g_sum if need_y else None,
              torch.zeros_like(weight) if need_w else None, None)
    if as_torch(g_sum, g_out):
      gx, gw = _backward_torch(s, weight, ctx.eps, g_out, g_sum)
    else:
      gx, gw = _backward(s, weight, ctx.eps, g_out, g_sum, need_w)
    return gx if need_x else None, gx if need_y else None, gw if need_w else None, None


def _no_grad(name, *tensors):
  """Refuses tensors that autograd, backward or forward, would have to differentiate."""
  tensors = [t for t in tensors if isinstance(t, torch.Tensor)]
  if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
    raise RuntimeError(f"{name} has no derivative")
  if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
    raise RuntimeError(f"{name} has no derivative")


def _needs(*tensors):
  """Whether autograd has to see the call (forward mode too: the Function refuses its tangents)."""
  if forward_ad._current_level >= 0:
    return True
  if torch.is_grad_enabled():
    for t in tensors:
      if t is not None and t.requires_grad:
        return True
  return False


def rms_norm(x, weight=None, *, eps=1e-6):
  """x / sqrt(mean(x^2) + eps) * weight over the last dimension (weight None: 1), in x's dtype.
  Differentiable in x and weight."""
  _check(x, "x")
  _check_weight(weight, x)
  if _needs(x, weight):
    return _RmsNorm.apply(x, None, weight, float(eps))
  return _forward(x, None, weight, eps, False)[1]


def add_rms_norm(x, y, weight=None, *, eps=1e-6):
  """(x + y, rms_norm(x + y, weight)) in one pass: a block's residual add with the norm that reads it. The
  sum is added in float32 and rounded once, and the norm is the stored sum's. Differentiable in x, y
  and weight; the gradient of the sum adds to the norm's in the norm's backward pass."""
  _check(x, "x")
  _check(y, "y", x)
  _check_weight(weight, x)
  if _needs(x, y, weight):
    return _RmsNorm.apply(x, y, weight, float(eps))
  return _forward(x, y, weight, eps, False)


def rms_norm_q8(x, weight=None, *, eps=1e-6):
  """(q, scale) of rms_norm(x, weight): OCP e4m3 values [..., channels] (torch.float8_e4m3fn) and a float32
  scale [...] a row, from the norm before any rounding: scale = max(max |row| / 448, 2^-126) and
  q = row * (1 / scale) in float32, rounded to the nearest code (a quotient within 2^-23 of the middle of
  two codes may go to either). A row with NaN gives NaN. Forward only."""
  _check(x, "x")
  _check_weight(weight, x)
  _no_grad("rms_norm_q8", x, weight)
  return _forward(x, None, weight, eps, True)[1:]


def add_rms_norm_q8(x, y, weight=None, *, eps=1e-6):
  """(x + y, q, scale): add_rms_norm with the norm in 8 bits as rms_norm_q8 gives it. Forward only."""
  _check(x, "x")
  _check(y, "y", x)
  _check_weight(weight, x)
  _no_grad("add_rms_norm_q8", x, y, weight)
  return _forward(x, y, weight, eps, True)


def quantize_rows(x):
  """(q, scale) of the rows of x [..., channels] as they are, as rms_norm_q8 quantises them: the weights
  [outs, ins] of ``linear_act_q8``, quantised once. Forward only."""
  _check(x, "x")
  _no_grad("quantize_rows", x)
  xr, xs = rows_of(x)
  d = _desc(x, None, 0.0, xs)
  q = x.new_empty(x.shape, dtype=_Q8)
  scale = x.new_empty(x.shape[:-1], dtype=torch.float32)
  launch(x, nat.lib().fwn_quantize_rows_launch, d, _addr(xr), _addr(q), _addr(scale))
  return q, scale
