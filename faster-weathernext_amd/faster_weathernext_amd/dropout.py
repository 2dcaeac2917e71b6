"""Dropout whose mask is generated from a counter, forward and backward, and never stored.

    out = kept(row, channel) ? x * m : 0, + residual        # in float32, rounded once to x's dtype

``dropout`` is one HIP pass each way, with the residual's addition that follows a block's branch in the same pass. What is
kept is a function of a seed, an offset and the element's place alone (``include/fwn_rows.h``: 16 bits of
Philox-4x32-10 a channel), so that the backward pass, a recomputed forward pass, tensors of other strides or types, and
another machine drop the same elements. ``sandwich.sandwich_norm`` takes the same numbers.

The state ``rng`` is a pair (seed, offset) of whole numbers, or an int64 tensor of the two on x's device that the kernels
read when they run: a captured graph drops anew at each replay if the program changes it in between. Calls
that should drop independently need another offset (or seed) each; two calls with the same state drop the same places.
The tensor is kept for the backward pass, so it must not change before that (autograd refuses one that did):
a call's offset is a new tensor, or written after the backward pass.
"""
import operator

import torch

from . import _native as nat
from .rms import _needs, dense, launch, new_like, rows_of
from .rows import _DTYPES, _addr, as_torch

_WORD = (1 << 64) - 1


def rng_of(rng, x):
  """(state tensor or None, seed, offset) of an `rng` argument for a call on x's device."""
  if isinstance(rng, torch.Tensor):
    if rng.dtype != torch.int64 or rng.shape != (2,):
      raise ValueError("rng must be a pair (seed, offset) or an int64 tensor of the two")
    if rng.get_device() != x.get_device() or not rng.is_cuda:
      raise ValueError("rng must be on the device of x")
    return dense(rng), 0, 0
  try:
    seed, offset = (operator.index(v) for v in rng)
  except (TypeError, ValueError):
    raise ValueError("rng must be a pair (seed, offset) or an int64 tensor of the two") from None
  return None, seed & _WORD, offset & _WORD


def check_number(v, name):
  """v, refused as a tensor: it would be copied to the host, and get no gradient."""
  if isinstance(v, torch.Tensor):
    raise TypeError(f"{name} must be a number, got a tensor")
  return v


def check_p(p):
  p = float(check_number(p, "p"))
  if not 0 <= p <= 1:
    raise ValueError(f"p must be 0 to 1, got {p}")
  return p


def _forward(x, residual, p, rng):
  """One HIP pass (no autograd); rng as rng_of gives it, or with the state as autograd gives it back."""
  c = x.shape[-1]
  xr, xs = rows_of(x)
  rr, rs = rows_of(residual) if residual is not None else (None, 0)
  out = new_like(x)
  state, seed, offset = rng
  state = dense(state)
  d = nat.DropoutDesc(x.numel() // c, xs, rs, c, _DTYPES[x.dtype], nat.Dropout(p, seed, offset, _addr(state)))
  launch(x, nat.lib().fwn_dropout_launch, d, _addr(xr), _addr(rr), _addr(out))
  return out


def multipliers(shape, like, p, rng):
  """What dropout multiplies elements of this shape by, as a float32 tensor on `like`'s device; no autograd."""
  with torch.no_grad():
    return _forward(torch.ones(shape, dtype=torch.float32, device=like.device), None, p, rng)


def dropped(t, m):
  """float32 t times the multipliers m; zeros where that is zero, whatever t is there."""
  return torch.where(m != 0, t * m, torch.zeros((), dtype=t.dtype, device=t.device))


class _Dropout(torch.autograd.Function):

  @staticmethod
  def forward(ctx, x, residual, p, state, seed, offset):
    ctx.save_for_backward(state)
    ctx.p, ctx.seed, ctx.offset, ctx.shape = p, seed, offset, x.shape
    return _forward(x, residual, p, (state, seed, offset))

  @staticmethod
  def backward(ctx, g):
    state, = ctx.saved_tensors
    need_x, need_r = ctx.needs_input_grad[:2]
    gx = None
    if need_x:
      rng = state, ctx.seed, ctx.offset
      if as_torch(g):
        gx = dropped(g.float(), multipliers(ctx.shape, g, ctx.p, rng)).to(g.dtype)
      else:
        gx = _forward(g, None, ctx.p, rng)
    return gx, g if need_r else None, None, None, None, None


def dropout(x, p, rng, *, residual=None):
  """Each element of x [..., channels] with probability p zero, else times 1 / (1 - p), and the residual of x's shape
  and dtype added: in float32, rounded once to x's dtype. p is taken to the nearest 2^-16, the multiplier being that of the p
  taken; p = 0 keeps and p = 1 drops everything. Dropped elements are zeros whatever they were, NaN included.
  float32 or bfloat16 on a GPU, rows of any stride whose channels are contiguous are read where they lie; fewer than 2^32 rows
  of 1 to 2^30 channels. `rng`: see the module. Differentiable in x and residual (to any order); the residual's gradient is the output's."""
  if not isinstance(x, torch.Tensor) or not x.is_cuda:
    raise ValueError("x must be a CUDA tensor")
  if x.dtype not in _DTYPES:
    raise TypeError(f"x must be float32 or bfloat16, got {x.dtype}")
  if x.dim() < 1 or not 1 <= x.shape[-1] <= nat.DROPOUT_MAX_CHANNELS:
    raise ValueError(f"x must be [..., channels] with 1 to {nat.DROPOUT_MAX_CHANNELS} channels, got shape {tuple(x.shape)}")
  if residual is not None and (not isinstance(residual, torch.Tensor) or residual.shape != x.shape or
                               residual.dtype != x.dtype or residual.get_device() != x.get_device()):
    raise ValueError("residual must be a tensor of x's shape, dtype and device")
  p, rng = check_p(p), rng_of(rng, x)
  if _needs(x, residual):
    return _Dropout.apply(x, residual, p, *rng)
  return _forward(x, residual, p, rng)
