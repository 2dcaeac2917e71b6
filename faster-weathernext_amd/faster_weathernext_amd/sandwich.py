"""The norms after a block and before the next one, with the block's gate, the residual's scale and dropout between them.

    s = scale * x + dropout(gate * rms_norm(y) * post_weight)      # in float32, rounded once to x's dtype
    out = rms_norm(s) * pre_weight                                 # of the sum as stored

for the residual x and the output y of an attention or feed-forward block, as blocks have it that norm their output
("sandwich" norms), gate their branch (a learned gate a channel, or one a member from the conditioning vector as
``NormConditioning`` gives its multipliers, or one an element), scale the residual, and drop in training. ``sandwich_norm`` is
one HIP pass forward and one, plus the small reductions of the weights' and the gate's gradients, backward.
"""
import ctypes
import functools

import torch

from . import _native as nat
from .dropout import check_number, check_p, dropped, multipliers, rng_of
from .rms import _check, _needs, dense, launch, new_like, rows_of
from .rows import _DTYPES, _addr, as_torch


def _check_weight(t, name, x):
  if t is None:
    return
  if not isinstance(t, torch.Tensor) or t.get_device() != x.get_device() or t.shape != x.shape[-1:]:
    raise ValueError(f"{name} must be a tensor of shape {tuple(x.shape[-1:])} on the device of x")
  if t.dtype not in (x.dtype, torch.float32):
    raise TypeError(f"{name} must be {x.dtype} or float32, got {t.dtype}")


def _gate_rows(gate, x):
  """How many rows of x share a row of the gate."""
  rows = x.numel() // x.shape[-1]
  if gate is None:
    return rows
  if not isinstance(gate, torch.Tensor) or gate.get_device() != x.get_device():
    raise ValueError("gate must be a tensor on the device of x")
  if gate.dtype not in (x.dtype, torch.float32):
    raise TypeError(f"gate must be {x.dtype} or float32, got {gate.dtype}")
  if gate.shape == x.shape:
    return 1
  if gate.shape == x.shape[-1:]:
    return max(rows, 1)
  if x.dim() > 2 and gate.shape == (x.shape[0], x.shape[-1]):
    return max(rows // x.shape[0], 1) if x.shape[0] else 1
  raise ValueError(f"gate must be [channels], x's shape {tuple(x.shape)}, or [members, channels] for x of "
                   f"[members, ..., channels], got {tuple(gate.shape)}")


def _kind(t, dtype):
  return dtype if t is None else _DTYPES[t.dtype]


@functools.lru_cache(maxsize=256)
def _workspace_bytes(rows, gate_rows, channels, dtype, gate):
  """The backward's workspace, a function of the sizes alone (the query takes 3 us of host time)."""
  d = nat.SandwichDesc(rows, gate_rows, channels, channels, channels, dtype, dtype, dtype, dtype, 1, 0.0, 1.0, nat.Dropout(0.0, 0, 0, None))
  size = ctypes.c_uint64(0)
  nat.check(nat.lib().fwn_sandwich_norm_bwd_workspace_size(d, gate, ctypes.byref(size)))
  return size.value


def _for_launch(d, x_stride, y_stride, state):
  """d for one launch: a copy of its own, as passes over one graph may run at once, with the address of the state that the launch
  holds. What autograd gives back of a saved state may be another tensor than the forward pass had (hooks, checkpoints)."""
  d = nat.SandwichDesc.from_buffer_copy(d)
  d.x_stride, d.y_stride, d.drop.state = x_stride, y_stride, _addr(state)
  return d


def _forward(x, y, post, pre, gate, state, d):
  """(s, out): one HIP pass (no autograd)."""
  xr, xs = rows_of(x)
  yr, ys = rows_of(y)
  d = _for_launch(d, xs, ys, state)
  post, pre, gate = dense(post), dense(pre), dense(gate)
  s, out = new_like(x), new_like(x)
  launch(x, nat.lib().fwn_sandwich_norm_launch, d, _addr(xr), _addr(yr), _addr(gate), _addr(post), _addr(pre), _addr(s),
         _addr(out))
  return s, out


def _backward(s, y, post, pre, gate, state, d, g_sum, g_out, needs):
  """The gradients that `needs` asks for of x, y, post, pre and gate: fwn_sandwich_norm_bwd_launch."""
  if not s.numel():
    return tuple(torch.zeros_like(t) if n else None for t, n in zip((s, y, post, pre, gate), needs))
  yr, ys = rows_of(y)
  state = dense(state)
  d = _for_launch(d, 0, ys, state)
  s, post, pre, gate, g_sum, g_out = dense(s), dense(post), dense(pre), dense(gate), dense(g_sum), dense(g_out)
  need_x, need_y, need_post, need_pre, need_gate = needs
  gx = torch.empty_like(s) if need_x else None
  gy = torch.empty_like(s) if need_y else None
  g_post = torch.empty_like(post) if need_post else None
  g_pre = torch.empty_like(pre) if need_pre else None
  g_gate = torch.empty_like(gate) if need_gate else None
  ws, size = None, 0
  if need_post or need_pre or (need_gate and d.gate_rows > 1):
    size = _workspace_bytes(d.rows, d.gate_rows, d.channels, d.dtype, gate is not None)
    ws = torch.empty(size, dtype=torch.uint8, device=s.device)
  launch(s, nat.lib().fwn_sandwich_norm_bwd_launch, d, _addr(s), _addr(yr), _addr(gate), _addr(post), _addr(pre), _addr(g_sum),
         _addr(g_out), _addr(gx), _addr(gy), _addr(g_gate), _addr(g_post), _addr(g_pre), _addr(ws), size)
  return gx, gy, g_post, g_pre, g_gate


def _backward_torch(s, y, post, pre, gate, state, d, g_sum, g_out, needs):
  """The same gradients as torch operations, for backwards under create_graph or of batched gradients."""
  c = s.shape[-1]
  one = torch.ones((), device=s.device)
  f, z = s.float(), y.float()
  w_post, w_pre = (one if t is None else t.float() for t in (post, pre))
  per_member = gate is not None and gate.shape != s.shape and gate.dim() == 2
  w_gate = one if gate is None else gate.float()
  if per_member:
    w_gate = w_gate.reshape(gate.shape[0], *[1] * (s.dim() - 2), c)
  ds = torch.zeros_like(f) if g_sum is None else g_sum.float()
  r2 = torch.rsqrt(f.square().mean(-1, keepdim=True) + d.eps)
  if g_out is not None:
    a = g_out.float() * w_pre
    ds = ds + r2 * (a - f * r2.square() * (a * f).mean(-1, keepdim=True))
  db = ds
  if d.drop.p > 0:
    db = dropped(ds, multipliers(s.shape, s, d.drop.p, (state, d.drop.seed, d.drop.offset)))
  r1 = torch.rsqrt(z.square().mean(-1, keepdim=True) + d.eps) if d.post_norm else one
  unit, q = z * r1, db * w_gate * w_post
  gy = r1 * (q - z * r1.square() * (q * z).mean(-1, keepdim=True)) if d.post_norm else q
  need_x, need_y, need_post, need_pre, need_gate = needs
  g_post = (db * w_gate * unit).reshape(-1, c).sum(0).to(post.dtype) if need_post else None
  g_pre = None
  if need_pre:
    g_pre = torch.zeros_like(pre) if g_out is None else (g_out.float() * f * r2).reshape(-1, c).sum(0).to(pre.dtype)
  g_gate = None
  if need_gate:
    g_gate = db * unit * w_post
    if per_member:
      g_gate = g_gate.reshape(gate.shape[0], -1, c).sum(1)
    elif gate.shape != s.shape:
      g_gate = g_gate.reshape(-1, c).sum(0)
    g_gate = g_gate.to(gate.dtype)
  return (d.scale * ds).to(s.dtype) if need_x else None, gy.to(s.dtype) if need_y else None, g_post, g_pre, g_gate


class _Sandwich(torch.autograd.Function):
  """Tensors are kept as they came: of a contiguous copy autograd would not know whose it is, and a second derivative would
  miss what comes through it."""

  @staticmethod
  def forward(ctx, x, y, post, pre, gate, state, d):
    s, out = _forward(x, y, post, pre, gate, state, d)
    ctx.save_for_backward(s, y, post, pre, gate, state)
    ctx.set_materialize_grads(False)
    ctx.desc = d
    return s, out

  @staticmethod
  def backward(ctx, g_sum, g_out):
    if g_sum is None and g_out is None:
      return (None,) * 7
    run = _backward_torch if as_torch(g_sum, g_out) else _backward
    return (*run(*ctx.saved_tensors, ctx.desc, g_sum, g_out, ctx.needs_input_grad[:5]), None, None)


def sandwich_norm(x, y, post_weight=None, pre_weight=None, *, gate=None, scale=1.0, post_norm=True, p=0.0, rng=None, eps=1e-6):
  """(s, out) with s = scale * x + dropout(gate * rms_norm(y) * post_weight) and out = rms_norm(s) * pre_weight, for x
  and y [..., channels] of one shape, float32 or bfloat16 on a GPU, with 1 to 16,384 channels and fewer than 2^32 rows.

  Weights [channels] and the gate are in x's dtype or float32, None is 1. The gate is [channels], [members, channels] for
  x of [members, ..., channels], or of x's shape. Without `post_norm` y is gated as it is, and there is no post_weight. `scale`, `p`
  and `eps` are numbers: a learned scale is applied to x before the call. With p > 0 the gated branch is dropped as
  ``dropout`` drops it, by the state `rng`. s is formed in float32 and stored rounded once; statistics are float32 and
  those of s are the stored rows'. Rows of any stride are read where they lie if their channels are contiguous. Differentiable in x, y, the weights and the gate; the gradient of s adds to the norm's."""
  _check(x, "x")
  _check(y, "y", x)
  _check_weight(post_weight, "post_weight", x)
  _check_weight(pre_weight, "pre_weight", x)
  if post_weight is not None and not post_norm:
    raise ValueError("post_weight is the norm's: there is none without post_norm")
  scale, eps = check_number(scale, "scale"), check_number(eps, "eps")
  p, state, seed, offset = check_p(p), None, 0, 0
  if p > 0:
    if rng is None:
      raise ValueError("dropout needs rng, its state")
    state, seed, offset = rng_of(rng, x)
  c, dtype = x.shape[-1], _DTYPES[x.dtype]
  # Strides and the state's address are each launch's own (_for_launch): autograd keeps the descriptor without them.
  d = nat.SandwichDesc(x.numel() // c, _gate_rows(gate, x), 0, 0, c, dtype, _kind(gate, dtype), _kind(post_weight, dtype),
                       _kind(pre_weight, dtype), bool(post_norm), eps, scale, nat.Dropout(p, seed, offset, None))
  if _needs(x, y, post_weight, pre_weight, gate):
    return _Sandwich.apply(x, y, post_weight, pre_weight, gate, state, d)
  return _forward(x, y, post_weight, pre_weight, gate, state, d)
