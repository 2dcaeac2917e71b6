"""Second derivatives of the RMS norms and linear layers at tensors of any strides, against torch's own of the
same formulas in float64. The chains here are at most a few hundred float32 operations on terms of one
size: within 2^-12 of the gradients' norms. A gradient that one side has not counts as zeros there."""
import pytest
import torch

import faster_weathernext_amd as fwn
from faster_weathernext_amd import rms

DEV = "cuda"
gpu = pytest.mark.gpu
NEAR = 2.0 ** -12


def _normal(shape, seed, device):
  return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(device)


def _second(fn, leaves, gs):
  outs = fn(*leaves)
  outs = outs if isinstance(outs, tuple) else (outs,)
  first = torch.autograd.grad(outs, leaves, gs, create_graph=True)
  total = sum(t.square().sum() for t in first)
  return first, torch.autograd.grad(total, leaves, materialize_grads=True)


def _compare(fn, plain, leaves, gs):
  wide = [t.detach().double().requires_grad_() for t in leaves]
  got, want = _second(fn, leaves, gs), _second(plain, wide, tuple(g.double() for g in gs))
  for a, b in zip((*got[0], *got[1]), (*want[0], *want[1])):
    assert (a.double() - b).norm() <= NEAR * b.norm(), ((a.double() - b).norm() / b.norm()).item()


def _rms_plain(x, y, weight):
  s = x if y is None else x + y
  out = s / (s.square().mean(-1, keepdim=True) + 1e-6).sqrt() * weight
  return out if y is None else (s, out)


def _leaves(kind, channels, device):
  """(x, y, weight): rows and weights that are contiguous, slices, or every other element."""
  base = lambda k: _normal((6, 2 * channels + 3), k, device)
  view = {"dense": lambda t: t[:, :channels].contiguous(), "rows": lambda t: t[:, 1:channels + 1],
          "columns": lambda t: t[:, :2 * channels:2]}[kind]
  return [view(base(1)).requires_grad_(), view(base(2)).requires_grad_(), view(base(3))[0].detach().requires_grad_()]


@pytest.mark.parametrize("weight_kind", ["dense", "columns"])
@pytest.mark.parametrize("kind", ["dense", "rows", "columns"])
def test_rms_norm_without_a_gpu(kind, weight_kind, monkeypatch):
  """The autograd Function alone, its forward pass as torch operations."""
  def forward(x, y, weight, eps, q8):
    s = x if y is None else x + y
    out = s * torch.rsqrt(s.square().mean(-1, keepdim=True) + eps) * weight
    return None if y is None else s, out
  monkeypatch.setattr(rms, "_forward", forward)
  (x, y, _), (_, _, w) = _leaves(kind, 8, "cpu"), _leaves(weight_kind, 8, "cpu")
  g, g_sum = _normal((6, 8), 4, "cpu"), _normal((6, 8), 5, "cpu")
  _compare(lambda x, w: rms._RmsNorm.apply(x, None, w, 1e-6), lambda x, w: _rms_plain(x, None, w), [x, w], (g,))
  _compare(lambda x, y, w: rms._RmsNorm.apply(x, y, w, 1e-6), _rms_plain, [x, y, w], (g_sum, g))


@gpu
@pytest.mark.parametrize("weight_kind", ["dense", "columns"])
@pytest.mark.parametrize("kind", ["dense", "rows", "columns"])
def test_rms_norm(kind, weight_kind):
  (x, y, _), (_, _, w) = _leaves(kind, 72, DEV), _leaves(weight_kind, 72, DEV)
  g, g_sum = _normal((6, 72), 4, DEV), _normal((6, 72), 5, DEV)
  _compare(fwn.rms_norm, lambda x, w: _rms_plain(x, None, w), [x, w], (g,))
  _compare(fwn.add_rms_norm, _rms_plain, [x, y, w], (g_sum, g))
  # The first derivatives by the kernels, at the same tensors.
  wide = [t.detach().double().requires_grad_() for t in (x, y, w)]
  want = torch.autograd.grad(_rms_plain(*wide), wide, (g_sum.double(), g.double()))
  for a, b in zip(torch.autograd.grad(fwn.add_rms_norm(x, y, w), (x, y, w), (g_sum, g)), want):
    assert (a.double() - b).norm() <= NEAR * b.norm()
  want = torch.autograd.grad(_rms_plain(wide[0], None, wide[2]), (wide[0], wide[2]), g.double())
  for a, b in zip(torch.autograd.grad(fwn.rms_norm(x, w), (x, w), g), want):
    assert (a.double() - b).norm() <= NEAR * b.norm()


ACTIVATIONS = {None: lambda t: t, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu,
               "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}


@gpu
@pytest.mark.parametrize("kind", ["dense", "rows", "columns"])
@pytest.mark.parametrize("activation", ACTIVATIONS)
def test_linear_act(activation, kind):
  x, w, b = _leaves(kind, 24, DEV)[0], _leaves(kind, 24, DEV)[1], _normal((12,), 6, DEV)[::2].requires_grad_()
  r, g = _normal((6, 6), 7, DEV).requires_grad_(), _normal((6, 6), 8, DEV)
  _compare(lambda x, w, b, r: fwn.linear_act(x, w, b, activation=activation, residual=r),
           lambda x, w, b, r: ACTIVATIONS[activation](x @ w.t() + b) + r, [x, w, b, r], (g,))
