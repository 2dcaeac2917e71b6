"""Dropout without a stored mask (``dropout.py``, ``fwn_dropout_launch``) against its definition on the host.

What is kept is whole numbers and has to be equal. A value is x m (+ residual) in float32 and one rounding: m is rounded to
float32 (2^-24), the product and the sum may be (2^-24 each), so that float64's result is off by at most 4 x 2^-24 of the terms'
magnitudes and half a step of the output's type."""
import ctypes

import numpy as np
import pytest
import torch

import faster_weathernext_amd as fwn
from faster_weathernext_amd import _native as nat
from oracle import dropout as oracle

DEV = "cuda"
gpu = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float32]
SEED, OFFSET = 0x0123456789abcdef, 0xfedcba9876543210


def _normal(shape, dtype, seed):
  return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def _kept(shape, p, seed=SEED, offset=OFFSET):
  rows, c = int(np.prod(shape[:-1])), shape[-1]
  return torch.from_numpy(oracle.kept(rows, c, p, seed, offset)).to(DEV).view(shape)


def _check(got, x, residual, p, kept):
  m = 65536 / (65536 - oracle.border(p)) if oracle.border(p) < 65536 else 0.0
  b = torch.where(kept, x.double() * m, 0.0)
  r = torch.zeros_like(b) if residual is None else residual.double()
  off = (got.double() - (b + r)).abs()
  assert got.dtype == x.dtype and got.shape == x.shape and got.is_contiguous()
  assert (off <= torch.finfo(x.dtype).eps / 2 * (b + r).abs() + 4 * 2.0 ** -24 * (b.abs() + r.abs())).all()
  if residual is None:
    assert torch.equal(got == 0, ~kept | (x == 0))


# ---- the numbers, on the host


def test_published_vectors():
  """Random123's known answers of Philox-4x32-10."""
  ones = 0xffffffff
  for counter, key, want in (
      ((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
      ((ones,) * 4, (ones,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
      ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0),
       (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))):
    assert tuple(int(w) for w in oracle.philox(counter, key)) == want


@pytest.mark.parametrize("p", [0.05, 0.1, 0.5, 0.9])
def test_frequencies(p):
  """Kept shares of rows, columns and neighbours: within five standard deviations."""
  k = oracle.kept(2000, 400, p, SEED, 7).astype(float)
  sd = (p * (1 - p)) ** 0.5
  assert abs(k.mean() - (1 - p)) < 5 * sd / k.size ** 0.5
  assert abs(k.mean(0) - (1 - p)).max() < 5 * sd / 2000 ** 0.5 and abs(k.mean(1) - (1 - p)).max() < 5 * sd / 400 ** 0.5
  c = k - (1 - p)
  for a, b in ((c[:, 1:], c[:, :-1]), (c[1:], c[:-1]), (c[:, 8:], c[:, :-8])):
    assert abs((a * b).mean()) < 5 * sd ** 2 / a.size ** 0.5
  for other in (oracle.kept(2000, 400, p, SEED, 8), oracle.kept(2000, 400, p, SEED + 1, 7)):
    assert abs((c * (other - (1 - p))).mean()) < 5 * sd ** 2 / c.size ** 0.5


# ---- the kernels


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (3, 8), (5, 9), (2, 3, 64), (67, 129), (1000,), (301, 768), (40, 1283),
                                   (3000, 12), (7, 16400), (2, 100003)])
def test_forward(shape, dtype):
  x, r = _normal(shape, dtype, 1), _normal(shape, dtype, 2)
  flat = (1, *shape) if len(shape) == 1 else shape
  for p in (0.0, 0.1, 0.5, 1 - 2.0 ** -16, 1.0):
    kept = _kept(flat, p).view(shape)
    for residual in (None, r):
      _check(fwn.dropout(x, p, (SEED, OFFSET), residual=residual), x, residual, p, kept)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_states(dtype):
  """Numbers, negative ones and a tensor of them give the same; seeds and offsets of every word count."""
  x = _normal((9, 40), dtype, 1)
  word = lambda v: v - (1 << 64) if v >> 63 else v
  for seed, offset in ((0, 0), (1, 0), (0, 1), (1 << 32, 0), (0, 1 << 32), (SEED, OFFSET), ((1 << 64) - 1, (1 << 64) - 1)):
    want = fwn.dropout(x, 0.5, (seed, offset))
    _check(want, x, None, 0.5, _kept((9, 40), 0.5, seed, offset))
    state = torch.tensor([word(seed), word(offset)], device=DEV)
    assert torch.equal(fwn.dropout(x, 0.5, state), want)
    assert torch.equal(fwn.dropout(x, 0.5, (word(seed), word(offset))), want)
    assert torch.equal(fwn.dropout(x, 0.5, torch.stack([state, state], 1)[:, 0]), want)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(dtype):
  big = _normal((33, 400), dtype, 1)
  w = _normal((12000,), dtype, 2)
  views = [big[:, :264], big[:, 1:265], big[::2, 8:272], big[:1, :264].expand(33, 264), big.t()[:264, :33].t(),
           big.view(3, 11, 400)[:, :, :264], big.view(3, 11, 400).transpose(0, 1)[..., 16:280], big[:, :264][5], w[1:1000],
           w[::3][:500], big[:, :1], big[3, 5:6]]
  for x in views:
    r = x.flip(0)
    for residual in (None, r, x):
      got = fwn.dropout(x, 0.25, (3, 4), residual=residual)
      dense = fwn.dropout(x.contiguous(), 0.25, (3, 4), residual=None if residual is None else residual.contiguous())
      assert torch.equal(got, dense) and got.is_contiguous()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients(dtype):
  x, r, g = (_normal((37, 203), dtype, k).requires_grad_(k < 2) for k in range(3))
  kept = _kept((37, 203), 0.3)
  out = fwn.dropout(x, 0.3, (SEED, OFFSET), residual=r)
  gx, gr = torch.autograd.grad(out, (x, r), g, retain_graph=True)
  _check(gx, g, None, 0.3, kept)
  assert torch.equal(gr, g)
  # A strided and an expanded gradient, and one leaf alone.
  strided = g.t().contiguous().t()
  assert torch.equal(torch.autograd.grad(out, x, strided, retain_graph=True)[0], gx)
  one = torch.ones((), dtype=dtype, device=DEV).expand(37, 203)
  assert torch.equal(torch.autograd.grad(out, x, one)[0], torch.autograd.grad(fwn.dropout(x, 0.3, (SEED, OFFSET)).sum(), x)[0])
  alone = fwn.dropout(x.detach(), 0.3, (SEED, OFFSET), residual=r)
  assert torch.equal(torch.autograd.grad(alone, r, g)[0], g)
  # The same tensor in both places.
  both, = torch.autograd.grad(fwn.dropout(x, 0.3, (SEED, OFFSET), residual=x), x, g)
  assert torch.equal(both, gx + g)


@gpu
def test_gradient_against_differences():
  """The function is linear: its difference along d is its gradient's product with d, up to float32's roundings."""
  x, d, g = (_normal((6, 40), torch.float32, k) for k in range(3))
  leaf = x.clone().requires_grad_()
  gx, = torch.autograd.grad(fwn.dropout(leaf, 0.5, (1, 2)), leaf, g)
  f = lambda t: (fwn.dropout(x + t * d, 0.5, (1, 2)).double() * g.double()).sum()
  # Two float32 roundings of each of 240 terms of a few units, over 2 h.
  assert abs((f(0.5) - f(-0.5)) - (gx.double() * d.double()).sum()) < 240 * 16 * 2.0 ** -22


@gpu
def test_second_derivative_and_batched_gradients():
  x, g = _normal((5, 64), torch.float32, 1).requires_grad_(), _normal((5, 64), torch.float32, 2).requires_grad_()
  k = _kept((5, 64), 0.5).float() * 2
  gx, = torch.autograd.grad(fwn.dropout(x.square(), 0.5, (SEED, OFFSET)), x, g, create_graph=True)
  torch.testing.assert_close(gx, 2 * x * g * k)
  second = torch.autograd.grad(gx.sum(), (x, g))
  torch.testing.assert_close(second[0], 2 * g * k)
  torch.testing.assert_close(second[1], 2 * x * k)
  gs = torch.stack([g.detach(), 2 * g.detach()])
  got, = torch.autograd.grad(fwn.dropout(x, 0.5, (SEED, OFFSET)), x, gs, is_grads_batched=True)
  torch.testing.assert_close(got, gs * k)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_values_that_are_not_finite(dtype):
  x = _normal((8, 64), dtype, 1)
  kept = _kept((8, 64), 0.5)
  x[0], x[1], x[2] = float("nan"), float("inf"), torch.finfo(dtype).max
  out = fwn.dropout(x, 0.5, (SEED, OFFSET))
  assert not out[~kept].any()
  assert out[0][kept[0]].isnan().all() and out[1:3][kept[1:3]].isinf().all() and out[3:].isfinite().all()
  # Dropped NaN add nothing to a residual, and NaN gradients of dropped places none.
  assert torch.equal(fwn.dropout(x, 0.5, (SEED, OFFSET), residual=torch.ones_like(x))[~kept], torch.ones_like(x)[~kept])
  leaf = torch.ones_like(x).requires_grad_()
  g, = torch.autograd.grad(fwn.dropout(leaf, 0.5, (SEED, OFFSET)), leaf, x)
  assert not g[~kept].any()


@gpu
def test_empty():
  x = torch.zeros(2, 0, 64, device=DEV, requires_grad=True)
  out = fwn.dropout(x, 0.5, (1, 2), residual=x)
  assert out.shape == x.shape and torch.autograd.grad(out.sum(), x)[0].shape == x.shape


@gpu
def test_side_stream_and_graph():
  """On another stream, and captured with a state that the program moves on between replays."""
  x, g = _normal((100, 520), torch.bfloat16, 1).requires_grad_(), _normal((100, 520), torch.bfloat16, 2)
  state = torch.tensor([5, 0], device=DEV)
  def step():
    out = fwn.dropout(x, 0.1, state, residual=g)
    return [out.detach(), *torch.autograd.grad(out, x, g)]
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    first = step()
  torch.cuda.current_stream().wait_stream(side)
  for a, b in zip(first, step()):
    assert torch.equal(a, b)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph, stream=side):
    held = step()
  seen = []
  for k in range(4):
    state[1] = k
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(held, step()):
      assert torch.equal(a, b), k
    seen.append(held[1].clone())
  assert not torch.equal(seen[0], seen[1])


@gpu
def test_state_changed_before_the_backward_pass():
  x, state = _normal((4, 64), torch.float32, 1).requires_grad_(), torch.tensor([5, 0], device=DEV)
  out = fwn.dropout(x, 0.1, state)
  state += 1
  with pytest.raises(RuntimeError, match="modified by an inplace operation"):
    out.sum().backward()


@gpu
def test_offsets_past_32_bits():
  """Rows whose bytes lie past 2^32 from the first, and a row that is itself that long."""
  rows, c, at = 140000, 16384, [0, 1, 70000, 139998, 139999]
  x = torch.ones(rows, c, device=DEV, dtype=torch.bfloat16)
  out = fwn.dropout(x, 0.5, (1, 2))
  for r in at:
    want = torch.from_numpy(oracle.kept(1, c, 0.5, 1, 2, first=r)[0]).to(DEV)
    assert torch.equal(out[r], 2 * want.to(out.dtype)), r
  del x, out
  n = (1 << 30)
  out = fwn.dropout(torch.ones(1, n, device=DEV), 0.5, (1, 2))
  eights = torch.tensor([0, 1, (n >> 4) + 3, (n >> 3) - 1])
  words = oracle.philox((eights.numpy(), 0, 2, 0), (1, 0))
  for k, e in enumerate(eights.tolist()):
    want = [float(2 * (((int(words[j // 2][k]) >> 16 * (j % 2)) & 0xffff) >= 32768)) for j in range(8)]
    assert out[0, 8 * e:8 * e + 8].tolist() == want


@gpu
def test_refusals():
  x = torch.zeros(4, 64, device=DEV)
  for call in (lambda: fwn.dropout(torch.zeros(4, 64), 0.1, (1, 2)), lambda: fwn.dropout(torch.zeros((), device=DEV), 0.1, (1, 2)),
               lambda: fwn.dropout(torch.zeros(4, 0, device=DEV), 0.1, (1, 2)), lambda: fwn.dropout(x, -0.1, (1, 2)),
               lambda: fwn.dropout(x, 1.1, (1, 2)), lambda: fwn.dropout(x, float("nan"), (1, 2)),
               lambda: fwn.dropout(x, 0.1, (1, 2), residual=x[:2]), lambda: fwn.dropout(x, 0.1, (1, 2), residual=x.bfloat16()),
               lambda: fwn.dropout(x, 0.1, (1, 2), residual=torch.zeros(4, 64)), lambda: fwn.dropout(x, 0.1, (1,)),
               lambda: fwn.dropout(x, 0.1, (1, 2, 3)), lambda: fwn.dropout(x, 0.1, (1.5, 2)), lambda: fwn.dropout(x, 0.1, "12"), lambda: fwn.dropout(x, 0.1, None), lambda: fwn.dropout(x, 0.1, 5),
               lambda: fwn.dropout(x, 0.1, torch.tensor([1, 2])), lambda: fwn.dropout(x, 0.1, torch.tensor([1., 2.], device=DEV)),
               lambda: fwn.dropout(x, 0.1, torch.tensor([1, 2, 3], device=DEV))):
    with pytest.raises(ValueError):
      call()
  for call in (lambda: fwn.dropout(x.half(), 0.1, (1, 2)), lambda: fwn.dropout(x.double(), 0.1, (1, 2))):
    with pytest.raises(TypeError):
      call()
  import torch.autograd.forward_ad as fwad
  with fwad.dual_level():
    dual = fwad.make_dual(x, torch.ones_like(x))
    with pytest.raises(RuntimeError):
      fwn.dropout(dual, 0.1, (1, 2))


# ---- host validation of the C ABI: no GPU calls

F = 4096  # an address that is only compared


def _desc(rows=4, channels=64, x_stride=64, r_stride=64, dtype=nat.BF16, p=0.1, state=None):
  return nat.DropoutDesc(rows, x_stride, r_stride, channels, dtype, nat.Dropout(p, 1, 2, state))


@pytest.mark.parametrize("bad,code", [(dict(rows=-1), 1), (dict(rows=1 << 32), 1), (dict(channels=0), 1), (dict(channels=(1 << 30) + 1), 1),
                                      (dict(x_stride=-1), 1), (dict(r_stride=1 << 62), 1), (dict(dtype=2), 2), (dict(p=-0.1), 1),
                                      (dict(p=1.01), 1), (dict(p=float("nan")), 1), (dict(state=F + 4), 1)])
def test_bad_descriptors(bad, code):
  assert nat.lib().fwn_dropout_launch(_desc(**bad), F, None, 4 * F, None) == code


def test_bad_pointers():
  L, d = nat.lib(), _desc()
  run = L.fwn_dropout_launch
  for rc in (run(None, F, None, 2 * F, None), run(d, None, None, 2 * F, None), run(d, F, None, None, None),
             run(d, F + 1, None, 2 * F, None), run(d, F, 3 * F + 1, 2 * F, None), run(d, F, None, 2 * F + 1, None),
             run(d, F, None, F + 16, None), run(d, F, 2 * F, 2 * F + 16, None), run(_desc(x_stride=65), F, None, F, None),
             run(_desc(r_stride=0), F, 2 * F, 2 * F, None), run(_desc(state=2 * F + 8), F, None, 2 * F, None)):
    assert rc == nat.ERR_INVALID_ARG
  assert run(_desc(rows=0), None, None, None, None) == nat.OK


def test_needs_a_gpu_tensor():
  with pytest.raises(ValueError, match="CUDA"):
    fwn.dropout(torch.zeros(2, 64), 0.1, (1, 2))
