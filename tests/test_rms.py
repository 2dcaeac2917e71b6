"""RMS norm of rows (``rms.py``, ``fwn_rms_norm_*``) against its formulas in float64.

Bounds. A row's sums are float32 chains of at most 32 products a thread and 10 additions across threads,
so a mean square is off by at most 64 x 2^-24 of itself and 1 / sqrt of it by half that; with the few
operations around them every value computed from it stays within 2^-18 of its terms' magnitudes. On top
comes the one rounding to the output's type: half a step, eps / 2 of the value."""
import ctypes

import pytest
import torch

import faster_weathernext_amd as fwn
from faster_weathernext_amd import _native as nat

DEV = "cuda"
gpu = pytest.mark.gpu
NEAR = 2.0 ** -18
DTYPES = [torch.bfloat16, torch.float32]


def _half(dtype):
  return torch.finfo(dtype).eps / 2


def _normal(shape, dtype, seed):
  gen = torch.Generator().manual_seed(seed)
  return torch.randn(shape, generator=gen).to(dtype).to(DEV)


def _norm64(s, weight, eps):
  s = s.double()
  v = s / (s.square().mean(-1, keepdim=True) + eps).sqrt()
  return v if weight is None else v * weight.double()


def _within(got, want, slack, what=""):
  off = (got.double() - want).abs() - slack
  assert torch.isfinite(got.float()).all(), what
  assert off.max() <= 0, (what, off.max().item())


# One thread a vector up to rows that take a workgroup; sizes about each change of instance; odd ones.
CHANNELS = [1, 7, 8, 64, 127, 128, 129, 250, 256, 264, 511, 512, 768, 1000, 1024, 1283, 2048, 2056, 4097, 5120, 8192, 8200,
            12289, 16384]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("channels", CHANNELS)
def test_forward(channels, dtype):
  for rows in (1, 5, 67):
    x, y = _normal((rows, channels), dtype, rows), _normal((rows, channels), dtype, rows + 1)
    for weight in (None, _normal((channels,), dtype, 3), _normal((channels,), torch.float32, 4)):
      s, out = fwn.add_rms_norm(x, y, weight, eps=1e-5)
      assert s.dtype == out.dtype == dtype and torch.equal(s, (x.float() + y.float()).to(dtype))
      want = _norm64(s, weight, 1e-5)
      _within(out, want, want.abs() * (_half(dtype) + NEAR) + 1e-37, (rows, channels))
      want = _norm64(x, weight, 1e-5)
      _within(fwn.rms_norm(x, weight, eps=1e-5), want, want.abs() * (_half(dtype) + NEAR) + 1e-37, (rows, channels))


def _check_q8(q, scale, v):
  """q * scale against the float64 rows v: half a step of e4m3, or of its subnormals (2^-9 of a scale)."""
  top = (v.abs().amax(-1) / 448).clamp(min=2.0 ** -126)
  _within(scale, top, top * 2 * NEAR)
  got = q.float().double() * scale.double()[..., None]
  _within(got, v, v.abs() * (2.0 ** -4 + 4 * NEAR) + 2.0 ** -10 * scale.double()[..., None])


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("channels", CHANNELS)
def test_8_bits(channels, dtype):
  for rows in (1, 67):
    x, y = _normal((rows, channels), dtype, rows), _normal((rows, channels), dtype, rows + 1)
    weight = _normal((channels,), dtype, 3)
    s, q, scale = fwn.add_rms_norm_q8(x, y, weight)
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and scale.shape == (rows,)
    assert torch.equal(s, (x.float() + y.float()).to(dtype))
    _check_q8(q, scale, _norm64(s, weight, 1e-6))
    _check_q8(*fwn.rms_norm_q8(x, weight), _norm64(x, weight, 1e-6))
    q, scale = fwn.quantize_rows(x)
    _check_q8(q, scale, x.double())
    assert q.float().abs().amax(-1).eq(448).all()  # the largest of each row is the largest code
    # Code for code what torch's own conversion makes of the scaled values.
    assert torch.equal(q.view(torch.uint8), (x.float() * (1 / scale)[:, None]).to(torch.float8_e4m3fn).view(torch.uint8))


@gpu
def test_8_bits_of_special_rows():
  x = torch.zeros(7, 72, device=DEV)
  x[1, 3] = float("nan")
  x[2, 4] = float("inf")
  x[3] = 1e-42  # subnormal: the scale stays at its least, 2^-126, and 1e-42 of it is under e4m3's least half step
  x[4, 0] = 3e38
  x[5, 0], x[5, 1] = 448.0, -448.0
  x[6, 0], x[6, 1] = 2.0 ** -126, -(2.0 ** -126)
  q, scale = fwn.quantize_rows(x)
  f = q.float()
  assert scale[0] == 2.0 ** -126 and not f[0].any()
  assert scale[1].isnan() and f[1].isnan().all()
  assert scale[2].isinf() and f[2, 4].isnan() and not f[2, :4].any()
  assert scale[3] == 2.0 ** -126 and not f[3].any()
  assert f[4, 0] == 448 and not f[4, 1:].any()
  assert scale[5] == 1 and f[5, 0] == 448 and f[5, 1] == -448
  assert scale[6] == 2.0 ** -126 and f[6, 0] == 1 and f[6, 1] == -1
  # The norm of a row of zeros is zeros; NaN stays in its row.
  x = torch.zeros(3, 40, device=DEV)
  x[1, 2], x[2] = float("nan"), 2.0
  out = fwn.rms_norm(x)
  assert not out[0].any() and out[1].isnan().all() and torch.allclose(out[2], torch.ones_like(out[2]))


def _grads64(s, weight, eps, g_out, g_sum):
  """(gx, gw, bounds of both): the formula, and the magnitudes of its terms times NEAR."""
  s, g = s.double(), g_out.double()
  w = torch.ones(s.shape[-1], device=DEV, dtype=torch.float64) if weight is None else weight.double()
  r = 1 / (s.square().mean(-1, keepdim=True) + eps).sqrt()
  h = g * w
  gs = torch.zeros_like(s) if g_sum is None else g_sum.double()
  gx = gs + r * (h - s * r.square() * (h * s).mean(-1, keepdim=True))
  terms = gs.abs() + r * (h.abs() + s.abs() * r.square() * (h * s).abs().mean(-1, keepdim=True))
  gw = (g * s * r).reshape(-1, s.shape[-1]).sum(0)
  # gw's chains: at most 64 rows a thread here, 16 places of a workgroup, 1024 / 16 + 16 partial rows.
  return gx, gw, NEAR * terms, 256 * 2.0 ** -24 * (g * s * r).abs().reshape(-1, s.shape[-1]).sum(0)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("channels", CHANNELS)
def test_gradients(channels, dtype):
  for rows in (1, 5, 301):
    x, y, g_out, g_sum = (_normal((rows, channels), dtype, rows + k) for k in range(4))
    for weight in (None, _normal((channels,), dtype, 9), _normal((channels,), torch.float32, 9)):
      leaves = [t.clone().requires_grad_() for t in ((x, y) if weight is None else (x, y, weight))]
      s, out = fwn.add_rms_norm(*leaves, eps=1e-5)
      grads = torch.autograd.grad((s, out), leaves, (g_sum, g_out))
      gx, gw, bx, bw = _grads64(s.detach(), weight, 1e-5, g_out, g_sum)
      _within(grads[0], gx, gx.abs() * _half(dtype) + bx, (rows, channels))
      assert torch.equal(grads[0], grads[1])
      if weight is not None:
        assert grads[2].dtype == weight.dtype
        _within(grads[2], gw, gw.abs() * _half(weight.dtype) + bw, (rows, channels))
      leaf = x.clone().requires_grad_()
      gx, _, bx, _ = _grads64(x, weight, 1e-5, g_out, None)
      got, = torch.autograd.grad(fwn.rms_norm(leaf, weight, eps=1e-5), leaf, g_out)
      _within(got, gx, gx.abs() * _half(dtype) + bx, (rows, channels))


@gpu
def test_many_rows():
  """More rows than one round of workgroups takes, and a weight gradient over all of them."""
  x, y, g = (_normal((20001, 264), torch.bfloat16, k) for k in range(3))
  weight = _normal((264,), torch.bfloat16, 4).requires_grad_()
  x.requires_grad_()
  s, out = fwn.add_rms_norm(x, y, weight)
  gx, gw = torch.autograd.grad(out, (x, weight), g)
  wx, ww, bx, bw = _grads64(s.detach(), weight.detach(), 1e-6, g, None)
  _within(gx, wx, wx.abs() * 2.0 ** -8 + bx)
  _within(gw, ww, ww.abs() * 2.0 ** -8 + bw)
  again = torch.autograd.grad(fwn.add_rms_norm(x, y, weight)[1], weight, g)[0]
  assert torch.equal(gw, again)


@gpu
def test_gradient_against_differences():
  """A directional difference of the float64 formula at the float32 inputs."""
  x, y, d, g = (_normal((6, 40), torch.float32, k) for k in range(4))
  w = _normal((40,), torch.float32, 7)
  leaf = x.clone().requires_grad_()
  s, out = fwn.add_rms_norm(leaf, y, w)
  gx, = torch.autograd.grad((s, out), leaf, (g, g))
  def f(t):
    total = x.double() + t * d.double() + y.double()
    return ((total + _norm64(total, w, 1e-6)) * g.double()).sum()
  h = 1e-5  # central: an error of h^2 times the third derivative, and 1e-16 / h
  assert abs((f(h) - f(-h)) / (2 * h) - (gx.double() * d.double()).sum()) < 1e-4


@gpu
def test_partial_gradients():
  x, y, g = (_normal((9, 128), torch.bfloat16, k) for k in range(3))
  w = _normal((128,), torch.bfloat16, 5)
  leaves = [t.clone().requires_grad_() for t in (x, y, w)]
  s, out = fwn.add_rms_norm(*leaves)
  gx, gy, gw = torch.autograd.grad(s, leaves, g, allow_unused=True, retain_graph=True)
  assert torch.equal(gx, g) and torch.equal(gy, g) and (gw is None or not gw.any())
  only_w = w.clone().requires_grad_()
  got = torch.autograd.grad(fwn.add_rms_norm(x, y, only_w)[1], only_w, g)[0]
  assert torch.equal(got, torch.autograd.grad(out, leaves[2], g)[0])
  frozen = x.clone().requires_grad_()
  gx, = torch.autograd.grad(fwn.rms_norm(frozen, w), frozen, g)
  assert gx.shape == x.shape


@gpu
def test_second_derivative_and_batched_gradients():
  x = _normal((5, 64), torch.float32, 1).requires_grad_()
  w = _normal((64,), torch.float32, 2).requires_grad_()
  g = _normal((5, 64), torch.float32, 3)
  def both(fn):
    first, = torch.autograd.grad(fn(x), x, g, create_graph=True)
    return torch.autograd.grad(first.square().sum(), (x, w))
  plain = lambda t: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * w
  for a, b in zip(both(lambda t: fwn.rms_norm(t, w)), both(plain)):
    torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-4)
  gs = torch.stack([g, 2 * g])
  got, = torch.autograd.grad(fwn.rms_norm(x, w), x, gs, is_grads_batched=True)
  want, = torch.autograd.grad(plain(x), x, gs, is_grads_batched=True)
  torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-5)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(dtype):
  """Slices, one row for all, transposed and misaligned tensors give the contiguous tensors' results."""
  big = _normal((33, 400), dtype, 1)
  views = [big[:, :264], big[:, 1:265], big[::2, 8:272], big[:1, :264].expand(33, 264), big.t()[:264, :33].t(),
           big.view(3, 11, 400)[:, :, :264], big.view(3, 11, 400).transpose(0, 1)[..., 16:280], big[:, :264][5]]
  w = _normal((800,), dtype, 2)
  for weight in (w[:264], w[1:265], w[::2][:264]):
    for x in views:
      y = x.flip(0)
      a, b = fwn.add_rms_norm(x, y, weight), fwn.add_rms_norm(x.contiguous(), y.contiguous(), weight.contiguous())
      assert a[0].shape == x.shape and torch.equal(a[0], b[0])
      # Other instances add in another order: within two roundings.
      assert ((a[1].double() - b[1].double()).abs() <= b[1].double().abs() * (2 * _half(dtype) + 2 * NEAR)).all()
      q, scale = fwn.rms_norm_q8(x, weight)
      assert q.is_contiguous() and scale.shape == x.shape[:-1]
      _check_q8(q, scale, _norm64(x, weight, 1e-6))
      leaf = x.detach().requires_grad_()
      s, out = fwn.add_rms_norm(leaf, y, weight)
      g = torch.ones_like(out).t().contiguous().t() if x.dim() == 2 else torch.ones_like(out)
      gx, = torch.autograd.grad(out, leaf, g)
      want, _, bx, _ = _grads64(s.detach(), weight, 1e-6, g, None)
      _within(gx, want, want.abs() * _half(dtype) + bx)


@gpu
def test_empty():
  w = torch.ones(64, device=DEV, requires_grad=True)
  x = torch.zeros(0, 64, device=DEV, requires_grad=True)
  s, out = fwn.add_rms_norm(x, x, w)
  assert s.shape == out.shape == (0, 64)
  gx, gw = torch.autograd.grad(out.sum(), (x, w))
  assert gx.shape == (0, 64) and not gw.any()
  with torch.no_grad():
    q, scale = fwn.rms_norm_q8(torch.zeros(2, 0, 64, device=DEV))
  assert q.shape == (2, 0, 64) and scale.shape == (2, 0)


@gpu
def test_side_stream_and_graph():
  """On another stream, and captured: each replay against the eager results for new inputs."""
  x, y, g = (_normal((100, 520), torch.bfloat16, k) for k in range(3))
  w = _normal((520,), torch.bfloat16, 5)
  x.requires_grad_()
  w.requires_grad_()
  def step():
    s, out = fwn.add_rms_norm(x, y, w)
    with torch.no_grad():
      q = fwn.add_rms_norm_q8(x, y, w)
    return [s.detach(), out.detach(), *torch.autograd.grad((s, out), (x, w), (g, g)), q[1].view(torch.uint8), q[2]]
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
  for k in range(4):
    with torch.no_grad():
      x.copy_(_normal((100, 520), torch.bfloat16, 20 + k))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(held, step()):
      assert torch.equal(a, b), k


@gpu
def test_refusals():
  x = torch.zeros(4, 64, device=DEV)
  for call in (lambda: fwn.rms_norm(torch.zeros(4, 64)), lambda: fwn.rms_norm(torch.zeros((), device=DEV)),
               lambda: fwn.rms_norm(torch.zeros(4, 0, device=DEV)), lambda: fwn.rms_norm(torch.zeros(1, 16385, device=DEV)),
               lambda: fwn.add_rms_norm(x, x[:2]), lambda: fwn.add_rms_norm(x, x.bfloat16()),
               lambda: fwn.add_rms_norm(x, torch.zeros(4, 64)), lambda: fwn.rms_norm(x, torch.ones(64)),
               lambda: fwn.rms_norm(x, torch.ones(63, device=DEV)), lambda: fwn.quantize_rows(torch.zeros(4, 64))):
    with pytest.raises(ValueError):
      call()
  for call in (lambda: fwn.rms_norm(x.half()), lambda: fwn.rms_norm(x, torch.ones(64, device=DEV, dtype=torch.bfloat16)),
               lambda: fwn.quantize_rows(x.to(torch.float64))):
    with pytest.raises(TypeError):
      call()
  with pytest.raises(nat.FwnError):
    fwn.rms_norm(x, eps=-1.0)
  leaf = x.clone().requires_grad_()
  for call in (lambda: fwn.rms_norm_q8(leaf), lambda: fwn.add_rms_norm_q8(x, leaf), lambda: fwn.quantize_rows(leaf)):
    with pytest.raises(RuntimeError, match="no derivative"):
      call()


# ---- host validation of the C ABI: no GPU calls

F = 4096  # an address that is only compared


def _desc(rows=4, channels=64, x_stride=64, y_stride=64, dtype=nat.BF16, weight_dtype=nat.BF16, eps=1e-6):
  return nat.RmsDesc(rows, x_stride, y_stride, channels, dtype, weight_dtype, eps)


@pytest.mark.parametrize("bad,code", [(dict(rows=-1), 1), (dict(channels=0), 1), (dict(channels=16385), 1), (dict(x_stride=-1), 1),
                                      (dict(y_stride=1 << 62), 1), (dict(rows=1 << 60), 1), (dict(dtype=2), 2),
                                      (dict(dtype=nat.F32), 2), (dict(eps=-1.0), 1), (dict(eps=float("nan")), 1),
                                      (dict(eps=float("inf")), 1)])
def test_bad_descriptors(bad, code):
  L, d = nat.lib(), _desc(**bad)
  size = ctypes.c_uint64()
  assert L.fwn_rms_norm_launch(d, F, None, None, None, 2 * F, None) == code
  assert L.fwn_rms_norm_q8_launch(d, F, None, None, None, 2 * F, 4 * F, None) == code
  assert L.fwn_quantize_rows_launch(d, F, 2 * F, 4 * F, None) == code
  assert L.fwn_rms_norm_bwd_workspace_size(d, ctypes.byref(size)) == code
  assert L.fwn_rms_norm_bwd_launch(d, F, None, 2 * F, None, 4 * F, None, None, 0, None) == code


def test_bad_pointers():
  L, d = nat.lib(), _desc()
  fwd, q8, bwd = L.fwn_rms_norm_launch, L.fwn_rms_norm_q8_launch, L.fwn_rms_norm_bwd_launch
  for rc in (fwd(None, F, None, None, None, 2 * F, None), fwd(d, None, None, None, None, 2 * F, None),
             fwd(d, F, None, None, None, None, None), fwd(d, F, 2 * F, None, None, 3 * F, None),
             fwd(d, F, None, None, 2 * F, 3 * F, None), fwd(d, F, None, None, None, F + 256, None),
             fwd(d, F, 2 * F, None, 3 * F, 3 * F, None), fwd(d, F, 2 * F, 3 * F, 4 * F, 3 * F, None),
             fwd(d, F + 1, None, None, None, 2 * F, None), fwd(d, F, None, 3 * F + 1, None, 2 * F, None),
             q8(d, F, None, None, None, None, 3 * F, None), q8(d, F, None, None, None, 2 * F, None, None),
             q8(d, F, None, None, None, 2 * F, 2 * F, None), q8(d, F, None, None, None, 2 * F, 3 * F + 2, None),
             bwd(d, None, None, 2 * F, None, 3 * F, None, None, 0, None), bwd(d, F, None, None, None, 3 * F, None, None, 0, None),
             bwd(d, F, None, 2 * F, None, None, None, None, 0, None), bwd(d, F, None, 2 * F, None, F, None, None, 0, None),
             bwd(d, F, None, 2 * F, None, 2 * F + 128, None, None, 0, None),
             bwd(d, F, None, 2 * F, None, 3 * F, 4 * F, None, 0, None), bwd(d, F, None, 2 * F, None, 3 * F, 4 * F, 5 * F, 8, None),
             bwd(d, F, None, 2 * F, None, 3 * F, 4 * F, 5 * F + 8, 1 << 20, None)):
    assert rc == nat.ERR_INVALID_ARG
  assert fwd(_desc(rows=0), None, None, None, None, None, None) == nat.OK


def test_needs_a_gpu_tensor():
  for call in (fwn.rms_norm, fwn.rms_norm_q8, fwn.quantize_rows):
    with pytest.raises(ValueError, match="CUDA"):
      call(torch.zeros(2, 64))


@gpu
def test_offsets_past_32_bits():
  """Rows whose bytes lie past 2^32 from the first, in the forward, the 8-bit output and the backward."""
  rows, c = 140000, 16384  # 4.6 GB
  gen = torch.Generator(device=DEV).manual_seed(1)
  x = torch.randint(-4, 5, (rows, c), generator=gen, device=DEV, dtype=torch.int8).to(torch.bfloat16)
  w = _normal((c,), torch.bfloat16, 2)
  at = [0, 1, rows // 2, rows - 2, rows - 1]
  out = fwn.rms_norm(x, w)
  want = _norm64(x[at], w, 1e-6)
  _within(out[at], want, want.abs() * (2.0 ** -8 + NEAR) + 1e-37)
  q, scale = fwn.rms_norm_q8(x, w)
  _check_q8(q[at], scale[at], want)
  leaf = x.requires_grad_()
  gx, = torch.autograd.grad(fwn.rms_norm(leaf, w), leaf, out)
  wx, _, bx, _ = _grads64(x.detach()[at], w, 1e-6, out[at], None)
  _within(gx[at], wx, wx.abs() * 2.0 ** -8 + bx)


@gpu
def test_the_same_tensor_twice():
  x, g = _normal((9, 72), torch.float32, 1), _normal((9, 72), torch.float32, 2)
  leaf = x.clone().requires_grad_()
  s, out = fwn.add_rms_norm(leaf, leaf)
  gx, = torch.autograd.grad(out, leaf, g)
  want, _, bx, _ = _grads64(s.detach(), None, 1e-6, g, None)
  _within(gx, 2 * want, 2.0 ** -23 * want.abs() + 2 * bx)


@gpu
def test_forward_mode_is_refused():
  import torch.autograd.forward_ad as fwad
  x = _normal((4, 64), torch.float32, 1)
  with fwad.dual_level():
    dual = fwad.make_dual(x, torch.ones_like(x))
    for call in (fwn.rms_norm, fwn.rms_norm_q8, fwn.quantize_rows, lambda t: fwn.add_rms_norm(t, x),
                 lambda t: fwn.linear_act(t, x)):
      with pytest.raises(RuntimeError):
        call(dual)
    assert torch.equal(fwn.rms_norm(x), fwn.rms_norm(x))


def test_backward_outputs_overlap_nothing():
  L, d = nat.lib(), _desc()
  for gx, gw, weight in ((3 * F, 3 * F + 256, 5 * F), (3 * F, 4 * F, 3 * F), (3 * F, 5 * F, 5 * F), (3 * F, F, 5 * F),
                         (3 * F, 2 * F, 5 * F)):
    assert L.fwn_rms_norm_bwd_launch(d, F, weight, 2 * F, None, gx, gw, 16 * F, 1 << 20, None) == nat.ERR_INVALID_ARG
