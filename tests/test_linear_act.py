"""Linear layers with bias, activation and residual in the epilogue (``linear_act.py``, ``fwn_linear_act_*``).

Two kinds of check. Inputs of small whole numbers, whose products and sums float32 holds exactly: the outputs
equal the float64 result rounded once, to the bit, so that no index, edge or stride can be wrong. Random
inputs against float64 with derived bounds: a float32 sum of k products is off by the roundings of its
partial sums, each at most 2^-24 of a partial sum that grows as sqrt(j) times a term's deviation, together at
most (2 / 3) sqrt(k) 2^-24 |a| |b| (norms of the two rows); twelve times that for partial sums several
deviations large, and 16 for the few operations of the epilogue."""
import ctypes

import pytest
import torch

import faster_weathernext_amd as fwn
from faster_weathernext_amd import _native as nat
from faster_weathernext_amd.linear_act import _slope

DEV = "cuda"
gpu = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float32]
ACTIVATIONS = [None, "relu", "gelu", "gelu_tanh", "silu"]

# rows, ins, outs: single tokens, a few, edges of tiles, odd widths, long sums, many rows.
SIZES = [(1, 1, 1), (1, 64, 64), (1, 768, 1000), (2, 7, 9), (3, 513, 65), (7, 4096, 512), (16, 256, 16), (17, 100, 33),
         (24, 1032, 136), (31, 8, 260), (32, 32, 32), (33, 96, 31), (63, 64, 129), (64, 128, 64), (65, 72, 250), (100, 515, 1027),
         (127, 1000, 128), (128, 64, 256), (129, 192, 257), (255, 264, 255), (256, 256, 256), (257, 320, 511),
         (513, 40, 770), (1000, 1024, 130), (2562, 515, 129), (5000, 136, 72), (9001, 64, 40), (300, 3, 4000), (40, 5000, 8)]


def _gen(seed):
  return torch.Generator().manual_seed(seed)


def _whole(shape, dtype, seed):
  return torch.randint(-2, 3, shape, generator=_gen(seed)).to(dtype).to(DEV)


def _normal(shape, dtype, seed, std=1.0):
  return (torch.randn(shape, generator=_gen(seed)) * std).to(dtype).to(DEV)


def _leaf(t):
  return t.detach().clone().requires_grad_()


def _half(dtype):
  return torch.finfo(dtype).eps / 2


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,ins,outs", SIZES)
def test_whole_numbers(rows, ins, outs, dtype):
  x, w, b = _whole((rows, ins), dtype, 1), _whole((outs, ins), dtype, 2), _whole((outs,), dtype, 3)
  r, g = _whole((rows, outs), dtype, 4), _whole((rows, outs), dtype, 5)
  z = x.double() @ w.double().t()
  assert torch.equal(fwn.linear_act(x, w), z.to(dtype))
  assert torch.equal(fwn.linear_act(x, w, b, residual=r), (z + b.double() + r.double()).to(dtype))
  assert torch.equal(fwn.linear_act(x, w, b, activation="relu"), (z + b.double()).relu().to(dtype))
  leaves = [_leaf(t) for t in (x, w, b, r)]
  out = fwn.linear_act(*leaves[:3], residual=leaves[3])
  assert torch.equal(out, (z + b.double() + r.double()).to(dtype))
  gx, gw, gb, gr = torch.autograd.grad(out, leaves, g)
  assert torch.equal(gx, (g.double() @ w.double()).to(dtype))
  assert torch.equal(gw, (g.double().t() @ x.double()).to(dtype))
  assert torch.equal(gb, g.double().sum(0).to(dtype)) and torch.equal(gr, g)
  leaves = [_leaf(t) for t in (x, w, b)]
  gx, gw, gb = torch.autograd.grad(fwn.linear_act(*leaves, activation="relu"), leaves, g)
  dz = g.double() * (z + b.double() > 0)
  assert torch.equal(gx, (dz @ w.double()).to(dtype)) and torch.equal(gw, (dz.t() @ x.double()).to(dtype))
  assert torch.equal(gb, dz.sum(0).to(dtype))


def _act64(z, name):
  z = z.clone().requires_grad_()
  a = {None: lambda t: t * 1, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu,
       "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[name](z)
  return a.detach(), torch.autograd.grad(a.sum(), z)[0]


def _sum_bound(k, a, b):
  """How far a float32 sum of k products is from exact, [rows of a, rows of b]; see above."""
  return (8 * k ** 0.5 + 16) * 2.0 ** -24 * a.norm(dim=1)[:, None] * b.norm(dim=1)[None]


def _check(got, want, slack, what):
  assert torch.isfinite(got.float()).all(), what
  over = (got.double() - want).abs() - slack
  assert over.max() <= 0, (what, over.max().item())


@gpu
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,ins,outs", [(1, 768, 1000), (5, 513, 130), (24, 1032, 136), (65, 72, 250), (300, 515, 257),
                                           (2000, 256, 512)])
def test_random(rows, ins, outs, dtype, activation):
  x, w, b = _normal((rows, ins), dtype, 1), _normal((outs, ins), dtype, 2, ins ** -0.5), _normal((outs,), dtype, 3)
  r, g = _normal((rows, outs), dtype, 4), _normal((rows, outs), dtype, 5)
  half = _half(dtype)
  leaves = [_leaf(t) for t in (x, w, b, r)]
  out = fwn.linear_act(*leaves[:3], activation=activation, residual=leaves[3])
  xd, wd, gd = x.double(), w.double(), g.double()
  z = xd @ wd.t() + b.double()
  a, slope = _act64(z, activation)
  # The activations' slopes stay below 1.2; their own arithmetic within 2^-20 of z.
  ez = _sum_bound(ins, xd, wd) + 2.0 ** -22 * b.double().abs()
  want = a + r.double()
  _check(out, want, half * want.abs() + 1.2 * ez + 2.0 ** -20 * (z.abs() + r.double().abs()), "out")
  assert torch.equal(fwn.linear_act(x, w, b, activation=activation, residual=r), out)
  grads = torch.autograd.grad(out, leaves, g)
  # dz: the pre-activation rounded to the dtype (slopes change by at most 1.2 a unit; relu's where z is within
  # its error of 0), dz rounded to it.
  dz = gd * slope
  near = (z.abs() <= ez).double() if activation == "relu" else 1.2 * (half * z.abs() + ez) + 2.0 ** -20
  if activation is None:
    edz = torch.zeros_like(dz)
  else:
    edz = gd.abs() * near + half * dz.abs()
  # Independent roundings add as the root of their squares: six times that.
  both = lambda e, f: 6 * ((e ** 2) @ (f ** 2)).sqrt()
  wx, ww, wb = dz @ wd, dz.t() @ xd, dz.sum(0)
  _check(grads[0], wx, half * wx.abs() + both(edz, wd) + _sum_bound(outs, dz, wd.t()), "gx")
  _check(grads[1], ww, half * ww.abs() + both(edz.t(), xd) + _sum_bound(rows, dz.t(), xd.t()), "gw")
  sums = 6 * (edz ** 2).sum(0).sqrt() + (8 * rows ** 0.5 + 16) * 2.0 ** -24 * dz.norm(dim=0) * rows ** 0.5
  _check(grads[2], wb, half * wb.abs() + sums, "gb")
  assert torch.equal(grads[3], g)


@gpu
@pytest.mark.parametrize("activation", ACTIVATIONS[1:])
def test_gradient_against_differences(activation):
  x, w, b, d, g = _normal((5, 24), torch.float32, 1), _normal((40, 24), torch.float32, 2, 0.2), _normal((40,), torch.float32, 3), \
      _normal((5, 24), torch.float32, 4), _normal((5, 40), torch.float32, 5)
  leaf = _leaf(x)
  gx, = torch.autograd.grad(fwn.linear_act(leaf, w, b, activation=activation), leaf, g)
  f = lambda t: (_act64((x.double() + t * d.double()) @ w.double().t() + b.double(), activation)[0] * g.double()).sum()
  h = 1e-6  # central: an error of h^2 times the third derivative, and 1e-16 / h; relu's corners stay further off
  assert abs((f(h) - f(-h)) / (2 * h) - (gx.double() * d.double()).sum()) < 1e-4


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(dtype):
  """Slices, misaligned rows, one row for all, transposed operands: whole numbers, to the bit."""
  big, wide, res = _whole((70, 400), dtype, 1), _whole((90, 400), dtype, 2), _whole((70, 200), dtype, 3)
  views = [big[:, :264], big[:, 1:265], big[::2, 8:272], big[:1, :264].expand(70, 264), big.t()[:264, :33].t(),
           big.view(7, 10, 400)[:, :, 3:267], big.view(7, 10, 400).transpose(0, 1)[..., 16:280], big[4, :264]]
  weights = [wide[:, :264], wide[:89, 5:269], wide[:1, :264].expand(90, 264), wide.t()[:264].t(),
             _whole((264, 90), dtype, 5).t()]
  for x in views:
    for w in weights:
      outs = w.shape[0]
      if x.dim() == 1:
        r = res[2, 1:1 + outs]
      elif x.dim() == 2:
        r = res[:x.shape[0], 7:7 + outs]
      else:
        r = res[:1, :outs].expand(*x.shape[:-1], outs)
      b = _whole((2 * outs,), dtype, 9)[::2]
      want = x.double() @ w.double().t() + b.double() + r.double()
      assert torch.equal(fwn.linear_act(x, w, b, residual=r), want.to(dtype)), (x.shape, x.stride(), w.shape, w.stride())
      lx, lw = x.detach().requires_grad_(), w.detach().requires_grad_()
      out = fwn.linear_act(lx, lw, b, residual=r)
      assert torch.equal(out, want.to(dtype))
      g = _whole((*x.shape[:-1], 2 * outs), dtype, 6)[..., ::2]
      gx, gw = torch.autograd.grad(out, (lx, lw), g)
      g2, x2 = g.double().reshape(-1, outs), x.double().reshape(-1, 264)
      assert torch.equal(gx.reshape(-1, 264), (g2 @ w.double()).to(dtype)) and torch.equal(gw, (g2.t() @ x2).to(dtype))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_reads_and_writes_stay_inside(dtype):
  """Operands inside NaNs, and the rows behind x's last one, change nothing."""
  for rows, ins, outs in [(1, 72, 40), (24, 264, 72), (130, 136, 200), (257, 100, 65)]:
    def framed(r, c, seed):
      buf = torch.full((r + 8, c), float("nan"), device=DEV, dtype=dtype)
      buf[4:r + 4] = _whole((r, c), dtype, seed)
      return buf[4:r + 4]
    x, w, g = framed(rows, ins, 1), framed(outs, ins, 2), framed(rows, outs, 3)
    lx, lw = x.detach().requires_grad_(), w.detach().requires_grad_()
    out = fwn.linear_act(lx, lw)
    assert torch.equal(out, (x.double() @ w.double().t()).to(dtype))
    gx, gw = torch.autograd.grad(out, (lx, lw), g)
    assert torch.equal(gx, (g.double() @ w.double()).to(dtype)) and torch.equal(gw, (g.double().t() @ x.double()).to(dtype))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_special_values(dtype):
  """NaN and infinities reach the outputs that their rows and columns feed, and no others."""
  for rows in (3, 40, 300):
    x, w = _whole((rows, 96), dtype, 1), _whole((80, 96), dtype, 2)
    x[0, 0], w[:, 0] = float("nan"), 1
    x[1, 1], w[:, 1] = float("inf"), 1
    x[2, 2], w[:, 2] = torch.finfo(dtype).max, 1
    out = fwn.linear_act(x, w)
    assert out[0].isnan().all() and (out[1] == float("inf")).all() and torch.isfinite(out[2:].float()).all()
    want = (x.double() @ w.double().t())[2:]
    assert ((out[2:].double() - want).abs() <= _half(dtype) * want.abs() * 1.01).all()
    out = fwn.linear_act(x, w, activation="relu")
    assert out[0].isnan().all() and (out[1] == float("inf")).all()
  z = torch.tensor([[-200.0, -30, -1, 0, 1, 30, 200, 1e18]], device=DEV).to(dtype)
  eye = torch.eye(8, device=DEV, dtype=dtype)
  for act in ACTIVATIONS[1:]:
    leaf = _leaf(z)
    out = fwn.linear_act(leaf, eye, activation=act)
    want, slope = _act64(z.double(), act)
    torch.testing.assert_close(out.double(), want, rtol=_half(dtype) * 2 + 1e-6, atol=1e-6)
    gx, = torch.autograd.grad(out, leaf, torch.ones_like(out))
    torch.testing.assert_close(gx.double(), slope, rtol=_half(dtype) * 2 + 1e-6, atol=1e-6)


@gpu
def test_small_float32_values():
  """float32 operands over its whole exponent range keep float32's precision."""
  for scale in (1e-30, 1e-12, 1.0, 1e12):
    x, w = _normal((70, 200), torch.float32, 1) * scale, _normal((90, 200), torch.float32, 2) / scale
    want = x.double() @ w.double().t()
    _check(fwn.linear_act(x, w), want, 2.0 ** -24 * want.abs() + _sum_bound(200, x.double(), w.double()), scale)


def _codes(shape, seed):
  """e4m3 values: small whole numbers."""
  return _whole(shape, torch.float32, seed).to(torch.float8_e4m3fn)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,ins,outs", SIZES)
def test_8_bits_whole_numbers(rows, ins, outs, dtype):
  x, w, b, r = _codes((rows, ins), 1), _codes((outs, ins), 2), _whole((outs,), dtype, 3), _whole((rows, outs), dtype, 4)
  gen = _gen(7)
  xs = (2.0 ** torch.randint(-2, 3, (rows,), generator=gen)).to(DEV)
  ws = (2.0 ** torch.randint(-2, 3, (outs,), generator=gen)).to(DEV)
  z = (x.float().double() @ w.float().double().t()) * xs.double()[:, None] * ws.double()
  assert torch.equal(fwn.linear_act_q8(x, xs, w, ws, dtype=dtype), z.to(dtype))
  assert torch.equal(fwn.linear_act_q8(x, xs, w, ws, b, residual=r, dtype=dtype), (z + b.double() + r.double()).to(dtype))
  assert torch.equal(fwn.linear_act_q8(x, xs, w, ws, b, activation="relu", dtype=dtype), (z + b.double()).relu().to(dtype))


@gpu
@pytest.mark.parametrize("activation", ACTIVATIONS)
def test_8_bits_random(activation):
  for rows, ins, outs in [(1, 768, 1000), (24, 1040, 136), (300, 515, 257), (2000, 256, 512)]:
    x, xs = fwn.quantize_rows(_normal((rows, ins), torch.float32, 1))
    w, ws = fwn.quantize_rows(_normal((outs, ins), torch.float32, 2, ins ** -0.5))
    b, r = _normal((outs,), torch.bfloat16, 3), _normal((rows, outs), torch.bfloat16, 4)
    xd, wd = x.float().double() * xs.double()[:, None], w.float().double() * ws.double()[:, None]
    z = xd @ wd.t() + b.double()
    want = _act64(z, activation)[0] + r.double()
    slack = 2.0 ** -8 * want.abs() + 1.2 * _sum_bound(ins, xd, wd) + 2.0 ** -20 * (z.abs() + r.double().abs() + b.double().abs())
    _check(fwn.linear_act_q8(x, xs, w, ws, b, activation=activation, residual=r), want, slack, (rows, activation))


@gpu
def test_8_bits_strides_and_values():
  big, wide = _codes((70, 400), 1), _codes((90, 400), 2)
  one = lambda n: torch.ones(n, device=DEV)
  for x in (big[:, :272], big[:, 1:273], big[:, 16:288], big[::2, 3:100], big[:1, :272].expand(70, 272)):
    w = wide[:, 5:5 + x.shape[1]]
    want = x.float().double() @ w.float().double().t()
    assert torch.equal(fwn.linear_act_q8(x, one(x.shape[0]), w, one(90), dtype=torch.float32), want.float())
  # Every code of e4m3 is read as torch reads it, NaN among them.
  codes = torch.arange(256, device=DEV).to(torch.uint8).view(torch.float8_e4m3fn)
  for rows in (256, 16):
    x = codes.view(-1, 1)[:rows] if rows == 256 else codes.view(-1, 1)[:16]
    full = torch.zeros(rows, 32, device=DEV).to(torch.float8_e4m3fn).view(torch.uint8)
    full[:, :1] = x.view(torch.uint8)
    w = torch.ones(32, 32, device=DEV).to(torch.float8_e4m3fn)
    got = fwn.linear_act_q8(full.view(torch.float8_e4m3fn), one(rows), w, one(32), dtype=torch.float32)
    assert torch.equal(got.nan_to_num(-1), x.float().expand(rows, 32).nan_to_num(-1))
  # A row whose scale is NaN is NaN, the others stay.
  scale = one(70)
  scale[3] = float("nan")
  got = fwn.linear_act_q8(big, scale, wide, one(90))
  assert got[3].isnan().all() and not got[:3].isnan().any() and not got[4:].isnan().any()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_feed_forward_block(dtype):
  """The operators as a pre-norm block uses them, forward and backward, against float64."""
  rows, d, hidden = 333, 128, 520
  x, y = _normal((rows, d), dtype, 1), _normal((rows, d), dtype, 2)
  nw = (1 + 0.1 * _normal((d,), torch.float32, 3)).to(dtype)
  w1, b1 = _normal((hidden, d), dtype, 4, d ** -0.5), _normal((hidden,), dtype, 5, 0.1)
  w2, b2 = _normal((d, hidden), dtype, 6, hidden ** -0.5), _normal((d,), dtype, 7, 0.1)
  g = _normal((rows, d), dtype, 8)
  leaves = [_leaf(t) for t in (x, y, nw, w1, b1, w2, b2)]
  s, h = fwn.add_rms_norm(leaves[0], leaves[1], leaves[2])
  out = fwn.linear_act(fwn.linear_act(h, leaves[3], leaves[4], activation="gelu_tanh"), leaves[5], leaves[6], residual=s)
  grads = torch.autograd.grad(out, leaves, g)
  wide = [_leaf(t.double()) for t in (x, y, nw, w1, b1, w2, b2)]
  t = wide[0] + wide[1]
  n = t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * wide[2]
  z = torch.nn.functional.gelu(n @ wide[3].t() + wide[4], approximate="tanh")
  ref = z @ wide[5].t() + wide[6] + t
  want = torch.autograd.grad(ref, wide, g.double())
  # Ten roundings of half a step each lie between the inputs and any gradient (stored sum, norm, pre-activation, the
  # hidden values, the gradients of each), none amplified by more than 2 here; float32's sums of 520 terms add
  # as in _sum_bound, a hundred times 2^-24 relative to the tensors' norms.
  bar = 20 * _half(dtype) + 100 * 2.0 ** -24
  for a, b in zip((out, *grads), (ref.detach(), *want)):
    assert (a.double() - b).norm() <= bar * b.norm()
  if dtype == torch.bfloat16:
    # The same block served in 8 bits: e4m3's half step (2^-4 of a value, random) on each operand of two products.
    with torch.no_grad():
      s, q, qs = fwn.add_rms_norm_q8(x, y, nw)
      q1, q2 = fwn.quantize_rows(w1), fwn.quantize_rows(w2)
      hidden8 = fwn.quantize_rows(fwn.linear_act_q8(q, qs, *q1, b1, activation="gelu_tanh"))
      got = fwn.linear_act_q8(*hidden8, *q2, b2, residual=s)
    assert (got.double() - ref.detach()).norm() <= 4 * 2.0 ** -4 * ref.norm()


@gpu
def test_partial_gradients_and_saved_tensors():
  x, w, b, g = (_normal(s, torch.bfloat16, k) for k, s in enumerate([(40, 64), (72, 64), (72,), (40, 72)]))
  for act in (None, "silu"):
    full = [_leaf(t) for t in (x, w, b)]
    want = torch.autograd.grad(fwn.linear_act(*full, activation=act), full, g)
    for k in range(3):
      args = [x, w, b]
      args[k] = _leaf(args[k])
      got, = torch.autograd.grad(fwn.linear_act(*args, activation=act), args[k], g)
      assert torch.equal(got, want[k])
  frozen, leaf = w.clone(), _leaf(b)
  out = fwn.linear_act(x, frozen, leaf)
  frozen.zero_()  # no gradient reads it
  assert torch.equal(torch.autograd.grad(out, leaf, g)[0], g.double().sum(0).bfloat16())
  r = _leaf(g)
  out = fwn.linear_act(x, w, residual=r)
  assert torch.equal(torch.autograd.grad(out, r, g)[0], g)
  out = fwn.linear_act(_leaf(x), w)
  out.add_(1)  # a tensor of its own
  # A residual of one row for all: its gradient is summed by the expansion.
  row = _leaf(_whole((72,), torch.float32, 3).bfloat16())
  whole = _whole((40, 72), torch.bfloat16, 5)
  got, = torch.autograd.grad(fwn.linear_act(x, w, residual=row.expand(40, 72)), row, whole)
  assert torch.equal(got, whole.double().sum(0).bfloat16())


@gpu
@pytest.mark.parametrize("activation", ACTIVATIONS)
def test_second_derivative_and_batched_gradients(activation):
  x, w, b = (_leaf(_normal(s, torch.float32, k)) for k, s in enumerate([(6, 20), (10, 20), (10,)]))
  g = _normal((6, 10), torch.float32, 5)
  plain = lambda: {None: lambda t: t, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu,
                   "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[activation](x @ w.t() + b)
  own = lambda: fwn.linear_act(x, w, b, activation=activation)
  def second(fn):
    first, = torch.autograd.grad(fn(), x, g, create_graph=True)
    return torch.autograd.grad(first.square().sum(), (w, b), allow_unused=True)
  for p, q in zip(second(own), second(plain)):
    if q is not None and p is not None:
      torch.testing.assert_close(p, q, rtol=1e-4, atol=1e-3)
  gs = torch.stack([g, 2 * g])
  for p, q in zip(torch.autograd.grad(own(), (x, w, b), gs, is_grads_batched=True),
                  torch.autograd.grad(plain(), (x, w, b), gs, is_grads_batched=True)):
    torch.testing.assert_close(p, q, rtol=1e-4, atol=1e-3)


@gpu
def test_empty():
  w, b = _leaf(torch.ones(8, 16, device=DEV)), _leaf(torch.ones(8, device=DEV))
  x = torch.zeros(0, 16, device=DEV, requires_grad=True)
  out = fwn.linear_act(x, w, b, activation="gelu")
  assert out.shape == (0, 8)
  gx, gw, gb = torch.autograd.grad(out.sum(), (x, w, b))
  assert gx.shape == (0, 16) and not gw.any() and not gb.any()
  q, s = fwn.quantize_rows(torch.zeros(0, 16, device=DEV))
  wq, ws = fwn.quantize_rows(w.detach())
  assert fwn.linear_act_q8(q, s, wq, ws).shape == (0, 8)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_side_stream_and_graph(dtype):
  """On another stream, and captured: each replay against the eager results for new inputs. Sizes whose sums
  are split over workgroups and whose operands are laid out first."""
  for rows, ins, outs in [(4, 512, 96), (70, 2048, 64), (600, 100, 130)]:
    x, w, b = _leaf(_whole((rows, ins), dtype, 1)), _leaf(_whole((outs, ins), dtype, 2)), _leaf(_whole((outs,), dtype, 3))
    g = _whole((rows, outs), dtype, 4)
    def step():
      out = fwn.linear_act(x, w, b, activation="silu")
      with torch.no_grad():
        q, s = fwn.quantize_rows(x)
        p, t = fwn.quantize_rows(w)
        low = fwn.linear_act_q8(q, s, p, t, b.detach(), dtype=dtype)
      return [out.detach(), low, *torch.autograd.grad(out, (x, w, b), g)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
      first = step()
    torch.cuda.current_stream().wait_stream(side)
    for p, q in zip(first, step()):
      assert torch.equal(p, q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
      held = step()
    for k in range(3):
      with torch.no_grad():
        x.copy_(_whole((rows, ins), dtype, 20 + k))
      graph.replay()
      torch.cuda.synchronize()
      for p, q in zip(held, step()):
        assert torch.equal(p, q), k


@gpu
def test_refusals():
  x, w = torch.zeros(4, 16, device=DEV), torch.zeros(8, 16, device=DEV)
  v = lambda *s: torch.zeros(*s, device=DEV)
  for call in (lambda: fwn.linear_act(torch.zeros(4, 16), w), lambda: fwn.linear_act(x, torch.zeros(8, 16)),
               lambda: fwn.linear_act(x, v(8, 15)), lambda: fwn.linear_act(x, v(16)), lambda: fwn.linear_act(v(4, 0), v(8, 0)),
               lambda: fwn.linear_act(x, v(0, 16)), lambda: fwn.linear_act(x, w, v(7)), lambda: fwn.linear_act(x, w, v(1, 8)),
               lambda: fwn.linear_act(x, w, residual=v(4, 7)), lambda: fwn.linear_act(x, w, residual=v(8)),
               lambda: fwn.linear_act(x, w, activation="tanh"), lambda: fwn.linear_act(x, w, torch.zeros(8))):
    with pytest.raises(ValueError):
      call()
  for call in (lambda: fwn.linear_act(x.half(), w.half()), lambda: fwn.linear_act(x, w.bfloat16()),
               lambda: fwn.linear_act(x, w, v(8).bfloat16()), lambda: fwn.linear_act(x, w, residual=v(4, 8).bfloat16())):
    with pytest.raises(TypeError):
      call()
  q, s = fwn.quantize_rows(x)
  p, t = fwn.quantize_rows(w)
  for call in (lambda: fwn.linear_act_q8(q, s[:3], p, t), lambda: fwn.linear_act_q8(q, s, p, t[:7]),
               lambda: fwn.linear_act_q8(q, s.cpu(), p, t), lambda: fwn.linear_act_q8(q.cpu(), s, p, t),
               lambda: fwn.linear_act_q8(q, s, p, t, activation="x"), lambda: fwn.linear_act_q8(q, s, p[:, :8], t)):
    with pytest.raises(ValueError):
      call()
  for call in (lambda: fwn.linear_act_q8(x, s, p, t), lambda: fwn.linear_act_q8(q, s, w, t),
               lambda: fwn.linear_act_q8(q, s.double(), p, t), lambda: fwn.linear_act_q8(q, s, p, t, dtype=torch.float16),
               lambda: fwn.linear_act_q8(q, s, p, t, v(8))):
    with pytest.raises(TypeError):
      call()
  with pytest.raises(RuntimeError, match="no derivative"):
    fwn.linear_act_q8(q, s, p, t, _leaf(v(8).bfloat16()))


# ---- host validation of the C ABI: no GPU calls

F = 1 << 20  # addresses that are only compared


def _desc(rows=4, ins=64, outs=32, x_stride=64, w_stride=64, r_stride=32, dtype=nat.BF16, activation=0):
  return nat.LinearDesc(rows, x_stride, w_stride, r_stride, ins, outs, dtype, activation)


@pytest.mark.parametrize("bad,code", [(dict(rows=-1), 1), (dict(rows=1 << 40), 1), (dict(ins=0), 1), (dict(outs=0), 1),
                                      (dict(ins=(1 << 20) + 1), 1), (dict(ins=1 << 20, outs=1 << 20), 1), (dict(rows=1 << 31, outs=4096), 1), (dict(x_stride=-1), 1), (dict(w_stride=1 << 40), 1),
                                      (dict(r_stride=-5), 1), (dict(dtype=2), 2), (dict(activation=5), 2),
                                      (dict(activation=-1), 2)])
def test_bad_descriptors(bad, code):
  L, d = nat.lib(), _desc(**bad)
  size = ctypes.c_uint64()
  for query in (L.fwn_linear_act_workspace_size, L.fwn_linear_act_q8_workspace_size):
    assert query(d, F, 2 * F, ctypes.byref(size)) == code
  assert L.fwn_linear_act_bwd_workspace_size(d, F, 2 * F, 3 * F, 4 * F, 5 * F, 6 * F, ctypes.byref(size)) == code
  assert L.fwn_linear_act_launch(d, F, 2 * F, None, None, 3 * F, None, None, 0, None) == code
  assert L.fwn_linear_act_q8_launch(d, F, 2 * F, 3 * F, 4 * F, None, None, 5 * F, None, 0, None) == code
  assert L.fwn_linear_act_bwd_launch(d, F, 2 * F, None, 3 * F, 4 * F, 5 * F, 6 * F, None, 0, None) == code


def test_bad_pointers():
  L, d = nat.lib(), _desc()
  fwd, q8, bwd = L.fwn_linear_act_launch, L.fwn_linear_act_q8_launch, L.fwn_linear_act_bwd_launch
  act = _desc(activation=2)
  for query in (L.fwn_linear_act_workspace_size, L.fwn_linear_act_q8_workspace_size):
    assert query(d, F, 2 * F, None) == nat.ERR_INVALID_ARG
  assert L.fwn_linear_act_bwd_workspace_size(d, F, 2 * F, 3 * F, 4 * F, 5 * F, 6 * F, None) == nat.ERR_INVALID_ARG
  size = ctypes.c_uint64()
  odd = _desc(ins=100, x_stride=100)  # x is laid out: no workspace is an error
  assert L.fwn_linear_act_workspace_size(odd, F, 2 * F, ctypes.byref(size)) == nat.OK and size.value >= 4 * 208
  assert fwd(odd, F, 2 * F, None, None, 3 * F, None, None, 0, None) == nat.ERR_INVALID_ARG
  assert fwd(odd, F, 2 * F, None, None, 3 * F, None, 4 * F, size.value - 1, None) == nat.ERR_INVALID_ARG
  assert fwd(odd, F, 2 * F, None, None, 3 * F, None, 4 * F + 16, size.value, None) == nat.ERR_INVALID_ARG
  # Aligned whole rows are read where they lie: nothing is kept for them; misaligned ones are laid out.
  wide = _desc(rows=4096, ins=4096, outs=4096, x_stride=4096, w_stride=4096)
  assert L.fwn_linear_act_workspace_size(wide, F, 2 * F, ctypes.byref(size)) == nat.OK and size.value == 0
  assert L.fwn_linear_act_workspace_size(wide, F + 2, 2 * F, ctypes.byref(size)) == nat.OK and size.value == 4096 * 8192
  for rc in (fwd(None, F, 2 * F, None, None, 3 * F, None, None, 0, None), fwd(d, None, 2 * F, None, None, 3 * F, None, None, 0, None),
             fwd(d, F, None, None, None, 3 * F, None, None, 0, None), fwd(d, F, 2 * F, None, None, None, None, None, 0, None),
             fwd(d, F, 2 * F, None, None, F + 256, None, None, 0, None), fwd(d, F, 2 * F, None, None, 3 * F, 3 * F, None, 0, None),
             fwd(d, F, 2 * F, None, 3 * F, 3 * F, None, None, 0, None), fwd(d, F + 1, 2 * F, None, None, 3 * F, None, None, 0, None),
             fwd(d, F, 2 * F, 4 * F + 1, None, 3 * F, None, None, 0, None),
             q8(d, F, None, 3 * F, 4 * F, None, None, 5 * F, None, 0, None), q8(d, F, 2 * F, 3 * F, None, None, None, 5 * F, None, 0, None),
             q8(d, F, 2 * F, 3 * F, 4 * F, None, None, 4 * F, None, 0, None), q8(d, F, 2 * F + 2, 3 * F, 4 * F, None, None, 5 * F, None, 0, None),
             bwd(d, F, 2 * F, None, None, 4 * F, 5 * F, 6 * F, None, 0, None), bwd(d, F, None, None, 3 * F, 4 * F, 5 * F, 6 * F, None, 0, None),
             bwd(d, None, 2 * F, None, 3 * F, 4 * F, 5 * F, 6 * F, None, 0, None), bwd(d, F, 2 * F, None, 3 * F, 3 * F, 5 * F, 6 * F, None, 0, None),
             bwd(d, F, 2 * F, None, 3 * F, 4 * F, 4 * F, 6 * F, None, 0, None),
             bwd(act, F, 2 * F, None, 3 * F, 4 * F, 5 * F, 6 * F, 7 * F, 1 << 30, None),
             bwd(act, F, 2 * F, 8 * F, 3 * F, 4 * F, 5 * F, 6 * F, None, 0, None),
             bwd(act, F, 2 * F, 8 * F, 3 * F, 4 * F, 5 * F, 6 * F, 7 * F, 16, None),
             bwd(act, F, 2 * F, 8 * F, 3 * F, 4 * F, 5 * F, 6 * F, 7 * F + 8, 1 << 30, None)):
    assert rc == nat.ERR_INVALID_ARG
  assert fwd(_desc(rows=0), None, None, None, None, None, None, None, 0, None) == nat.OK


def test_needs_a_gpu_tensor():
  with pytest.raises(ValueError, match="CUDA"):
    fwn.linear_act(torch.zeros(2, 8), torch.zeros(4, 8))
  with pytest.raises(ValueError, match="CUDA"):
    fwn.linear_act_q8(torch.zeros(2, 8).to(torch.float8_e4m3fn), torch.ones(2), torch.zeros(4, 8).to(torch.float8_e4m3fn), torch.ones(4))


def test_slopes_are_the_activations_derivatives():
  z = torch.linspace(-6, 6, 1001, dtype=torch.float64)
  z = z[z != 0]
  for name, code in nat.ACTIVATIONS.items():
    torch.testing.assert_close(_slope(z, code), _act64(z, name)[1], rtol=1e-6, atol=1e-7)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_far_apart_rows(dtype):
  """Rows more than 2^20 elements apart, of every operand."""
  far = (1 << 20) + 72
  def spread(rows, cols, seed):
    buf = torch.full((rows * far,), float("nan"), device=DEV, dtype=dtype)
    return buf.as_strided((rows, cols), (far, 1)).copy_(_whole((rows, cols), dtype, seed))
  for rows in (3, 40):
    x, w, r = spread(rows, 200, 1), spread(24, 200, 2), spread(rows, 24, 3)
    lx, lw = x.detach().requires_grad_(), w.detach().requires_grad_()
    out = fwn.linear_act(lx, lw, residual=r)
    assert torch.equal(out, (x.double() @ w.double().t() + r.double()).to(dtype))
    g = _whole((rows, 24), dtype, 4)
    gx, gw = torch.autograd.grad(out, (lx, lw), g)
    assert torch.equal(gx, (g.double() @ w.double()).to(dtype)) and torch.equal(gw, (g.double().t() @ x.double()).to(dtype))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_offsets_past_32_bits(dtype):
  """x and its gradient past 2^32 bytes: rows near the end, to the bit."""
  size = 2 if dtype == torch.bfloat16 else 4
  ins = 16384
  rows = (1 << 32) // (ins * size) + 1000
  gen = torch.Generator(device=DEV).manual_seed(1)
  x = torch.randint(-2, 3, (rows, ins), generator=gen, device=DEV, dtype=torch.int8).to(dtype)
  w = _whole((40, ins), dtype, 2)
  g = torch.randint(-2, 3, (rows, 40), generator=gen, device=DEV, dtype=torch.int8).to(dtype)
  at = [0, 255, rows // 2, rows - 3, rows - 2, rows - 1]
  lx, lw = x.requires_grad_(), w.clone().requires_grad_()
  out = fwn.linear_act(lx, lw)
  assert torch.equal(out[at], (x.detach()[at].double() @ w.double().t()).to(dtype))
  gx, gw = torch.autograd.grad(out, (lx, lw), g)
  assert torch.equal(gx[at], (g[at].double() @ w.double()).to(dtype))
  cols = [0, 100, ins - 1]
  assert torch.equal(gw[:, cols], (g.double().t() @ x.detach()[:, cols].double()).to(dtype))


@gpu
def test_the_same_tensor_twice():
  """One tensor as x, weight and residual: small whole numbers, so that every sum is exact in float32."""
  for n in (24, 130):
    x = _leaf(_whole((n, n), torch.float32, 1))
    g = _whole((n, n), torch.float32, 2)
    out = fwn.linear_act(x, x, residual=x)
    gx, = torch.autograd.grad(out, x, g)
    d, e = x.detach().double(), g.double()
    assert torch.equal(out.double(), d @ d.t() + d)
    assert torch.equal(gx.double(), e @ d + e.t() @ d + e)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_two_streams_at_once(dtype):
  """Calls on two streams that may overlap, with split sums and operands laid out: the results of one after the other."""
  sizes = [(70, 2048, 64), (600, 100, 130), (24, 1030, 200), (300, 640, 512)]
  calls = []
  for k, (rows, ins, outs) in enumerate(sizes):
    x, w, b = _leaf(_whole((rows, ins), dtype, k)), _leaf(_whole((outs, ins), dtype, k + 10)), _leaf(_whole((outs,), dtype, k + 20))
    g = _whole((rows, outs), dtype, k + 30)
    calls.append(lambda x=x, w=w, b=b, g=g: [*torch.autograd.grad(fwn.linear_act(x, w, b, activation="silu"), (x, w, b), g),
                                             fwn.linear_act(x.detach(), w.detach(), b.detach())])
  want = [call() for call in calls]
  torch.cuda.synchronize()
  streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], {}
  for repeat in range(3):
    for k, call in enumerate(calls):
      with torch.cuda.stream(streams[(k + repeat) % 2]):
        got[repeat, k] = call()
  torch.cuda.synchronize()
  for (repeat, k), outs in got.items():
    for p, q in zip(outs, want[k]):
      assert torch.equal(p, q), (repeat, sizes[k])
