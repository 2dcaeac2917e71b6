"""The norms around a block (``sandwich.py``, ``fwn_sandwich_norm_*``) against their formulas in float64.

Bounds. A row's sums are float32 chains of at most 32 products a thread and 10 additions across threads, so a mean square is
off by at most 64 x 2^-24 of itself and 1 / sqrt of it by half that; with the few operations around them every value
computed from it stays within NEAR = 2^-18 of its terms' magnitudes. What is computed from such a value carries its error on: the
functions below add the errors up beside the values. Sums over rows add a chain of at most 256 roundings. On top comes the one
rounding to the output's type, half a step: eps / 2 of the value."""
import ctypes

import pytest
import torch

import faster_weathernext_amd as fwn
from faster_weathernext_amd import _native as nat
from oracle import dropout as oracle

DEV = "cuda"
gpu = pytest.mark.gpu
NEAR = 2.0 ** -18
CHAIN = 256 * 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float32]
STATE = (0x0123456789abcdef, 0xfedcba9876543210)


def _half(dtype):
  return torch.finfo(dtype).eps / 2


def _normal(shape, dtype, seed, mean=0.0):
  return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) + mean).to(dtype).to(DEV)


def _mean(t):
  return t.mean(-1, keepdim=True)


def _kept(shape, p):
  rows = 1
  for n in shape[:-1]:
    rows *= n
  m = 65536 / (65536 - oracle.border(p)) if oracle.border(p) < 65536 else 0.0
  return torch.from_numpy(oracle.kept(rows, shape[-1], p, *STATE)).to(DEV).view(shape).double() * m


class Case:
  """One call's inputs and its formula in float64."""

  def __init__(self, shape, dtype, gate=None, gate_dtype=None, post=True, pre=True, weight_dtype=None, scale=1.0,
               post_norm=True, p=0.0, seed=0, eps=1e-5):
    c = shape[-1]
    self.dtype, self.scale, self.post_norm, self.p, self.eps = dtype, scale, post_norm, p, eps
    weight_dtype = weight_dtype or dtype
    self.x, self.y = _normal(shape, dtype, seed), _normal(shape, dtype, seed + 1)
    self.post = _normal((c,), weight_dtype, seed + 2, 1.0) if post and post_norm else None
    self.pre = _normal((c,), weight_dtype, seed + 3, 1.0) if pre else None
    gate_shape = {None: None, "channel": (c,), "member": (shape[0], c), "full": shape}[gate]
    self.gate = None if gate is None else _normal(gate_shape, gate_dtype or dtype, seed + 4, 0.5)
    self.member = gate == "member"
    self.leaves = [t for t in (self.x, self.y, self.post, self.pre, self.gate) if t is not None]

  def call(self, **other):
    args = dict(gate=self.gate, scale=self.scale, post_norm=self.post_norm, p=self.p, rng=STATE, eps=self.eps)
    return fwn.sandwich_norm(self.x, self.y, self.post, self.pre, **{**args, **other})

  def wide(self):
    """(gate, post, pre, keep) as float64 tensors that broadcast."""
    one = torch.ones((), dtype=torch.float64, device=DEV)
    gate, post, pre = (one if t is None else t.detach().double() for t in (self.gate, self.post, self.pre))
    if self.member:
      gate = gate.view(gate.shape[0], *[1] * (self.x.dim() - 2), -1)
    return gate, post, pre, _kept(self.x.shape, self.p) if self.p else one

  def check_forward(self, s, out, note=""):
    assert s.dtype == out.dtype == self.dtype and s.shape == out.shape == self.x.shape
    gate, post, pre, keep = self.wide()
    y = self.y.double()
    r1 = (_mean(y.square()) + self.eps) ** -0.5 if self.post_norm else 1.0
    branch, base = keep * gate * y * r1 * post, self.scale * self.x.double()
    near(s, base + branch, _half(self.dtype) * (base + branch).abs() + NEAR * (base.abs() + branch.abs()) + 1e-37, note)
    t = s.double()
    want = t * (_mean(t.square()) + self.eps) ** -0.5 * pre
    near(out, want, (_half(self.dtype) + NEAR) * want.abs() + 1e-37, note)

  def gradients(self, s, g_sum, g_out):
    """{name: (value, bound without the last rounding)} at the stored rows s."""
    gate, post, pre, keep = self.wide()
    s, y, c = s.detach().double(), self.y.detach().double(), s.shape[-1]
    zero = torch.zeros_like(s)
    gs, go = (zero if g is None else g.double() for g in (g_sum, g_out))
    r2 = (_mean(s.square()) + self.eps) ** -0.5
    a = go * pre
    ds = gs + r2 * (a - s * r2.square() * _mean(a * s))
    e_ds = NEAR * (gs.abs() + r2 * (a.abs() + s.abs() * r2.square() * _mean((a * s).abs())))
    db, e_db = ds * keep, e_ds * keep
    r1 = (_mean(y.square()) + self.eps) ** -0.5 if self.post_norm else torch.ones_like(y[..., :1])
    unit, w = y * r1, gate * post
    q, e_q = db * w, (e_db + NEAR * db.abs()) * w.abs()
    gy, e_gy = q, e_q
    if self.post_norm:
      gy = r1 * (q - unit * _mean(q * unit))
      e_gy = r1 * (e_q + unit.abs() * _mean(e_q * unit.abs()) + NEAR * (q.abs() + unit.abs() * _mean((q * unit).abs())))
    res = {"x": (self.scale * ds, abs(self.scale) * e_ds), "y": (gy, e_gy)}
    def total(term, e_term, over):
      e_term = e_term + (NEAR + CHAIN) * term.abs()
      return over(term), over(e_term)
    rows = lambda t: t.reshape(-1, c).sum(0)
    if self.post is not None:
      res["post"] = total(db * gate * unit, e_db * (gate * unit).abs(), rows)
    if self.pre is not None:
      res["pre"] = total(go * s * r2, zero, rows)
    if self.gate is not None:
      over = rows
      if self.member:
        over = lambda t: t.reshape(self.gate.shape[0], -1, c).sum(1)
      elif self.gate.shape == self.x.shape and self.x.dim() > 1:
        over = lambda t: t
      res["gate"] = total(db * unit * post, e_db * (unit * post).abs(), over)
    return res

  def check_gradients(self, g_sum, g_out, note=""):
    names = [n for n in ("x", "y", "post", "pre", "gate") if getattr(self, n) is not None]
    leaves = [getattr(self, n).detach().clone().requires_grad_() for n in names]
    call = dict(zip(names, leaves))
    s, out = fwn.sandwich_norm(call["x"], call["y"], call.get("post"), call.get("pre"), gate=call.get("gate"), scale=self.scale,
                               post_norm=self.post_norm, p=self.p, rng=STATE, eps=self.eps)
    self.check_forward(s.detach(), out.detach(), note)
    outs, gs = zip(*[(o, g) for o, g in ((s, g_sum), (out, g_out)) if g is not None])
    got = torch.autograd.grad(outs, leaves, gs, allow_unused=True)
    want = self.gradients(s, g_sum, g_out)
    for name, g, leaf in zip(names, got, leaves):
      value, bound = want[name]
      if g is None:
        assert not value.any()
        continue
      assert g.dtype == leaf.dtype and g.shape == leaf.shape
      near(g, value, bound + _half(leaf.dtype) * value.abs() + 1e-37, (note, name))
    return got


def near(got, want, slack, note=""):
  off = (got.double() - want).abs() - slack
  assert torch.isfinite(got.float()).all(), note
  assert off.max() <= 0, (note, off.max().item())


# Sizes about each change of instance; odd ones.
CHANNELS = [1, 7, 8, 64, 127, 129, 250, 256, 264, 511, 768, 1000, 1283, 2048, 2056, 4097, 5120, 8200, 12289, 16384]
GATES = [None, "channel", "member", "full"]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("channels", CHANNELS)
def test_forward(channels, dtype):
  for k, (members, n) in enumerate(((1, 1), (2, 3), (3, 23))):
    shape = (members, n, channels)
    for gate in GATES:
      case = Case(shape, dtype, gate, scale=(1.0, 0.5, -1.25)[k])
      case.check_forward(*case.call(), (shape, gate))
    Case(shape, dtype, "member", torch.float32, weight_dtype=torch.float32, p=0.1).check_forward(
        *Case(shape, dtype, "member", torch.float32, weight_dtype=torch.float32, p=0.1).call(), shape)
    for other in (dict(post_norm=False), dict(post_norm=False, gate="channel", p=0.5), dict(post=False), dict(pre=False),
                  dict(post=False, pre=False, p=1.0)):
      case = Case(shape, dtype, **other)
      case.check_forward(*case.call(), (shape, other))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("channels", CHANNELS)
def test_gradients(channels, dtype):
  for k, (members, n) in enumerate(((1, 1), (5, 1), (2, 3), (3, 101))):
    shape = (members, n, channels)
    g_sum, g_out = _normal(shape, dtype, 11), _normal(shape, dtype, 12)
    for gate in GATES:
      Case(shape, dtype, gate, scale=(1.0, 0.5, -1.25, 1.0)[k], p=0.0 if k % 2 else 0.25).check_gradients(g_sum, g_out, (shape, gate))
  shape = (2, 37, channels)
  g_sum, g_out = _normal(shape, dtype, 11), _normal(shape, dtype, 12)
  for other in (dict(gate="member", gate_dtype=torch.float32, weight_dtype=torch.float32, p=0.1),
                dict(gate="full", gate_dtype=torch.float32, p=0.1), dict(post_norm=False, gate="channel"),
                dict(post_norm=False, p=0.5), dict(post=False, gate="member"), dict(pre=False, gate="full"), dict(p=1.0)):
    Case(shape, dtype, **other).check_gradients(g_sum, g_out, other)
  for one in ((g_sum, None), (None, g_out)):
    Case(shape, dtype, "member", p=0.1).check_gradients(*one)


@gpu
@pytest.mark.parametrize("members,n", [(1, 20001), (7, 3001), (1500, 3), (4099, 1), (1025, 2), (40, 512)])
def test_many_rows(members, n):
  """More rows than one round of workgroups takes; a few groups of many rows, and more groups than workgroups. CHAIN counts the
  longest sum: 20,001 rows over 1,024 workgroups are 20 a thread, 4 places, and 16 + 16 partial rows."""
  shape = (members, n, 264)
  g = _normal(shape, torch.bfloat16, 5)
  for gate in GATES:
    case = Case(shape, torch.bfloat16, gate, torch.float32, p=0.1, scale=0.7)
    first = case.check_gradients(g, g.flip(0), gate)
    for a, b in zip(first, case.check_gradients(g, g.flip(0), gate)):
      assert torch.equal(a, b)  # sums in a fixed order


@gpu
def test_gradient_against_differences():
  """A directional difference of the float64 formula at the float32 inputs."""
  case = Case((2, 3, 40), torch.float32, "member", scale=0.8, p=0.3)
  g_sum, g_out = _normal((2, 3, 40), torch.float32, 11), _normal((2, 3, 40), torch.float32, 12)
  names = ["x", "y", "post", "pre", "gate"]
  dirs = {n: _normal(getattr(case, n).shape, torch.float32, 20 + k).double() for k, n in enumerate(names)}
  keep = _kept((2, 3, 40), 0.3)
  def f(t):
    v = {n: getattr(case, n).double() + t * dirs[n] for n in names}
    y = v["y"] * (_mean(v["y"].square()) + case.eps) ** -0.5
    s = 0.8 * v["x"] + keep * v["gate"][:, None] * y * v["post"]
    return (s * g_sum.double() + s * (_mean(s.square()) + case.eps) ** -0.5 * v["pre"] * g_out.double()).sum()
  leaves = [getattr(case, n).clone().requires_grad_() for n in names]
  s, out = fwn.sandwich_norm(leaves[0], leaves[1], leaves[2], leaves[3], gate=leaves[4], scale=0.8, p=0.3, rng=STATE, eps=case.eps)
  grads = torch.autograd.grad((s, out), leaves, (g_sum, g_out))
  slope = sum((g.double() * dirs[n]).sum() for g, n in zip(grads, names))
  h = 1e-5  # central: an error of h^2 times the third derivative, and 1e-14 / h
  assert abs((f(h) - f(-h)) / (2 * h) - slope) < 1e-3


@gpu
def test_partial_gradients():
  """Each leaf alone has the gradient that it has among all."""
  case = Case((2, 9, 128), torch.bfloat16, "member", p=0.2)
  g = _normal((2, 9, 128), torch.bfloat16, 9)
  names = ["x", "y", "post", "pre", "gate"]
  def grads(which):
    leaves = {n: getattr(case, n).clone().requires_grad_(n in which) for n in names}
    s, out = fwn.sandwich_norm(leaves["x"], leaves["y"], leaves["post"], leaves["pre"], gate=leaves["gate"], p=0.2, rng=STATE)
    return torch.autograd.grad((s, out), [leaves[n] for n in which], (g, g))
  every = dict(zip(names, grads(names)))
  for n in names:
    assert torch.equal(grads([n])[0], every[n]), n
  for pair in (["x", "pre"], ["post", "gate"], ["y", "gate"]):
    for n, got in zip(pair, grads(pair)):
      assert torch.equal(got, every[n]), (pair, n)


def _plain(x, y, post, pre, gate, keep, scale, eps):
  unit = y * torch.rsqrt(_mean(y.square()) + eps)
  s = scale * x + keep * gate * unit * post
  return s, s * torch.rsqrt(_mean(s.square()) + eps) * pre


@gpu
@pytest.mark.parametrize("gate", ["channel", "member", "full"])
def test_second_derivative_and_batched_gradients(gate):
  case = Case((2, 3, 64), torch.float32, gate, p=0.25)
  leaves = [t.clone().requires_grad_() for t in case.leaves]
  keep = _kept((2, 3, 64), 0.25).float()
  g = _normal((2, 3, 64), torch.float32, 30)
  def own():
    x, y, post, pre, w = leaves
    return fwn.sandwich_norm(x, y, post, pre, gate=w, scale=0.5, p=0.25, rng=STATE, eps=1e-5)
  def plain():
    x, y, post, pre, w = leaves
    return _plain(x, y, post, pre, w[:, None] if gate == "member" else w, keep, 0.5, 1e-5)
  def both(fn):
    first = torch.autograd.grad(fn(), leaves, (g, g), create_graph=True)
    return torch.autograd.grad(sum(t.square().sum() for t in first), leaves)
  for a, b in zip(both(own), both(plain)):
    torch.testing.assert_close(a, b, rtol=2e-3, atol=2e-3 * float(b.abs().max()))
  gs = torch.stack([g, 2 * g])
  for a, b in zip(torch.autograd.grad(own()[1], leaves, gs, is_grads_batched=True),
                  torch.autograd.grad(plain()[1], leaves, gs, is_grads_batched=True)):
    torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-4)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(dtype):
  """Slices, one row for all, transposed and misaligned tensors."""
  big = _normal((33, 400), dtype, 1)
  views = [big[:, :264], big[:, 1:265], big[::2, 8:272], big[:1, :264].expand(33, 264), big.t()[:264, :33].t(),
           big.view(3, 11, 400)[:, :, :264], big.view(3, 11, 400).transpose(0, 1)[..., 16:280], big[:, :264][5]]
  w = _normal((1600,), dtype, 2)
  for k, x in enumerate(views):
    for post, pre in ((w[:264], w[300:564]), (w[1:265], w[::2][:264])):
      y = x.flip(0)
      for gate in (None, pre, x[0] if x.dim() == 3 else x):
        if gate is not None and x.dim() == 3 and gate.dim() == 2:
          gate = big[:x.shape[0], 3:267]  # [members, channels]
        case = Case((1, 264), dtype)
        case.x, case.y, case.post, case.pre, case.gate = x, y, post, pre, gate
        case.member = x.dim() == 3 and gate is not None and gate.dim() == 2
        case.check_forward(*case.call(), k)
        g = _normal(x.shape, dtype, 7)
        strided = g.t().contiguous().t() if g.dim() == 2 else g
        got = case.check_gradients(strided, g, k)
        assert all(t is None or t.is_contiguous() for t in got)


@gpu
def test_the_same_tensor_in_every_place():
  w = _normal((72,), torch.float32, 1).requires_grad_()
  x = _normal((9, 72), torch.float32, 2).requires_grad_()
  g = _normal((9, 72), torch.float32, 3)
  s, out = fwn.sandwich_norm(x, x, w, w, gate=w)
  got = torch.autograd.grad((s, out), (x, w), (g, g))
  want = torch.autograd.grad(_plain(x, x, w, w, w, 1.0, 1.0, 1e-6), (x, w), (g, g))
  for a, b in zip(got, want):
    torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-4)


@gpu
def test_one_row_is_every_gate():
  """[channels], [1, channels] and x's shape are the same gate of one row."""
  case = Case((1, 1, 520), torch.bfloat16, "channel", p=0.3)
  g = _normal((1, 1, 520), torch.bfloat16, 8)
  results = []
  for shape in ((520,), (1, 520), (1, 1, 520)):
    gate = case.gate.view(shape).clone().requires_grad_()
    s, out = case.call(gate=gate)
    results.append([s, out, torch.autograd.grad((s, out), gate, (g, g))[0].view(-1)])
  for other in results[1:]:
    for a, b in zip(results[0], other):
      assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_are_not_finite(dtype):
  """NaN and infinities stay in their rows; rows of zeros are zeros."""
  case = Case((6, 72), dtype, "channel")
  case.x[1, 3], case.y[2, 5], case.x[3], case.y[4] = float("nan"), float("inf"), 0, 0
  s, out = case.call()
  assert s[1].isnan().sum() == 1 and out[1].isnan().all()
  assert s[2].isnan().sum() == 1 and out[2].isnan().all()  # the infinity times 1 / infinity
  for row in (0, 3, 4, 5):
    assert s[row].isfinite().all() and out[row].isfinite().all()
  assert torch.equal(s[4], case.x[4])
  case.x[3], case.y[3] = 0, 0
  s, out = case.call()
  assert not s[3].any() and not out[3].any()
  leaves = [t.clone().requires_grad_() for t in (case.x, case.y)]
  g = _normal((6, 72), dtype, 3)
  grads = torch.autograd.grad(fwn.sandwich_norm(*leaves, case.post, case.pre, gate=case.gate, eps=1e-5), leaves, (g, g))
  for row in (0, 3, 4, 5):
    assert all(t[row].isfinite().all() for t in grads)


@gpu
def test_empty():
  w = torch.ones(64, device=DEV, requires_grad=True)
  for shape, gate in (((0, 64), (64,)), ((3, 0, 64), (3, 64)), ((0, 5, 64), (0, 64)), ((2, 0, 64), (2, 0, 64))):
    x, gate = torch.zeros(shape, device=DEV, requires_grad=True), torch.ones(gate, device=DEV, requires_grad=True)
    s, out = fwn.sandwich_norm(x, x, w, w, gate=gate, p=0.1, rng=STATE)
    assert s.shape == out.shape == shape
    gx, gw, gg = torch.autograd.grad((s.sum() + out.sum()), (x, w, gate))
    assert gx.shape == shape and not gw.any() and gg.shape == gate.shape and not gg.any()


@gpu
def test_side_stream_and_graph():
  """On another stream, and captured: each replay against the eager results for new inputs and a new state."""
  case = Case((4, 25, 520), torch.bfloat16, "member", torch.float32)
  state = torch.tensor([5, 0], device=DEV)
  g = _normal((4, 25, 520), torch.bfloat16, 9)
  for t in case.leaves:
    t.requires_grad_()
  def step():
    s, out = case.call(p=0.1, rng=state)
    return [s.detach(), out.detach(), *torch.autograd.grad((s, out), case.leaves, (g, g))]
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
    state[1] = k
    with torch.no_grad():
      case.x.copy_(_normal(case.x.shape, torch.bfloat16, 20 + k))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(held, step()):
      assert torch.equal(a, b), k


@gpu
def test_against_the_separate_calls():
  """The forward as rms_norm, dropout and rms_norm one after the other, in float32; the same elements are dropped."""
  case = Case((3, 40, 264), torch.float32, "member", p=0.4, scale=0.5)
  b = fwn.rms_norm(case.y, case.post, eps=case.eps) * case.gate[:, None]
  s = fwn.dropout(b, 0.4, STATE, residual=0.5 * case.x)
  own = case.call()
  torch.testing.assert_close(own[0], s, rtol=1e-5, atol=1e-5)
  torch.testing.assert_close(own[1], fwn.rms_norm(s, case.pre, eps=case.eps), rtol=1e-5, atol=1e-5)


@gpu
def test_offsets_past_32_bits():
  """Rows whose bytes lie past 2^32 from the first, forward and backward."""
  rows, c, at = 140000, 16384, [0, 1, 70000, 139998, 139999]  # 4.6 GB a tensor
  gen = torch.Generator(device=DEV).manual_seed(1)
  make = lambda: torch.randint(-4, 5, (rows, c), generator=gen, device=DEV, dtype=torch.int8).to(torch.bfloat16)
  x, y, gate = make().requires_grad_(), make().requires_grad_(), make().requires_grad_()
  w = _normal((c,), torch.bfloat16, 2, 1.0)
  s, out = fwn.sandwich_norm(x, y, w, w, gate=gate)
  gx, gy, gg = torch.autograd.grad((s, out), (x, y, gate), (x.detach(), y.detach()))
  case = Case((5, c), torch.bfloat16, "full", eps=1e-6)
  case.x, case.y, case.post, case.pre, case.gate = x.detach()[at], y.detach()[at], w, w, gate.detach()[at]
  case.check_forward(s.detach()[at], out.detach()[at])
  want = case.gradients(s.detach()[at], case.x, case.y)
  for name, got in (("x", gx), ("y", gy), ("gate", gg)):
    value, bound = want[name]
    near(got[at], value, bound + 2.0 ** -8 * value.abs() + 1e-37, name)


@gpu
def test_refusals():
  x, w = torch.zeros(2, 4, 64, device=DEV), torch.ones(64, device=DEV)
  n = fwn.sandwich_norm
  for call in (lambda: n(torch.zeros(4, 64), torch.zeros(4, 64)), lambda: n(x, x[:1]), lambda: n(x, x.bfloat16()),
               lambda: n(torch.zeros(1, 16385, device=DEV), torch.zeros(1, 16385, device=DEV)), lambda: n(x, x, w[:63]),
               lambda: n(x, x, w, w[:63]), lambda: n(x, x, torch.ones(64)), lambda: n(x, x, w, post_norm=False),
               lambda: n(x, x, gate=torch.ones(64)), lambda: n(x, x, gate=torch.ones(4, 64, device=DEV)),
               lambda: n(x, x, gate=torch.ones(2, 4, 1, device=DEV)), lambda: n(x, x, gate=torch.ones(2, 1, 64, device=DEV)),
               lambda: n(x, x, gate=0.5), lambda: n(x, x, p=0.1), lambda: n(x, x, p=1.5, rng=STATE), lambda: n(x, x, p=0.1, rng=7),
               lambda: n(x, x, p=0.1, rng=torch.zeros(2, dtype=torch.int64))):
    with pytest.raises(ValueError):
      call()
  for call in (lambda: n(x.half(), x.half()), lambda: n(x, x, w.bfloat16()), lambda: n(x, x, w, w.double()),
               lambda: n(x, x, gate=w.bfloat16())):
    with pytest.raises(TypeError):
      call()
  for call in (lambda: n(x, x, eps=-1.0), lambda: n(x, x, scale=float("inf"))):
    with pytest.raises(nat.FwnError):
      call()
  import torch.autograd.forward_ad as fwad
  with fwad.dual_level():
    dual = fwad.make_dual(x, torch.ones_like(x))
    with pytest.raises(RuntimeError):
      n(x, dual)


# ---- host validation of the C ABI: no GPU calls

F = 4096  # an address that is only compared


def _desc(rows=4, gate_rows=4, channels=64, x_stride=64, y_stride=64, dtype=nat.BF16, gate=nat.BF16, post=nat.BF16, pre=nat.BF16,
          post_norm=1, eps=1e-6, scale=1.0, p=0.0, state=None):
  return nat.SandwichDesc(rows, gate_rows, x_stride, y_stride, channels, dtype, gate, post, pre, post_norm, eps, scale,
                          nat.Dropout(p, 1, 2, state))


@pytest.mark.parametrize("bad,code", [(dict(rows=-1), 1), (dict(rows=1 << 32), 1), (dict(channels=0), 1), (dict(channels=16385), 1),
                                      (dict(x_stride=-1), 1), (dict(y_stride=1 << 62), 1), (dict(dtype=2), 2),
                                      (dict(dtype=nat.F32), 2), (dict(gate=3), 2), (dict(post=-1), 2), (dict(pre=9), 2),
                                      (dict(post_norm=2), 1), (dict(eps=-1.0), 1), (dict(eps=float("nan")), 1),
                                      (dict(scale=float("inf")), 1), (dict(p=2.0), 1), (dict(p=float("nan")), 1),
                                      (dict(state=F + 4), 1), (dict(gate_rows=0), 1), (dict(gate_rows=3), 1),
                                      (dict(gate_rows=8), 1)])
def test_bad_descriptors(bad, code):
  L, d = nat.lib(), _desc(**bad)
  size = ctypes.c_uint64()
  assert L.fwn_sandwich_norm_launch(d, F, 2 * F, 3 * F, 4 * F, 5 * F, 6 * F, 7 * F, None) == code
  assert L.fwn_sandwich_norm_bwd_workspace_size(d, 1, ctypes.byref(size)) == code
  assert L.fwn_sandwich_norm_bwd_launch(d, F, 2 * F, 3 * F, 4 * F, 5 * F, 6 * F, 7 * F, 8 * F, 9 * F, 10 * F, 11 * F, 12 * F, 64 * F,
                                        1 << 20, None) == code


def test_bad_pointers():
  L, d = nat.lib(), _desc()
  fwd, bwd = L.fwn_sandwich_norm_launch, L.fwn_sandwich_norm_bwd_launch
  good = [F, 2 * F, 3 * F, 4 * F, 5 * F, 6 * F, 7 * F]  # x y gate post pre, sum out
  for at, value in ((0, None), (1, None), (5, None), (6, None), (0, F + 1), (1, 2 * F + 1), (2, 3 * F + 1), (3, 4 * F + 1),
                    (4, 5 * F + 1), (5, 6 * F + 1), (6, 7 * F + 1), (5, F + 64), (5, 2 * F), (5, 3 * F), (5, 4 * F), (5, 5 * F),
                    (5, 7 * F + 64), (6, F), (6, 6 * F)):
    args = list(good)
    args[at] = value
    assert fwd(d, *args, None) == nat.ERR_INVALID_ARG, (at, value)
  assert fwd(None, *good, None) == nat.ERR_INVALID_ARG
  assert fwd(_desc(rows=0), *[None] * 7, None) == nat.OK
  # s y gate post pre g_sum g_out, gx gy g_gate g_post g_pre, workspace
  good = [k * F for k in range(1, 13)] + [64 * F]
  for at, value in ((0, None), (1, None), (2, None), (3, None), (4, None), (12, None), (12, 64 * F + 8), (7, F), (8, 2 * F), (9, 3 * F),
                    (10, 4 * F), (11, 5 * F), (7, 9 * F), (9, 11 * F), (10, 12 * F), (12, 7 * F), (7, 7 * F + 32), (5, 6 * F + 1)):
    args = list(good)
    args[at] = value
    assert bwd(d, *args, 1 << 20, None) == nat.ERR_INVALID_ARG, (at, value)
  assert bwd(d, *good, 64, None) == nat.ERR_INVALID_ARG


def test_workspace_is_small():
  L = nat.lib()
  size = ctypes.c_uint64()
  for rows, gate_rows in ((1 << 31, 1 << 31), (1 << 31, 2), (1 << 31, 1 << 20), (40962, 40962), (5, 5), (0, 1)):
    for gate in (0, 1):
      assert L.fwn_sandwich_norm_bwd_workspace_size(_desc(rows=rows, gate_rows=gate_rows, channels=512, x_stride=512, y_stride=512),
                                                    gate, ctypes.byref(size)) == nat.OK
      assert 0 < size.value <= 3 * 2048 * 512 * 4


def test_needs_a_gpu_tensor():
  with pytest.raises(ValueError, match="CUDA"):
    fwn.sandwich_norm(torch.zeros(2, 64), torch.zeros(2, 64))
