"""``linear_act`` at values where a product, a scale or an activation can lose float32's precision, against float64."""
import pytest
import torch

import faster_weathernext_amd as fwn

DEV = "cuda"
gpu = pytest.mark.gpu
STEP = 2.0 ** -24  # half a step of float32


def _normal(shape, seed, std=1.0):
  return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(DEV)


def _bound(k, a, b):
  """A float32 sum of k products: (8 sqrt(k) + 16) 2^-24 of the rows' norms, as in test_linear_act."""
  return (8 * k ** 0.5 + 16) * STEP * a.norm(dim=1)[:, None] * b.norm(dim=1)


def _near(got, want, bound):
  assert torch.isfinite(got).all()
  assert ((got.double() - want).abs() - bound - STEP * want.abs() - 2.0 ** -149).max() <= 0


@gpu
@pytest.mark.parametrize("rows", [24, 300])
def test_float32_single_products(rows):
  """Products of one term, mantissas of all ones among them: the parts' products that are left out are below
  2^-24 (1 + 2^-9) of the product, and each of the last additions rounds by as much: four half steps. Over many
  products the errors have no direction: their mean is within a tenth of a half step of zero (the
  mean of 30,000 errors of at most four has a deviation below 0.03)."""
  x, w = _normal((rows, 1), 1), _normal((128, 1), 2)
  for mask in (0, 0xffff, 0xff, 0xff00):
    a, b = ((t.view(torch.int32) | mask).view(torch.float32) for t in (x, w))
    want = a.double() @ b.double().t()
    off = (fwn.linear_act(a, b).double() - want) / want.abs()
    assert off.abs().max() <= 4 * STEP, off.abs().max().item() / STEP
    if mask == 0 and rows == 300:
      assert ((off * want.sign()).mean() / STEP).abs() <= 0.1
  one = torch.tensor([[0x3f80ffff]], dtype=torch.int32, device=DEV).view(torch.float32)
  got = fwn.linear_act(one.expand(rows, 1), one)
  assert ((got.double() - one.double() ** 2).abs() <= 4 * STEP * one.double() ** 2).all()


@gpu
def test_float32_sums_of_one_sign():
  """Sums of positive terms: errors of products that all point one way would add up. A float32 sum's do
  not: its roundings, at most STEP of the sum each, add as a root, sqrt(k) of them."""
  x, w = _normal((300, 64), 1).abs(), _normal((128, 64), 2).abs()
  want = x.double() @ w.double().t()
  off = (fwn.linear_act(x, w).double() - want) / want
  assert off.mean().abs() <= 0.15 * STEP, off.mean().item() / STEP
  assert off.abs().max() <= 8 * STEP


@gpu
@pytest.mark.parametrize("rows", [24, 300])
@pytest.mark.parametrize("scale", [1e-38, 1e-37, 1e-36, 1e-35, 1e-33, 1e-30, 1e30, 1e33, 1e35, 1e36])
def test_float32_exponents(rows, scale):
  """Operands near either end of float32's range, subnormal ones among them, in the output and both gradients.
  A product below the least normal number rounds to 2^-150 by itself: as many of them as the sum has terms."""
  x, w, g = _normal((rows, 200), 1, scale), _normal((90, 200), 2, 0.01 / scale), _normal((rows, 90), 3)
  lx, lw = x.clone().requires_grad_(), w.clone().requires_grad_()
  out = fwn.linear_act(lx, lw)
  gx, gw = torch.autograd.grad(out, (lx, lw), g)
  xd, wd, gd = x.double(), w.double(), g.double()
  _near(out.detach(), xd @ wd.t(), _bound(200, xd, wd))
  _near(gx, gd @ wd, _bound(90, gd, wd.t()) + 90 * 2.0 ** -150)
  _near(gw, gd.t() @ xd, _bound(rows, gd.t(), xd.t()) + rows * 2.0 ** -150)


@gpu
@pytest.mark.parametrize("rows", [24, 300])
def test_float32_small_results(rows):
  """Tiny times ordinary: results about and below float32's least normal number, in the output and both gradients."""
  for scale in (1e-36, 1e-38, 1e-40):
    x, w, g = _normal((rows, 72), 1, scale), _normal((65, 72), 2, 0.1), _normal((rows, 65), 3, scale)
    lx, lw = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = fwn.linear_act(lx, lw)
    xd, wd, gd = x.double(), w.double(), g.double()
    # A product below the least normal number is held to 2^-150 by its own rounding: 72 (or 65) of them a sum.
    floor = 100 * 2.0 ** -150
    _near(out.detach(), xd @ wd.t(), _bound(72, xd, wd) + floor)
    gx, = torch.autograd.grad(out, lx, g, retain_graph=True)
    _near(gx, gd @ wd, _bound(65, gd, wd.t()) + floor)
    gw, = torch.autograd.grad(out, lw, _normal((rows, 65), 4))
    gd = _normal((rows, 65), 4).double()
    _near(gw, gd.t() @ xd, _bound(rows, gd.t(), xd.t()) + rows * 2.0 ** -150)


@gpu
@pytest.mark.parametrize("rows", [24, 300])
def test_float32_large_results(rows):
  """Sums up to float32's largest, split over ranges too (ins 4,096); past it they are infinite."""
  for ins in (64, 4096):
    x, w = _normal((rows, ins), 1, 1e19), _normal((72, ins), 2, 1e19 / ins ** 0.5 / 10)
    xd, wd = x.double(), w.double()
    _near(fwn.linear_act(x, w), xd @ wd.t(), _bound(ins, xd, wd))
  x, w = torch.full((rows, 64), 1e20, device=DEV), torch.full((72, 64), 1e20, device=DEV)
  w[3] = -1e20
  w[4] = 0
  out = fwn.linear_act(x, w)
  assert (out[:, 3] == -float("inf")).all() and not out[:, 4].any()
  assert (out[:, 5:] == float("inf")).all() and (out[:, :3] == float("inf")).all()


def _points():
  z = torch.cat([torch.linspace(-20, 20, 4001), torch.logspace(-6, 0, 400), -torch.logspace(-6, 0, 400),
                 torch.logspace(-37, -6, 100), torch.linspace(-110, 110, 441)])
  return z.float().to(DEV)


def _act64(z, name):
  """act, act' and p with act = z p. gelu_tanh by p = 1 / (1 + e^-2u): z (1 + tanh(u)) / 2 is off by |z| 2^-54
  in float64 where tanh nears -1, 4e-16 at z = -7.2, where its value is 2e-16."""
  z = z.double().requires_grad_()
  phi = {"gelu": torch.special.ndtr, "silu": torch.sigmoid,
         "gelu_tanh": lambda t: torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (t + 0.044715 * t ** 3))}[name]
  a = torch.nn.functional.gelu(z) if name == "gelu" else z * phi(z)
  return a.detach(), torch.autograd.grad(a.sum(), z)[0], phi(z.detach())


@gpu
@pytest.mark.parametrize("rows", [32, 500])
def test_the_lower_tail_of_gelu(rows):
  """z (1 + erf) / 2 of negative z, relative to itself. float32: the argument's two roundings change erfc by z^2 of
  each, erfc is within four steps and two products round. bf16: the output rounds by 2^-8, and the
  approximation of erfc is within 0.4% down to z = -6."""
  exact = lambda z: z.double() * 0.5 * torch.special.erfc(-z.double() * 0.5 ** 0.5)
  z = torch.linspace(-9, -1, rows, device=DEV)[:, None]
  one = torch.ones(1, 1, device=DEV)
  want = exact(z)
  got = fwn.linear_act(z, one, activation="gelu").double()
  assert ((got - want).abs() <= (10 + 2 * z.double() ** 2) * STEP * want.abs()).all()
  z = torch.linspace(-6, -1, rows, device=DEV)[:, None].bfloat16()
  want = exact(z)
  got = fwn.linear_act(z, one.bfloat16(), activation="gelu").double()
  assert ((got - want).abs() <= (2.0 ** -8 + 4e-3) * want.abs()).all()


@gpu
@pytest.mark.parametrize("name", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("outs", [1, 8])
@pytest.mark.parametrize("rows", [32, 5342])
def test_float32_activations(name, rows, outs):
  """act and act' of float32 pre-activations that are exact (a weight of one). Half steps that each may take:

  gelu: erf is within two steps of its value below 1 (4 of 2^-24), its sum with 1 rounds below 2 by 2^-24: half of
  five, 2.5, of z; two products round the value. The slope adds the density's exponent, z^2 / 2 rounded twice.
  silu and gelu_tanh: z p, p = 1 / (1 + e^-u): e within two steps, the sum a half step, the reciprocal one step
  and the product a half: 8 of the value, and (1 - p) times the exponent's own roundings (none of silu's -z;
  four of gelu_tanh's u, which grow with u). Where p is below the least normal number it has steps of 2^-149, a few
  of them, times what it is multiplied by."""
  z = _points()
  if rows == 32:
    z = z[torch.randperm(z.numel(), generator=torch.Generator().manual_seed(1))[:32].to(DEV)]
  one, g = torch.ones(outs, 1, device=DEV), torch.zeros(rows, outs, device=DEV)
  g[:, 0] = 1
  leaf = z[:, None].contiguous().requires_grad_()
  out = fwn.linear_act(leaf, one, activation=name)
  want, slope, p = _act64(z, name)
  y, u = z.double().abs(), 2 * (2 / torch.pi) ** 0.5 * (z.double() + 0.044715 * z.double() ** 3).abs()
  if name == "gelu":
    bound = 2.5 * y + 2 * want.abs()
  else:
    bound = want.abs() * (8 + (4 * u * (1 - p) if name == "gelu_tanh" else 0))
  over = (out[:, 0].double() - want).abs() - bound * STEP - (1 + y) * 2.0 ** -147
  assert over.max() <= 0, (name, z[over.argmax()].item())
  gx, = torch.autograd.grad(out, leaf, g)
  if name == "gelu":
    density = y * torch.exp(-0.5 * y * y) * (0.5 / torch.pi) ** 0.5
    bound = 2.5 + density * (8 + 2 * y * y) + 2 * slope.abs()
  elif name == "silu":
    # p (1 + z (1 - p)): p's 8 in each place, and the difference 1 - p rounds by 2^-24 of 1.
    bound = p * (8 * (1 + y * (1 - p)) + y * (1 + 8 * p) + 4 * (1 + y))
  else:
    c = 2 * y * p * (1 - p) * (2 / torch.pi) ** 0.5 * (1 + 3 * 0.044715 * y * y)
    e = 8 + 4 * u * (1 - p)
    bound = p * e + c * (2 * e + 8) + 2 * y * p * (1 + e * p) * (2 / torch.pi) ** 0.5 * (1 + 3 * 0.044715 * y * y)
  over = (gx[:, 0].double() - slope).abs() - bound * STEP - (1 + 2 * y * (1 + 0.134145 * y * y)) * 2.0 ** -147
  assert over.max() <= 0, (name, z[over.argmax()].item(), over.max().item() / STEP)
