"""``linear_act`` at values where a product, a scale or an activation can lose float32's precision, against float64."""
import pytest
import torch

import faster_weathernext_amd as fwn

DEV = "cuda"
gpu = pytest.mark.gpu
STEP = 2.0 ** -24  # half a step of float32


def _normal(shape, seed, std=1.0):
  return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(DEV)


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
