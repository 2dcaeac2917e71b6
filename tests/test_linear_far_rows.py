"""Rows more elements apart than the launches take: whole numbers, to the bit."""
import pytest
import torch

import faster_weathernext_amd as fwn

DEV = "cuda"
FAR = (1 << 30) + 64


def _far(rows, cols, dtype, seed):
  """[rows, cols] of small whole numbers, FAR elements apart; what lies between is never read."""
  buf = torch.empty((rows - 1) * FAR + cols, dtype=dtype, device=DEV)
  t = buf.as_strided((rows, cols), (FAR, 1))
  t.copy_(torch.randint(-2, 3, (rows, cols), generator=torch.Generator().manual_seed(seed)).to(dtype))
  return t


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2])
def test_linear_act(rows):
  x, w, r = _far(2, 40, torch.bfloat16, 1)[:rows], _far(2, 40, torch.bfloat16, 2), _far(2, 2, torch.bfloat16, 3)[:rows]
  lx, lw = x.detach().requires_grad_(), w.detach().requires_grad_()
  out = fwn.linear_act(lx, lw, residual=r)
  assert torch.equal(out, (x.double() @ w.double().t() + r.double()).bfloat16())
  g = torch.ones_like(out)
  gx, gw = torch.autograd.grad(out, (lx, lw), g)
  assert torch.equal(gx, (g.double() @ w.double()).bfloat16()) and torch.equal(gw, (g.double().t() @ x.double()).bfloat16())


@pytest.mark.gpu
def test_8_bits_and_norms():
  x = _far(2, 48, torch.float8_e4m3fn, 1)
  one = torch.ones(2, device=DEV)
  want = x.float().double() @ x.float().double().t()
  assert torch.equal(fwn.linear_act_q8(x, one, x, one, dtype=torch.float32).double(), want)
  x = _far(2, 48, torch.bfloat16, 2)
  for a, b in zip((fwn.rms_norm(x), *fwn.add_rms_norm(x, x), *fwn.quantize_rows(x)),
                  (fwn.rms_norm(x.contiguous()), *fwn.add_rms_norm(x.contiguous(), x.contiguous()),
                   *fwn.quantize_rows(x.contiguous()))):
    assert torch.equal(a.float(), b.float())
