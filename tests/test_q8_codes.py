"""The codes of ``rms_norm_q8``, ``add_rms_norm_q8`` and ``quantize_rows``: of v * (1 / scale), the reciprocal and the
product each rounded to float32, to the nearest e4m3 value, ties to even. The two roundings are 2^-24 of
the quotient each, so a code is the nearest to v / scale but for quotients that close to the middle of
two codes, which bf16 rows often are: there either neighbour is as near."""
import pytest
import torch

import faster_weathernext_amd as fwn

DEV = "cuda"
gpu = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def _rows(shape, dtype, seed):
  return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _codes(v):
  """(codes, scale) of float32 rows v on the CPU."""
  scale = (v.abs().amax(-1) / 448).clamp(min=2.0 ** -126)
  return (v * (1 / scale)[..., None]).to(E4M3), scale


def _check(q, scale, v):
  codes, want = _codes(v)
  assert torch.equal(scale.cpu(), want) and torch.equal(q.cpu().view(torch.uint8), codes.view(torch.uint8))
  quotient, near = v.double() / want.double()[..., None], q.cpu().double()
  # The spacing of e4m3 about the quotient: 2^-3 of its power of two, 2^-9 below 2^-6.
  step = (2.0 ** (torch.floor(torch.log2(quotient.abs().clamp(min=2.0 ** -6))) - 3))
  assert ((quotient - near).abs() <= step / 2 + 2.0 ** -22 * quotient.abs()).all()
  return ((quotient - near).abs() >= step / 2 - 2.0 ** -22 * quotient.abs()).sum().item()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("channels", [64, 1024, 4096])
def test_codes(channels, dtype):
  """Rows of +1 and -1 have a mean square of exactly 1, so that their norm is the weight with their signs."""
  sign = _rows((40, channels), torch.float32, 1).sign().to(dtype)
  middles = 0
  for seed in range(8):
    w = _rows((channels,), dtype, 10 + seed)
    v = sign.float() * w.float()
    middles += _check(*fwn.rms_norm_q8(sign.to(DEV), w.to(DEV), eps=0.0), v)
    zero = torch.zeros_like(sign)
    s, q, scale = fwn.add_rms_norm_q8(sign.to(DEV), zero.to(DEV), w.to(DEV), eps=0.0)
    assert torch.equal(s.cpu(), sign)
    _check(q, scale, v)
    x = _rows((40, channels), dtype, 30 + seed)
    middles += _check(*fwn.quantize_rows(x.to(DEV)), x.float())
  assert dtype == torch.float32 or channels == 64 or middles > 0  # the middles of two codes were among them
