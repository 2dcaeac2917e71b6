"""4-bit weights with group scales (``linear_q4.py``, ``fwn_quantize_q4_launch``, ``fwn_linear_act_q4_*``) against float64.

A widened weight is exact in bfloat16 and float32, so the products with bfloat16 x are exact and their float32 sum of k is off by
at most (8 sqrt(k) + 16) 2^-24 |a| |b| (norms of the two rows; 2 / 3 sqrt(k) 2^-24 of them for the roundings of partial sums, twelve
times that, and 16 for the epilogue); float32 products are rounded once each, which the same bound holds."""
import ctypes

import pytest
import torch

import faster_weathernext_amd as fwn
from faster_weathernext_amd import _native as nat

DEV = "cuda"
gpu = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float32]
CODES, SCALES = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
SIZES = [(1, 1, 1), (1, 64, 64), (1, 768, 1000), (2, 7, 9), (3, 513, 65), (7, 4096, 512), (16, 256, 16), (17, 100, 33),
         (24, 1032, 136), (31, 8, 260), (32, 32, 32), (1, 5120, 4112), (20, 2051, 4099), (33, 96, 31), (63, 64, 129), (64, 128, 64),
         (65, 72, 250), (100, 515, 1027), (128, 64, 256), (129, 192, 257), (257, 320, 511), (513, 40, 770), (1000, 1024, 130),
         (300, 3, 4000), (40, 5000, 8), (2562, 515, 129), (5, 20000, 3)]


def _gen(seed):
  return torch.Generator().manual_seed(seed)


def _normal(shape, dtype, seed, std=1.0):
  return (torch.randn(shape, generator=_gen(seed)) * std).to(dtype).to(DEV)


def _half(dtype):
  return torch.finfo(dtype).eps / 2


def _powers(e):
  """2^(e - 127) exactly, which the middles of two codes need and the GPU's exp2 and pow do not give."""
  return torch.tensor([2.0 ** (k - 127) for k in range(256)], dtype=torch.float64, device=e.device)[e.long()]


def _values(codes, scales, ins):
  """The weight in float64; infinite where it has no place in float32."""
  table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=codes.device)
  c, e = codes.view(torch.uint8).long(), scales.view(torch.uint8)
  v = torch.cat((table, -table))[torch.stack((c & 15, c >> 4), -1).view(*e.shape, 32)]
  v = v * _powers(e)[..., None]
  v = torch.where((e == 255)[..., None], float("nan"), v)
  v = torch.where(v.abs() >= 2.0 ** 128, v * float("inf"), v)
  return v.reshape(e.shape[0], -1)[:, :ins]


def _random_codes(outs, ins, seed, low=120, high=128):
  groups = -(-ins // 32)
  codes = torch.randint(0, 256, (outs, 16 * groups), generator=_gen(seed), dtype=torch.uint8)
  scales = torch.randint(low, high, (outs, groups), generator=_gen(seed + 1), dtype=torch.uint8)
  return codes.to(DEV).view(CODES), scales.to(DEV).view(SCALES)


def _act64(z, name):
  return {None: lambda t: t, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu,
          "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[name](z)


# ---- quantisation


def _quantized64(w):
  """(codes, scales) by the definition, from float64 rows on the host."""
  outs, ins = w.shape
  groups = -(-ins // 32)
  w = torch.nn.functional.pad(w, (0, 32 * groups - ins)).view(outs, groups, 32)
  top = w.abs().amax(-1)
  bad = ~w.isfinite().all(-1)
  e = torch.zeros(outs, groups, dtype=torch.long)
  for k in range(254):  # the least power of two that holds it
    e = torch.where((top > 7 * _powers(e)) & ~bad, k + 1, e)
  v = torch.where(bad[..., None], 0.0, w) / _powers(e)[..., None]
  table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
  off = (v.abs()[..., None] - table).abs()
  best = off.amin(-1, keepdim=True)
  at = off == best
  even = at[..., 0::2].any(-1)  # of two as near the even code
  first = at.float().argmax(-1)
  first = torch.where((at.sum(-1) == 2) & even & (first % 2 == 1), first + 1, first)
  # Sign bits as they are, those of zeros too.
  sign = (w.signbit() & ~bad[..., None]).long()
  codes = (first | sign << 3) * (~bad[..., None]).long()
  codes = codes.view(outs, -1)
  return (codes[:, 0::2] | codes[:, 1::2] << 4).to(torch.uint8), torch.where(bad, 255, e).to(torch.uint8)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("outs,ins", [(1, 1), (3, 31), (5, 32), (7, 33), (65, 515), (1000, 768), (2, 20000)])
def test_quantization(outs, ins, dtype):
  w = _normal((outs, ins), dtype, outs)
  w *= _powers(torch.randint(97, 157, (outs, 1), generator=_gen(1))).to(dtype).to(DEV)
  codes, scales = fwn.quantize_q4(w)
  assert codes.dtype == CODES and scales.dtype == SCALES and codes.shape == (outs, 16 * -(-ins // 32))
  want = _quantized64(w.double().cpu())
  assert torch.equal(codes.view(torch.uint8).cpu(), want[0]) and torch.equal(scales.view(torch.uint8).cpu(), want[1])
  # Half a step: a quarter of the scale below 2, then a half, one, and up to one where seven is cut to six.
  top = w.double().abs()
  got = _values(codes, scales, ins)
  step = _powers(scales.view(torch.uint8)).repeat_interleave(32, 1)[:, :ins]
  assert ((got - w.double()).abs() <= torch.maximum(top / 5, step / 4)).all()
  # Values of the format stay as they are.
  again = fwn.quantize_q4(got.to(dtype))
  assert torch.equal(_values(*again, ins), got)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantization_of_special_groups(dtype):
  w = torch.zeros(12, 64, dtype=torch.float64)
  w[0, 3], w[1, 40], w[2, 0] = float("nan"), float("inf"), -float("inf")
  w[3, :10] = torch.tensor([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -5])    # middles of two codes
  w[4, :4] = torch.tensor([7, 6.5, -7, 1])                                         # beyond six
  w[5, 0], w[6, 0], w[7, 0] = 7.0625, 2.0 ** -126, 2.0 ** -133                      # subnormal numbers
  w[8, 0], w[9, 0] = 3 * 2.0 ** 126, 2.0 ** -149 if dtype == torch.float32 else 2.0 ** -132
  w[10, 0], w[11] = -0.0, 1e-30
  codes, scales = fwn.quantize_q4(w.to(dtype).to(DEV))
  want = _quantized64(w.to(dtype).double())
  assert torch.equal(codes.view(torch.uint8).cpu(), want[0]) and torch.equal(scales.view(torch.uint8).cpu(), want[1])
  e = scales.view(torch.uint8)
  assert e[0].tolist() == [255, 0] and e[1].tolist() == [0, 255] and e[2, 0] == 255 and e[3, 0] == 127 and e[4, 0] == 127
  assert e[5, 0] == 128 and e[7, 0] == 0


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantization_of_strided_rows(dtype):
  big = _normal((40, 300), dtype, 1)
  for w in (big[:, :100], big[:, 1:101], big[::2, 7:263], big.t(), big[:1].expand(9, 300), big[:, ::3]):
    a, b = fwn.quantize_q4(w), fwn.quantize_q4(w.contiguous())
    assert all(torch.equal(s.view(torch.uint8), t.view(torch.uint8)) for s, t in zip(a, b))


# ---- products


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,ins,outs", SIZES)
def test_whole_numbers(rows, ins, outs, dtype):
  """Sums of halves that float32 holds exactly; codes past ins are not used."""
  codes, scales = _random_codes(outs, ins, 1, 127, 129)
  w = _values(codes, scales, ins)
  whole = lambda shape, seed: torch.randint(-2, 3, shape, generator=_gen(seed)).to(dtype).to(DEV)
  x, b, r = whole((rows, ins), 3), whole((outs,), 4), whole((rows, outs), 5)
  z = x.double() @ w.t()
  assert torch.equal(fwn.linear_act_q4(x, codes, scales), z.to(dtype))
  assert torch.equal(fwn.linear_act_q4(x, codes, scales, b, residual=r), (z + b.double() + r.double()).to(dtype))
  assert torch.equal(fwn.linear_act_q4(x, codes, scales, b, activation="relu"), (z + b.double()).relu().to(dtype))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,ins,outs", SIZES)
@pytest.mark.parametrize("activation", [None, "gelu", "gelu_tanh", "silu"])
def test_normal_numbers(rows, ins, outs, dtype, activation):
  codes, scales = fwn.quantize_q4(_normal((outs, ins), dtype, 1, ins ** -0.5))
  w = _values(codes, scales, ins)
  x, b, r = _normal((rows, ins), dtype, 2), _normal((outs,), dtype, 3), _normal((rows, outs), dtype, 4)
  z = x.double() @ w.t() + b.double()
  e = (8 * ins ** 0.5 + 16) * 2.0 ** -24 * x.double().norm(dim=1)[:, None] * w.norm(dim=1) + 2.0 ** -22 * (z.abs() + b.double().abs())
  a = _act64(z, activation)
  if activation:
    # Slopes up to 1.13; the functions for bf16 are off by a rounding of it, those of float32 by a few of its.
    e = 1.2 * e + (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -20) * a.abs() + 2.0 ** -20 * z.abs()
  got = fwn.linear_act_q4(x, codes, scales, b, activation=activation, residual=r)
  want = a + r.double()
  off = (got.double() - want).abs() - e - _half(dtype) * want.abs() - 2.0 ** -22 * (a.abs() + r.double().abs())
  assert got.dtype == dtype and off.max() <= 0, off.max().item()


@gpu
@pytest.mark.parametrize("rows,ins,outs", [(512, 1100, 8200), (300, 4096, 2056), (33, 8192, 300), (700, 2000, 3000), (32, 16384, 515),
                                           (17, 16384, 4104), (64, 1024, 16384), (2100, 640, 4097), (20, 900, 12800), (3, 700, 12900)])
def test_tiles_and_ranges(rows, ins, outs):
  """Whole numbers over sizes that take tiles of both widths, sums in several ranges, and many outputs a workgroup."""
  codes, scales = _random_codes(outs, ins, 1, 127, 129)
  x = torch.randint(-1, 2, (rows, ins), generator=_gen(3)).bfloat16().to(DEV)
  r = torch.randint(-2, 3, (rows, outs), generator=_gen(5)).bfloat16().to(DEV)
  z = x.double() @ _values(codes, scales, ins).t()  # below 2^18 in steps of a half: exact in float32
  for _ in range(2):
    assert torch.equal(fwn.linear_act_q4(x, codes, scales), z.bfloat16())
    assert torch.equal(fwn.linear_act_q4(x, codes, scales, residual=r), (z + r.double()).bfloat16())


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 20, 40])
def test_every_code_and_scale(rows, dtype):
  """Output o has the scale o and one code: its value, from the least subnormal number to infinity."""
  for code in range(16):
    codes = torch.zeros(256, 16, dtype=torch.uint8, device=DEV)
    codes[:, code] = code if code % 2 else code << 4
    scales = torch.arange(256, dtype=torch.uint8, device=DEV)[:, None]
    w = _values(codes.view(CODES), scales.view(SCALES), 32)
    x = torch.ones(rows, 32, dtype=dtype, device=DEV)
    got = fwn.linear_act_q4(x, codes.view(CODES), scales.view(SCALES))
    want = w.sum(1).to(dtype).expand(rows, 256)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0)), code


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [2, 40])
def test_codes_past_the_inputs_are_not_used(rows, dtype):
  for ins in (1, 5, 33, 100, 515):
    codes, scales = _random_codes(48, ins, 1)
    x = _normal((rows, ins), dtype, 3)
    want = fwn.linear_act_q4(x, codes, scales)
    other = codes.view(torch.uint8).clone()
    flat = torch.stack((other & 15, other >> 4), -1).view(48, -1)
    flat[:, ins:] = 15 - flat[:, ins:]
    other = flat[:, 0::2] | flat[:, 1::2] << 4
    assert torch.equal(fwn.linear_act_q4(x, other.view(CODES), scales), want)


@gpu
@pytest.mark.parametrize("rows", [3, 40])
def test_values_that_are_not_finite(rows):
  for dtype in DTYPES:
    codes, scales = _random_codes(40, 128, 1)
    x = _normal((rows, 128), dtype, 2)
    clean = fwn.linear_act_q4(x, codes, scales)
    x[1, 5] = float("nan")
    e = scales.view(torch.uint8).clone()
    e[7, 2] = 255
    out = fwn.linear_act_q4(x, codes, e.view(SCALES))
    assert out[1].isnan().all() and out[:, 7].isnan().all()
    keep = torch.ones_like(out, dtype=torch.bool)
    keep[1], keep[:, 7] = False, False
    assert torch.equal(out[keep], clean[keep])


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(dtype):
  big, res = _normal((99, 400), dtype, 1), _normal((99, 200), dtype, 2)
  codes, scales = _random_codes(260, 264, 3)
  w, e, b = codes[100:164], scales[100:164], _normal((300,), dtype, 4)[1:65]
  shifted = torch.empty(64 * codes.shape[1] + 1, dtype=torch.uint8, device=DEV)[1:].view(64, -1)
  shifted.copy_(w.contiguous().view(torch.uint8))
  wide = torch.zeros(64, 300, dtype=torch.uint8, device=DEV)
  wide[:, 3:3 + codes.shape[1]], wide[:, 200:200 + scales.shape[1]] = w.view(torch.uint8), e.view(torch.uint8)
  others = [(w, e), (shifted.view(CODES), e),
            (wide[:, 3:3 + codes.shape[1]].view(CODES), wide[:, 200:200 + scales.shape[1]].view(SCALES))]
  for rows in (5, 33, 99):
    for x in (big[:rows, :264], big[:rows, 1:265], big[:rows, 8:272], big[:1, :264].expand(rows, 264), big.t()[:264, :rows].t()):
      for r in (res[:rows, :64], res[:rows, 3:67], res[:1, :64].expand(rows, 64)):
        want = fwn.linear_act_q4(x.contiguous(), w, e, b, residual=r.contiguous())
        for weight, scale in others:
          assert torch.equal(fwn.linear_act_q4(x, weight, scale, b, residual=r), want)
  x = big[:6, :264]
  assert torch.equal(fwn.linear_act_q4(x.reshape(2, 3, 264), w, e).view(6, 64), fwn.linear_act_q4(x, w, e))
  assert torch.equal(fwn.linear_act_q4(x[0], w, e), fwn.linear_act_q4(x[:1], w, e)[0])


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_do_not_depend_on_each_other(dtype):
  """A row's result is the same among 1 to 16 others, and the same call gives the same bits."""
  codes, scales = _random_codes(520, 1000, 1)
  x = _normal((16, 1000), dtype, 2)
  all_rows = fwn.linear_act_q4(x, codes, scales)
  for rows in (1, 2, 7, 16):
    assert torch.equal(fwn.linear_act_q4(x[:rows], codes, scales), all_rows[:rows])
  x = _normal((700, 1000), dtype, 3)
  assert torch.equal(fwn.linear_act_q4(x, codes, scales), fwn.linear_act_q4(x, codes, scales))


@gpu
def test_empty():
  codes, scales = _random_codes(8, 64, 1)
  assert fwn.linear_act_q4(torch.zeros(2, 0, 64, device=DEV), codes, scales).shape == (2, 0, 8)


@gpu
@pytest.mark.parametrize("rows", [4, 50])
def test_side_stream_and_graph(rows):
  codes, scales = _random_codes(520, 300, 1)
  x = _normal((rows, 300), torch.bfloat16, 2)
  step = lambda: fwn.linear_act_q4(x, codes, scales, activation="silu")
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    first = step()
  torch.cuda.current_stream().wait_stream(side)
  assert torch.equal(first, step())
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph, stream=side):
    held = step()
  for k in range(4):
    x.copy_(_normal((rows, 300), torch.bfloat16, 20 + k))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, step()), k


@gpu
def test_a_block_in_4_bits():
  """A feed-forward between sandwich norms, as it is served: against the same block with the widened weights."""
  d, h = 256, 1000
  for rows in (1, 24, 300):
    x, y = _normal((rows, d), torch.float32, 1), _normal((rows, d), torch.float32, 2)
    post, pre = (1 + 0.1 * _normal((d,), torch.float32, k) for k in (3, 4))
    up, down = fwn.quantize_q4(_normal((h, d), torch.float32, 5, d ** -0.5)), fwn.quantize_q4(_normal((d, h), torch.float32, 6, h ** -0.5))
    b = _normal((h,), torch.float32, 7)
    s, n = fwn.sandwich_norm(x, y, post, pre, gate=post)
    f = fwn.linear_act_q4(fwn.linear_act_q4(n, *up, b, activation="gelu_tanh"), *down)
    s, n = fwn.sandwich_norm(s, f, post, pre, scale=0.5)
    norm = lambda t: t * (t.square().mean(-1, keepdim=True) + 1e-6) ** -0.5
    wide = lambda t: t.double()
    s64 = wide(x) + norm(wide(y)) * wide(post) ** 2
    z = norm(s64) * wide(pre) @ _values(*up, d).t() + wide(b)
    f64 = _act64(z, "gelu_tanh") @ _values(*down, h).t()
    s64 = 0.5 * s64 + norm(f64) * wide(post)
    # float32 throughout: each of the six steps within 2^-16 of the values' size.
    assert (s.double() - s64).norm() <= 6 * 2.0 ** -16 * s64.norm()
    assert (n.double() - norm(s64) * wide(pre)).norm() <= 6 * 2.0 ** -16 * n.double().norm()


@gpu
def test_refusals():
  codes, scales = _random_codes(8, 64, 1)
  x = torch.zeros(2, 64, device=DEV)
  f = fwn.linear_act_q4
  for call in (lambda: f(x.cpu(), codes, scales), lambda: f(x, codes.cpu(), scales), lambda: f(x, codes, scales.cpu()),
               lambda: f(x[:, :32], codes, scales), lambda: f(x, codes[:4], scales), lambda: f(x, codes, scales[:, :1]),
               lambda: f(x, codes[0], scales), lambda: f(x, codes, scales, torch.zeros(7, device=DEV)),
               lambda: f(x, codes, scales, residual=torch.zeros(8, device=DEV)), lambda: f(x, codes, scales, activation="tanh"),
               lambda: f(torch.zeros((), device=DEV), codes, scales), lambda: fwn.quantize_q4(torch.zeros(2, 64)),
               lambda: fwn.quantize_q4(x[0]), lambda: fwn.quantize_q4(x[:, :0]), lambda: fwn.quantize_q4(x[:0])):
    with pytest.raises(ValueError):
      call()
  for call in (lambda: f(x.half(), codes, scales), lambda: f(x, codes.view(torch.uint8), scales),
               lambda: f(x, codes, scales.view(torch.uint8)), lambda: f(x, codes, scales, torch.zeros(8, device=DEV).bfloat16()),
               lambda: fwn.quantize_q4(x.double())):
    with pytest.raises(TypeError):
      call()
  leaf = x.clone().requires_grad_()
  for call in (lambda: f(leaf, codes, scales), lambda: fwn.quantize_q4(leaf),
               lambda: f(x, codes, scales, residual=torch.zeros(2, 8, device=DEV, requires_grad=True))):
    with pytest.raises(RuntimeError, match="no derivative"):
      call()
  with torch.no_grad():
    assert f(leaf, codes, scales).shape == (2, 8)


# ---- host validation of the C ABI: no GPU calls

F = 65536  # an address that is only compared


def _desc(rows=4, ins=64, outs=32, x_stride=64, r_stride=32, dtype=nat.BF16, activation=0):
  return nat.LinearDesc(rows, x_stride, 0, r_stride, ins, outs, dtype, activation)


@pytest.mark.parametrize("bad,code", [(dict(rows=-1), 1), (dict(ins=0), 1), (dict(outs=(1 << 20) + 1), 1), (dict(x_stride=-1), 1),
                                      (dict(x_stride=(1 << 30) + 1), 1), (dict(r_stride=(1 << 20) + 1), 1), (dict(dtype=2), 2),
                                      (dict(activation=9), 2), (dict(rows=1 << 31, ins=1 << 20), 1)])
def test_bad_descriptors(bad, code):
  L, d, size = nat.lib(), _desc(**bad), ctypes.c_uint64()
  assert L.fwn_linear_act_q4_workspace_size(d, F, 3 * F, ctypes.byref(size)) == code
  assert L.fwn_linear_act_q4_launch(d, F, 2 * F, 3 * F, None, None, 4 * F, 8 * F, 1 << 30, None) == code


def test_bad_pointers():
  L, d = nat.lib(), _desc()
  good = [F, 2 * F, 3 * F, 4 * F, 5 * F, 6 * F]  # x codes scales bias residual out
  for at, value in ((0, None), (1, None), (2, None), (5, None), (0, F + 1), (1, 2 * F + 8), (3, 4 * F + 1), (4, 5 * F + 1), (5, 6 * F + 1),
                    (5, F + 64), (5, 2 * F), (5, 3 * F), (5, 4 * F), (5, 5 * F)):
    args = list(good)
    args[at] = value
    assert L.fwn_linear_act_q4_launch(d, *args, None, 0, None) == nat.ERR_INVALID_ARG, (at, value)
  d, size = _desc(rows=40), ctypes.c_uint64()
  assert L.fwn_linear_act_q4_workspace_size(d, F, 3 * F, ctypes.byref(size)) == nat.OK and size.value >= 32 * 16
  for work, n in ((None, 0), (8 * F, 16), (8 * F + 16, 1 << 20), (F, 1 << 20), (6 * F, 1 << 20)):
    assert L.fwn_linear_act_q4_launch(d, *good, work, n, None) == nat.ERR_INVALID_ARG
  assert L.fwn_linear_act_q4_launch(_desc(rows=0), *[None] * 7, 0, None) == nat.OK
  q = L.fwn_quantize_q4_launch
  for args in ((-1, 64, 64, 0, F, 2 * F, 3 * F), (4, 0, 64, 0, F, 2 * F, 3 * F), (4, 64, -1, 0, F, 2 * F, 3 * F),
               (4, 64, 64, 0, None, 2 * F, 3 * F), (4, 64, 64, 0, F, None, 3 * F), (4, 64, 64, 0, F, 2 * F, None),
               (4, 64, 64, 0, F, 2 * F + 8, 3 * F), (4, 64, 64, 0, F, F, 3 * F), (4, 64, 64, 0, F, 2 * F, 2 * F),
               (4, 64, 64, 1, F + 1, 2 * F, 3 * F), ((1 << 20) + 1, 64, 64, 0, F, 2 * F, 3 * F)):
    assert q(*args, None) == nat.ERR_INVALID_ARG, args
  assert q(4, 64, 64, 7, F, 2 * F, 3 * F, None) == nat.ERR_UNSUPPORTED
  assert q(0, 64, 64, 0, None, None, None, None) == nat.OK


def test_needs_a_gpu_tensor():
  with pytest.raises(ValueError, match="CUDA"):
    fwn.linear_act_q4(torch.zeros(2, 64), torch.zeros(8, 32, dtype=torch.uint8).view(CODES),
                      torch.zeros(8, 2, dtype=torch.uint8).view(SCALES))
  with pytest.raises(ValueError, match="CUDA"):
    fwn.quantize_q4(torch.zeros(2, 64))
