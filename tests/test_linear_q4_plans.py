"""How 4-bit linear layers of bfloat16 rows are formed: each way that the plan takes, at sizes that it sends there, against whole
numbers in float64. The plan is an estimate from measured times: the host's part of the library is compiled into a program that
prints it, so that another estimate does not leave a way untested unseen.

Whole numbers: x is -1, 0 or 1 and a weight at most 12 in halves, so that sums of 16,384 stay below 2^18 in steps of a half, which
float32 holds in any order of adding. Normal numbers: the bound of the sums in ``test_linear_q4.py``, the same for any order."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

import faster_weathernext_amd as fwn
from faster_weathernext_amd import _native as nat
from test_linear_q4 import _gen, _half, _normal, _random_codes, _values

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "faster-weathernext_amd")
DEV = "cuda"
gpu = pytest.mark.gpu
ROWS, WIDENED, TWO, FOUR = -1, 0, 2, 4  # few rows; a widened weight; tiles of 64 x 128 and of 64 x 256 outputs

# (rows, ins, outs): the way, and whether the sum is split. Last ranges that are shorter, inputs that are not whole 128s, groups that are
# not whole fours, outputs that are not whole eights or tiles, rows that are copied.
PLANS = {
    (24, 5120, 8192): (ROWS, False), (32, 16384, 515): (ROWS, False), (24, 15000, 4097): (ROWS, False),
    (32, 16384, 4096): (FOUR, True), (24, 16384, 8192): (FOUR, True), (17, 16384, 4096): (FOUR, True),
    (20, 16300, 4096): (FOUR, True), (33, 4096, 5120): (FOUR, True), (33, 5000, 5120): (FOUR, True),
    (100, 5000, 4100): (FOUR, True), (200, 3333, 5120): (FOUR, True), (513, 10000, 1000): (FOUR, True),
    (20, 16384, 2048): (TWO, True), (300, 4096, 2056): (TWO, True), (128, 4096, 4096): (TWO, True), (64, 5120, 8192): (TWO, True),
    (512, 1100, 8200): (FOUR, False), (700, 2000, 3000): (FOUR, False), (64, 1024, 16384): (TWO, False), (100, 515, 1027): (TWO, False),
    (33, 8192, 300): (WIDENED, False), (2100, 640, 4097): (WIDENED, False),
}
SPLIT = [s for s, (way, split) in PLANS.items() if split]

PROGRAM = """
#include "%s"
#include <cstdio>
int main() {
  long m, k, n;
  while (std::scanf("%%ld %%ld %%ld", &m, &k, &n) == 3) {
    const auto p = fwn::plan_q4(m, n, k);
    std::printf("%%d %%d %%d\\n", p.tile, p.splits, p.chunk);
  }
}
"""


def test_plans(tmp_path):
  """The ways are those of PLANS, and every range of a split sum has inputs."""
  sys.path.insert(0, PKG)
  try:
    import build
  finally:
    sys.path.remove(PKG)
  source, program = tmp_path / "plan.cpp", tmp_path / "plan"
  source.write_text(PROGRAM % os.path.join(PKG, "csrc", "linear_act_api.cpp"))
  # No launch is called: what the kernels' files define stays unresolved.
  subprocess.run(["g++", "-O0", "-std=c++17", "-ffunction-sections", "-I", build.INCLUDE, "-I", os.path.join(build.ROCM, "include"),
                  "-D__HIP_PLATFORM_AMD__", "-Wl,--gc-sections", "-Wl,--unresolved-symbols=ignore-all", str(source), "-o", str(program)],
                 check=True, timeout=300)
  text = "".join("%d %d %d\n" % s for s in PLANS)
  lines = subprocess.run([str(program)], input=text, capture_output=True, text=True, check=True, timeout=60).stdout.split("\n")
  got = {s: tuple(map(int, line.split())) for s, line in zip(PLANS, lines)}
  assert {s: (way, splits > 1) for s, (way, splits, _) in got.items()} == PLANS
  spans = lambda s: -(-s[1] // 128)
  assert all((got[s][1] - 1) * got[s][2] < spans(s) <= got[s][1] * got[s][2] for s in SPLIT)
  assert any(spans(s) % got[s][2] for s in SPLIT)


def test_workspaces():
  """A split sum's partial products are what its workspace holds, and a way without them and without copies needs none."""
  size = ctypes.c_uint64()
  for (rows, ins, outs), (way, split) in PLANS.items():
    d = nat.LinearDesc(rows, ins, 0, 0, ins, outs, nat.BF16, 0)
    assert nat.lib().fwn_linear_act_q4_workspace_size(d, 4096, 4096, ctypes.byref(size)) == nat.OK
    if split:
      assert size.value >= 2 * rows * outs * 4
    if way == WIDENED:
      assert size.value >= outs * 2 * ins
    if not split and way != WIDENED and ins % 8 == 0 and -(-ins // 32) % 4 == 0:
      assert size.value == 0


def _whole(rows, ins, outs):
  codes, scales = _random_codes(outs, ins, 1, 127, 129)
  draw = lambda shape, seed, n: torch.randint(-n, n + 1, shape, generator=_gen(seed)).bfloat16().to(DEV)
  return codes, scales, draw((rows, ins), 3, 1), draw((outs,), 4, 2), draw((rows, outs), 5, 2)


@gpu
@pytest.mark.parametrize("rows,ins,outs", PLANS)
def test_whole_numbers(rows, ins, outs):
  codes, scales, x, b, r = _whole(rows, ins, outs)
  z = x.double() @ _values(codes, scales, ins).t()
  for _ in range(2):
    assert torch.equal(fwn.linear_act_q4(x, codes, scales), z.bfloat16())
  assert torch.equal(fwn.linear_act_q4(x, codes, scales, b, residual=r), (z + b.double() + r.double()).bfloat16())
  assert torch.equal(fwn.linear_act_q4(x, codes, scales, b, activation="relu"), (z + b.double()).relu().bfloat16())


@gpu
@pytest.mark.parametrize("rows,ins,outs", SPLIT)
def test_normal_numbers(rows, ins, outs):
  codes, scales = fwn.quantize_q4(_normal((outs, ins), torch.bfloat16, 1, ins ** -0.5))
  w = _values(codes, scales, ins)
  x, b, r = (_normal(s, torch.bfloat16, k) for k, s in enumerate(((rows, ins), (outs,), (rows, outs)), 2))
  z = x.double() @ w.t() + b.double()
  e = (8 * ins ** 0.5 + 16) * 2.0 ** -24 * x.double().norm(dim=1)[:, None] * w.norm(dim=1) + 2.0 ** -22 * (z.abs() + b.double().abs())
  got = fwn.linear_act_q4(x, codes, scales, b, residual=r)
  want = z + r.double()
  off = (got.double() - want).abs() - e - _half(torch.bfloat16) * want.abs() - 2.0 ** -22 * (z.abs() + r.double().abs())
  assert off.max() <= 0, off.max().item()
  assert torch.equal(got, fwn.linear_act_q4(x, codes, scales, b, residual=r))


@gpu
@pytest.mark.parametrize("rows,ins,outs", [(32, 16384, 4096), (20, 16300, 4096), (33, 5000, 5120), (100, 5000, 4100), (20, 16384, 2048),
                                           (300, 4096, 2056), (100, 515, 1027)])
def test_nothing_beside_the_outputs(rows, ins, outs):
  """The library's call with its output and workspace inside larger ones: what lies around them stays as it was."""
  codes, scales, x, _, _ = _whole(rows, ins, outs)
  d, size = nat.LinearDesc(rows, ins, 0, 0, ins, outs, nat.BF16, 0), ctypes.c_uint64()
  nat.check(nat.lib().fwn_linear_act_q4_workspace_size(d, x.data_ptr(), scales.data_ptr(), ctypes.byref(size)))
  n, around, edge = rows * outs, 64 * outs, 4096
  out = torch.full((n + 2 * around,), 77.0, dtype=torch.bfloat16, device=DEV)
  work = torch.full((size.value + 2 * edge,), 99, dtype=torch.uint8, device=DEV)
  nat.check(nat.lib().fwn_linear_act_q4_launch(d, x.data_ptr(), codes.data_ptr(), scales.data_ptr(), None, None,
                                               out.data_ptr() + 2 * around, work.data_ptr() + edge, size.value,
                                               torch.cuda.current_stream().cuda_stream))
  assert torch.equal(out[around:around + n].view(rows, outs), (x.double() @ _values(codes, scales, ins).t()).bfloat16())
  assert (out[:around] == 77).all() and (out[around + n:] == 77).all()
  assert (work[:edge] == 99).all() and (work[edge + size.value:] == 99).all()
