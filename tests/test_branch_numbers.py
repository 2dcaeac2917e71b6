"""``p``, ``scale`` and ``eps`` of dropout and of the norms around a block are numbers: a tensor there would get no gradient, and
one on the GPU would be waited for. Nothing is launched."""
import importlib

import numpy as np
import pytest
import torch

import faster_weathernext_amd as fwn

TENSORS = [torch.tensor(0.5), torch.full((1,), 0.5), torch.nn.Parameter(torch.tensor(0.5)), torch.tensor(0.5, dtype=torch.float64)]


@pytest.fixture
def norms(monkeypatch):
  """sandwich_norm for tensors on the host; gives the descriptors of its launches."""
  module = importlib.import_module("faster_weathernext_amd.sandwich")
  seen = []
  monkeypatch.setattr(module, "_check", lambda *args: None)
  monkeypatch.setattr(module, "launch", lambda t, fn, d, *args: seen.append(d))
  x = torch.zeros(2, 64)
  def call(**args):
    module.sandwich_norm(x, x, **args)
    return seen.pop()
  return call


@pytest.mark.parametrize("value", TENSORS)
def test_norms_refuse_tensors(norms, value):
  for name in ("scale", "eps", "p"):
    with pytest.raises(TypeError, match=f"{name} must be a number"):
      norms(**{name: value}, rng=(1, 2))


def test_norms_take_numbers(norms):
  for value in (0.5, np.float32(0.5), np.float64(0.5)):
    d = norms(scale=value, eps=value, p=value, rng=(1, 2))
    assert (d.scale, d.eps, d.drop.p) == (0.5, 0.5, 0.5)
  assert norms(scale=-2).scale == -2.0 and norms(p=1, rng=(1, 2)).drop.p == 1.0


@pytest.mark.parametrize("value", TENSORS)
def test_dropout_refuses_tensors(value):
  dropout = importlib.import_module("faster_weathernext_amd.dropout")
  with pytest.raises(TypeError, match="p must be a number"):
    dropout.check_p(value)


@pytest.mark.gpu
def test_the_calls():
  x = torch.zeros(2, 64, device="cuda")
  for value in (*TENSORS, torch.tensor(0.5, device="cuda"), torch.tensor(0.5, device="cuda", requires_grad=True)):
    for call in (lambda: fwn.dropout(x, value, (1, 2)), lambda: fwn.sandwich_norm(x, x, scale=value),
                 lambda: fwn.sandwich_norm(x, x, eps=value), lambda: fwn.sandwich_norm(x, x, p=value, rng=(1, 2))):
      with pytest.raises(TypeError, match="must be a number"):
        call()
