"""The differentiable forms and the trainable modules on a machine without a GPU: what they ask of ``ops``, with the
calls themselves replaced by their formulas."""
import pytest
import torch

from sparsefold_b200 import modules, ops, synth, training

ACT = {None: lambda z: z, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}


@pytest.fixture
def calls(monkeypatch):
  """ops.linear_act and ops.gated_linear as formulas; the list of (name, save) that were called."""
  seen = []

  def linear_act(x, wt, bias=None, *, activation=None, residual=None, save=False):
    seen.append(("linear_act", save))
    y = ACT[activation](torch.nn.functional.linear(x, wt, bias)) + (0 if residual is None else residual)
    return (y, y.new_zeros(1)) if save else y

  def gated_linear(x, wt, bias=None, *, activation="silu", save=False):
    seen.append(("gated_linear", save))
    gate, up = torch.nn.functional.linear(x, wt, bias).chunk(2, -1)
    return (ACT[activation](gate) * up, gate.new_zeros(1)) if save else ACT[activation](gate) * up

  monkeypatch.setattr(training.ops, "linear_act", linear_act)
  monkeypatch.setattr(training.ops, "gated_linear", gated_linear)
  return seen


@pytest.mark.parametrize("bias", [False, True])
def test_nothing_is_kept_without_a_gradient_to_compute(calls, bias):
  x, w = torch.randn(3, 8), torch.randn(12, 8, requires_grad=True)
  b = torch.randn(12, requires_grad=True) if bias else None
  with torch.no_grad():
    training.gated_linear(x, w, b)
    training.linear_act(x, w, b, activation="gelu")
    training.linear_act(x, w, b, activation="gelu", residual=torch.zeros(3, 12, requires_grad=True))
  training.gated_linear(x, w.detach(), None if b is None else b.detach())
  training.linear_act(x, w.detach())
  assert [save for _, save in calls] == [False] * 5
  assert training.gated_linear(x, w, b).requires_grad and calls[-1] == ("gated_linear", True)


def test_only_the_residual_is_differentiated(calls):
  x, w, r = torch.randn(3, 8), torch.randn(12, 8), torch.randn(1, 12, requires_grad=True)
  y = training.linear_act(x, w, activation="silu", residual=r)
  assert calls == [("linear_act", False)]
  dy = torch.randn(3, 12)
  y.backward(dy)
  assert torch.allclose(r.grad, dy.sum(0, keepdim=True))
  training.linear_act(x.requires_grad_(True), w, activation="silu", residual=r)
  assert calls[-1] == ("linear_act", True)


def test_the_fused_kernel_sees_the_trained_weights():
  blk = modules.TransitionBlock(16, 2)
  synth.init_params(blk, seed=1)
  modules.trainable(blk)
  modules.trainable(blk, False)                      # not prepared: nothing to pack, and a call still says so
  with pytest.raises(RuntimeError, match="prepare"):
    blk(torch.zeros(2, 16))
  modules.prepare(blk)
  params = modules.trainable(blk)
  with torch.no_grad():
    for p in params:
      p.mul_(-2.0)
  modules.trainable(blk, False)
  assert torch.equal(blk._packed("w1", torch.float32), blk.transition1.weight.detach().t())
  assert torch.equal(blk._packed("w2", torch.bfloat16), blk.transition2.weight.detach().t().to(torch.bfloat16))
  assert torch.equal(blk._kept("ln_w"), blk.input_layer_norm.weight.detach())
  assert torch.equal(blk._kept("ln_b"), blk.input_layer_norm.bias.detach())


class OnOne(torch.Tensor):
  """A host tensor that says it is on the second GPU."""
  is_cuda = True

  def get_device(self):
    return 1

  def contiguous(self):
    return self


def test_layer_norm_runs_on_its_tensors_device(monkeypatch):
  """The launch and its stream belong to x's device, whichever device is current."""
  current, launched = [0], []

  class Device:
    def __init__(self, index):
      self.index = index

    def __enter__(self):
      self.before, current[0] = current[0], self.index

    def __exit__(self, *_):
      current[0] = self.before

  monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
  monkeypatch.setattr(torch.cuda, "device", Device)
  monkeypatch.setattr(ops, "_stream", lambda: 100 + current[0])
  monkeypatch.setattr(ops.N, "call", lambda name, *args: launched.append((name, current[0], args[-1])))
  ops.layer_norm(torch.zeros(2, 8).as_subclass(OnOne), None, None)
  assert launched == [("sf_layernorm", 1, 101)] and current == [0]


@pytest.mark.parametrize("bad", [torch.ones(7), torch.ones(9), torch.ones(1, 8), torch.ones(8, dtype=torch.bfloat16),
                                 torch.ones(8, dtype=torch.float64)], ids=str)
def test_layer_norm_refuses_other_weights(monkeypatch, bad):
  """The kernel reads [cols] fp32 values of weight and bias: a shorter one would be read out of range."""
  monkeypatch.setattr(ops.N, "call", lambda *_: pytest.fail("launched"))
  x, bad = torch.zeros(2, 8).as_subclass(OnOne), bad.as_subclass(OnOne)
  for args in ((bad, None), (None, bad)):
    with pytest.raises(ValueError, match="layer_norm"):
      ops.layer_norm(x, *args)

  class OnZero(OnOne):
    def get_device(self):
      return 0

  with pytest.raises(ValueError, match="layer_norm"):
    ops.layer_norm(x, torch.ones(8).as_subclass(OnZero), None)


def test_layer_norm_of_no_rows(monkeypatch):
  monkeypatch.setattr(ops.N, "call", lambda *_: pytest.fail("launched"))
  w = torch.ones(8).as_subclass(OnOne)
  for shape in ((0, 8), (3, 0, 8)):
    assert ops.layer_norm(torch.zeros(shape).as_subclass(OnOne), w, w).shape == shape


def test_a_forward_only_module_warns_where_a_gradient_ends(recwarn):
  class Forward(modules.B200Module, torch.nn.Module):
    _native_prepared = True

    @modules._require_prepared
    def forward(self, x, *, residual=None):
      return x.detach()

  m, x = Forward(), torch.zeros(3)
  m(x)
  m(x, residual=torch.zeros(3))
  with torch.no_grad():
    m(torch.zeros(3, requires_grad=True))
  m._sf_trainable = True
  m(torch.zeros(3, requires_grad=True))
  assert not recwarn.list
  m._sf_trainable = False
  with pytest.warns(UserWarning, match="Forward runs forward only"):
    m(torch.zeros(3, requires_grad=True))
  with pytest.warns(UserWarning, match="none passes through"):
    m(x, residual=torch.zeros(3, requires_grad=True))
