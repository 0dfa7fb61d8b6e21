"""linear_act, gated_linear and their gradients where a single call's agreement with the formula shows too little:
repeated calls, forms that the C ABI allows, values at the ends of the activations, errors of whole tensors."""
import pytest
import torch

from sparsefold_b200 import _native, ops

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _device():
  if not torch.cuda.is_available():
    pytest.skip("no CUDA device")
  _native.check(_native.load().sf_device_check(), "sf_device_check")
  yield
  assert _native.device_status() == 0


def rnd(seed, *s):
  return torch.randn(*s, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def gap(got, ref):
  """The error's norm over the reference's."""
  return float((got.double() - ref).norm() / ref.norm())


@pytest.mark.parametrize("rows,k,n,kn", [(4700, 136, 600, False), (9400, 72, 600, True), (3840, 768, 768, False),
                                         (20000, 128, 512, True), (2500, 2056, 1300, False)])
def test_pairs_of_ctas_give_the_same_bits_every_time(rows, k, n, kn):
  """Products of clusters of two, the two halves of each stage loaded by one CTA each: thirty calls, with others between
  that leave different values in the shared memories.  A bf16 sum of one rounding is off by 2^-9 of a value on average
  over its binade (2^-8 at most); the products' own error is far below."""
  x, dy = rnd(1, rows, k).to(BF), rnd(2, rows, n).to(BF)
  w = rnd(3, k, n).div_(k ** 0.5).to(BF).t() if kn else rnd(3, n, k).div_(k ** 0.5).to(BF)
  other = rnd(4, 1000, 264).to(BF), rnd(5, 700, 264).to(BF)
  want = ops.linear_act(x, w), *ops.linear_act_backward(dy, x, w)[:2]
  refs = x.double() @ w.double().t(), dy.double() @ w.double(), dy.double().t() @ x.double()
  for got, ref in zip(want, refs):
    assert gap(got, ref) <= 2.0 ** -8
  for _ in range(30):
    ops.linear_act(*other)
    got = ops.linear_act(x, w), *ops.linear_act_backward(dy, x, w)[:2]
    for a, b in zip(got, want):
      assert torch.equal(a, b)
