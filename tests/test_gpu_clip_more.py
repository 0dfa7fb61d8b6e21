"""clip_grad_norm: the scale's last bit, norms beyond fp32."""
import math

import numpy as np
import pytest
import torch

from sparsefold_b200 import ops

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _device():
  if not torch.cuda.is_available():
    pytest.skip("no CUDA device")


def whole_numbers(n, seed):
  """Small whole numbers: their squares and sums of eight of them are exact in fp32, all of them in fp64."""
  return torch.randint(-8, 9, (n,), generator=torch.Generator().manual_seed(seed)).float()


@pytest.mark.parametrize("sizes", [[7], [5000, 33, 100_001]])
def test_the_scale_is_rounded_once(sizes):
  """The norm's square is exact here, so the scale is limit / (norm + 1e-6) in fp64, to the last bit of its one rounding
  to fp32; ones among the gradients become that number."""
  host = [whole_numbers(n, i) for i, n in enumerate(sizes)]
  for h in host:
    h[0] = 1.0
  grads = [h.cuda() for h in host]
  norm = math.sqrt(sum(float(h.double().square().sum()) for h in host))
  outs = [torch.empty_like(g) for g in grads]
  for i in range(1, 33):
    limit = i / 8
    scale = min(1.0, limit / (norm + 1e-6))
    ops.clip_grad_norm(grads, limit, out=outs)
    for h, o in zip(host, outs):
      assert float(o[0]) == float(np.float32(scale))
      assert torch.equal(o.cpu(), h * torch.tensor(scale, dtype=F32))
    ops.clip_grad_norm(grads, limit, float("inf"), out=outs)      # the largest magnitude: 8 at most
    most = max(float(h.abs().max()) for h in host)
    assert all(float(o[0]) == float(np.float32(min(1.0, limit / (most + 1e-6)))) for o in outs)


def test_a_norm_beyond_fp32():
  """Finite gradients whose norm overflows fp32: the norm is infinite, the gradients are scaled by the true one.
  The scale 1e3 / 9.5e39 is subnormal (1.05e-37 is not): limit 1e3 keeps it normal, so it has one rounding of 2^-24."""
  g = torch.full((1000,), 3e38, device="cuda")
  norm = 3e38 * math.sqrt(1000)
  want = float(g[0].double()) * (1e3 / (float(g[0].double()) * math.sqrt(1000)))
  out = torch.empty_like(g)
  assert float(ops.clip_grad_norm([g], 1e3, out=[out])) == math.inf and norm > 3.5e38
  assert float((out.double() / want - 1).abs().max()) <= 3 * 2.0 ** -24 + 2.0 ** -22   # and runs of eight squares in fp64


def test_an_infinite_limit_leaves_finite_gradients():
  g = whole_numbers(3000, 1).cuda()
  before = g.clone()
  assert float(ops.clip_grad_norm([g], float("inf"))) == float(np.float32(math.sqrt(float(before.double().square().sum()))))
  assert torch.equal(g, before)
