"""linear_act, gated_linear and their gradients where a single call's agreement with the formula shows too little:
repeated calls, forms that the C ABI allows, values at the ends of the activations, errors of whole tensors."""
import ctypes as C
import threading

import pytest
import torch

from sparsefold_b200 import _native as N
from sparsefold_b200 import modules, ops, synth, training

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _device():
  if not torch.cuda.is_available():
    pytest.skip("no CUDA device")
  N.check(N.load().sf_device_check(), "sf_device_check")
  yield
  assert N.device_status() == 0


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


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,k,n", [(12346, 8, 4072), (16397, 16, 2048), (2976, 104, 4840), (9610, 40, 3320)])
def test_large_outputs_of_few_columns_give_the_same_bits_every_time(rows, k, n, dtype):
  """Bound by the stores, with warps that have no row in the last row tile: what the tile before it has staged must leave
  its buffer first.  Twenty calls of each form; a wrong buffer is 1024 elements of another tile."""
  x, w, b, res = rnd(1, rows, k).to(dtype), (rnd(2, n, k) / k ** 0.5).to(dtype), rnd(3, n), rnd(4, rows, n).to(dtype)
  dy, half = rnd(5, rows, k).to(dtype), n // 2
  z = x.double() @ w.double().t()
  calls = [(lambda: ops.linear_act(x, w), z),
           (lambda: ops.linear_act(x, w, b, activation="sigmoid", residual=res), torch.sigmoid(z + b.double()) + res.double()),
           (lambda: ops.gated_linear(x, w), torch.nn.functional.silu(z[:, :half]) * z[:, half:]),
           (lambda: ops.linear_act_backward(dy, res, w.t(), need_dwt=False)[0], dy.double() @ w.double().t())]
  for call, ref in calls:
    first = call()
    assert gap(first, ref) <= (2.0 ** -9 * 1.05 if dtype == BF else 3 * 6.8e-7)
    for _ in range(20):
      assert torch.equal(call(), first)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,k,n", [(4, 16, 48), (20, 16, 48), (20, 4096, 4104), (200, 72, 72), (200, 1200, 77), (9400, 72, 600)])
def test_gelu_keeps_its_tail(rows, k, n, dtype):
  """gelu and its derivative between -12 and 6, relatively, on every path (dot products, tiles with and without a staged
  epilogue, clusters of two, saved pre-activations): z is the bias alone, one value to a column, and dy is one in a
  single row, so that dbias is the derivative before any rounding to bf16.
  bf16: one rounding (2^-8) of a value off by 2^-17 of itself; the derivative Phi + z phi by 2^-16 of its two terms.
  fp32: Phi = erfc / 2, whose argument's rounding 2^-24 x costs 2 x^2 2^-24 of it (x^2 <= 72: 2^-16.8)."""
  z = torch.cat((torch.linspace(-12, -2, n - 8, device="cuda"), torch.linspace(-1, 6, 8, device="cuda")))
  x = rnd(1, rows, k).to(dtype)
  w = torch.zeros(n, k, dtype=dtype, device="cuda")
  dy = torch.zeros(rows, n, dtype=dtype, device="cuda")
  dy[rows // 2] = 1.0
  zd = z.double()
  phi, cdf = (-0.5 * zd * zd).exp() / (2 * torch.pi) ** 0.5, 0.5 * torch.special.erfc(-zd * 0.5 ** 0.5)
  a, da = zd * cdf, cdf + zd * phi
  y, saved = ops.linear_act(x, w, z, activation="gelu", save=True)
  tol = (2.0 ** -8 if dtype == BF else 0.0) + 2.0 ** -16
  assert bool(((y.double() - a).abs() <= tol * a.abs()).all())
  two, one = torch.cat((z, torch.ones_like(z))), torch.cat((w, w))
  assert bool(((ops.gated_linear(x, one, two, activation="gelu").double() - a).abs() <= tol * a.abs()).all())
  for s in {id(saved): saved, 0: None}.values():
    db = ops.linear_act_backward(dy, x, w, z, activation="gelu", saved=s)[2].double()
    assert bool(((db - da).abs() <= 2.0 ** -16 * (cdf + zd.abs() * phi)).all())
    db = ops.gated_linear_backward(dy, x, one, two, activation="gelu", saved=None)[2].double()
    assert bool(((db[:n] - da).abs() <= 2.0 ** -16 * (cdf + zd.abs() * phi)).all())
    assert bool(((db[n:] - a).abs() <= 2.0 ** -16 * a.abs()).all())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_transition_of_no_rows(dtype):
  """Outputs and input gradients without rows, zero gradients of the parameters."""
  x = torch.zeros(2, 0, 24, dtype=dtype, device="cuda", requires_grad=True)
  lw, lb = (torch.ones(24, device="cuda", requires_grad=True) for _ in range(2))
  w1, w2 = rnd(1, 64, 24).to(dtype).requires_grad_(True), rnd(2, 24, 32).to(dtype).requires_grad_(True)
  y = training.transition(x, lw, lb, w1, w2)
  assert y.shape == x.shape
  y.sum().backward()
  assert x.grad.shape == x.shape
  for p in (lw, lb, w1, w2):
    assert p.grad.shape == p.shape and not p.grad.any()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("n", [(1 << 16) * 128 + 3, (1 << 16) * 512 + 4])
def test_gradients_of_more_columns_than_a_grid_axis_has_blocks(n, gated):
  """dz from saved pre-activations, in ranges of 128 columns (n odd) and of 512.  One row: dbias is dz before its rounding,
  dy silu'(z) (2^-20 of the activation's terms, one product)."""
  wide = 2 * n if gated else n
  x, w = rnd(1, 1, 2).to(BF), torch.zeros(wide, 2, dtype=BF, device="cuda")
  saved = torch.linspace(-6, 6, wide, device="cuda")[None].contiguous()
  dy, b = torch.ones(1, n, dtype=BF, device="cuda"), torch.zeros(wide, device="cuda")
  fn = ops.gated_linear_backward if gated else ops.linear_act_backward
  got = fn(dy, x, w, b, activation="silu", saved=saved, need_dx=False, need_dwt=False)[2]
  z, s = saved[0, :n], torch.sigmoid(saved[0, :n])
  want = s * (1 + z * (1 - s)) * (saved[0, n:] if gated else 1.0)
  # against fp32 arithmetic of the same formula: a few roundings of terms that are at most 1 + |z| (times |up|)
  tol = 2.0 ** -18 * (1 + z.abs()) * (saved[0, n:].abs() if gated else 1.0) + 2.0 ** -30
  assert bool(((got[:n] - want).abs() <= tol).all())
  if gated:
    assert bool(((got[n:] - z * s).abs() <= 2.0 ** -18 * z.abs() + 2.0 ** -30).all())


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("k", [2048, 8192])
def test_bias_gradient_without_a_bias(k, gated):
  """The C ABI gives dbias without a bias too, to the same accuracy: z short by at most 512 * 1.1e-9 = 5.6e-7 of itself,
  whose part in dbias is at most 1.5 of that, and roundings that average out over the rows: 2^-20 of its norm."""
  rows, n = 2000, 72
  wide = 2 * n if gated else n
  x, w, dy = rnd(1, rows, k).to(BF), (rnd(2, wide, k) / k ** 0.5).to(BF), rnd(3, rows, n).to(BF)
  db = torch.empty(wide, device="cuda")
  op = N.SF_OP_GATED_LINEAR_BACKWARD if gated else N.SF_OP_LINEAR_ACT_BACKWARD
  a = N.LinearArgs(dtype=N.SF_BF16, activation=N.ACTIVATIONS["silu"], rows=rows, k=k, n=n, x=x.data_ptr(), x_sr=k,
                   wt=w.data_ptr(), w_sn=k, w_sk=1, dy=dy.data_ptr(), dy_sr=n, dbias=db.data_ptr())
  need = N.load().sf_linear_act_workspace(C.byref(a), op)
  ws = torch.empty(need, dtype=torch.uint8, device="cuda")
  N.call("sf_gated_linear_backward" if gated else "sf_linear_act_backward", C.byref(a), ws.data_ptr(), need,
         torch.cuda.current_stream().cuda_stream)
  z = (x.double() @ w.double().t()).requires_grad_(True)
  y = torch.nn.functional.silu(z[:, :n]) * (z[:, n:] if gated else 1.0)
  ref = torch.autograd.grad((y * dy.double()).sum(), z)[0].sum(0)
  assert gap(db, ref) <= 2.0 ** -20


def test_a_stack_trains_its_last_transitions_and_says_so():
  """Two Pairformer blocks: gradients reach the transitions behind the last forward-only module of each track, and the
  first block's, which feed such modules, stay without one; the second block's modules warn of it."""
  blocks = torch.nn.ModuleList(modules.PairFormerIteration() for _ in range(2))
  for i, b in enumerate(blocks):
    synth.init_params(b, seed=i)
  modules.prepare(blocks)
  blocks = blocks.cuda()
  modules.trainable(blocks)
  pair, single = rnd(1, 24, 24, 128).to(BF), rnd(2, 24, 384).to(BF)
  mask = torch.ones(24, dtype=torch.bool, device="cuda")
  with pytest.warns(UserWarning, match="runs forward only"):
    for b in blocks:
      pair, single = b(pair, seq_mask=mask, single_act=single)
  (pair.float().square().sum() + single.float().square().sum()).backward()
  for i, b in enumerate(blocks):
    for t in (b.pair_transition, b.single_act_update.single_transition):
      for p in (t.input_layer_norm.weight, t.input_layer_norm.bias, t.transition1.weight, t.transition2.weight):
        assert (p.grad is None) == (i == 0)
        assert i == 0 or (bool(torch.isfinite(p.grad).all()) and bool(p.grad.any()))


@pytest.mark.parametrize("rows,k,n,act,kn", [(40, 4_000_000, 64, "relu", False), (40, 4_000_003, 64, None, True),
                                             (300, 2_600_000, 300, "relu", False)])
def test_very_long_sums(rows, k, n, act, kn):
  """Sums of millions of positive bf16 products.  The tensor cores' accumulator cuts some 1e-9 of the sum for each column,
  over 0.004 for four million where the sum is not taken in pieces; rounding the result leaves 2^-9 of the norm at most."""
  x = (rnd(1, rows, k).uniform_(0.5, 1.5)).to(BF)
  w = (rnd(2, k, n).uniform_(0.5, 1.5) / k).to(BF).t() if kn else (rnd(2, n, k).uniform_(0.5, 1.5) / k).to(BF)
  ref = sum(x[:, i:i + 200_000].double() @ w[:, i:i + 200_000].double().t() for i in range(0, k, 200_000))
  assert gap(ops.linear_act(x, w, activation=act), ref) <= 2.0 ** -9
  both = torch.cat((w, w))
  one = ops.gated_linear(x, both, activation="relu")
  assert gap(one, ref * ref) <= 2.0 ** -9


def test_very_long_weight_gradients():
  """The same over the rows: dW of enough tiles that the rows are not split over the CTAs."""
  rows, k, n = 3_000_000, 1536, 1600
  x, dy = torch.empty(rows, k, dtype=BF, device="cuda"), torch.empty(rows, n, dtype=BF, device="cuda")
  ref = torch.zeros(n, k, dtype=torch.float64, device="cuda")
  for i in range(0, rows, 100_000):
    x[i:i + 100_000] = torch.rand(100_000, k, device="cuda") + 0.5
    dy[i:i + 100_000] = torch.rand(100_000, n, device="cuda") + 0.5
    ref += dy[i:i + 100_000].double().t() @ x[i:i + 100_000].double()
  w = torch.zeros(n, k, dtype=BF, device="cuda")
  assert gap(ops.linear_act_backward(dy, x, w, need_dx=False)[1], ref) <= 2.0 ** -9


# ---- errors of whole tensors ------------------------------------------------------------------------------
# Elementwise bounds over all magnitudes are far above what random signs leave, so that a term or a row may be missing
# within them.  Norm of the error over norm of the result, instead, with e = 6.8e-7 for one fp32 product: a sum of 512
# columns is short by at most 5.6e-7 of itself, the dropped terms are 2^-23.  An activation changes by at most 1.5 times
# what its argument does; a gated value has two factors; gradients are products of what dz carries, with their own e.
# bf16: one rounding to nearest is 2^-9 / sqrt(3) to 2^-8 / sqrt(3) of a value over its binade, 0.0017 over them all
# and below 2^-9 = 0.00195; two in a row (dz, the result) below sqrt(2) 2^-9.
E32 = 6.8e-7
SIZES = [(500, 512, 520), (2000, 4096, 264), (8000, 768, 128), (1000, 8192, 72), (600, 700, 4000), (4700, 1100, 600),
         (9401, 75, 601), (19000, 64, 40), (40, 4096, 2056), (33, 700, 96), (65, 2056, 1030)]


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("kn", [False, True])
@pytest.mark.parametrize("rows,k,n", SIZES)
def test_errors_of_whole_tensors(rows, k, n, kn, gated, dtype):
  wide = 2 * n if gated else n
  x, dy, b = rnd(1, rows, k).to(dtype), rnd(2, rows, n).to(dtype), 0.5 * rnd(3, wide)
  w = (rnd(4, k, wide) / k ** 0.5).to(dtype).t() if kn else (rnd(4, wide, k) / k ** 0.5).to(dtype)
  fw, bw = (ops.gated_linear, ops.gated_linear_backward) if gated else (ops.linear_act, ops.linear_act_backward)
  y, saved = fw(x, w, b, activation="silu", save=True)
  z = (x.double() @ w.double().t() + b.double()).requires_grad_(True)
  ref = torch.nn.functional.silu(z[:, :n]) * (z[:, n:] if gated else 1.0)
  dz = torch.autograd.grad((ref * dy.double()).sum(), z)[0]
  ref = ref.detach()
  one, two = (2.0 ** -9, 2.0 ** -8.5) if dtype == BF else ((2.5 if gated else 1.5) * E32, (3.5 if gated else 2.5) * E32)
  assert gap(y, ref) <= one
  for s in {id(saved): saved, 0: None}.values():
    dx, dw, db = bw(dy, x, w, b, activation="silu", saved=s)
    assert gap(dx, dz @ w.double()) <= two
    assert gap(dw, dz.t() @ x.double()) <= two
    assert gap(db, dz.sum(0)) <= (3.5 if gated else 2.5) * E32      # fp32 in both types, from unrounded dz


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,k,n", [(19000, 64, 40), (9401, 75, 601), (4700, 1100, 600), (2047, 139, 128), (513, 96, 384)])
def test_the_last_rows_count(rows, k, n, dtype):
  """dy is zero but in the rows behind the last whole 64, then in the last row alone, then in the rows around every
  512th (where sums of runs meet): dW and dbias have to come from those rows."""
  x, w, b = rnd(1, rows, k).to(dtype), (rnd(2, n, k) / k ** 0.5).to(dtype), rnd(3, n)
  full = rnd(4, rows, n).to(dtype)
  z = x.double() @ w.double().t() + b.double()
  s = torch.sigmoid(z)
  da = s * (1 + z * (1 - s))
  index = torch.arange(rows, device="cuda")
  for keep in (index >= rows // 64 * 64, index == rows - 1, (index + 2) % 512 < 4):
    dy = full * keep[:, None].to(dtype)
    dx, dw, db = ops.linear_act_backward(dy, x, w, b, activation="silu")
    if not bool(keep.any()):
      assert not (dx.any() or dw.any() or db.any())
      continue
    dz = dy.double() * da
    assert gap(dw, dz.t() @ x.double()) <= (2.0 ** -8.5 if dtype == BF else 2.5 * E32)
    assert gap(dx, dz @ w.double()) <= (2.0 ** -8.5 if dtype == BF else 2.5 * E32)
    assert gap(db, dz.sum(0)) <= 2.5 * E32 + 2.0 ** -20 * (dtype == BF)     # the fast activation's 2^-21, few rows
    assert not dx[~keep].any()


@pytest.mark.parametrize("rows", [4, 70, 9400])
def test_the_first_call_of_a_thread(rows):
  """A thread that has made no CUDA call yet, as an autograd worker on its first backward pass, has no current context
  until the runtime binds one; the tensor maps need it."""
  x, w, dy = rnd(1, rows, 64).to(BF), rnd(2, 96, 64).to(BF), rnd(3, rows, 96).to(BF)
  want = ops.linear_act_backward(dy, x, w)[:2]
  got = []
  for call in (lambda: got.append(ops.linear_act(x, w)), lambda: got.extend(ops.linear_act_backward(dy, x, w)[:2])):
    t = threading.Thread(target=call)
    t.start()
    t.join()
  assert len(got) == 3 and torch.equal(got[0], ops.linear_act(x, w))
  assert torch.equal(got[1], want[0]) and torch.equal(got[2], want[1])


# ---- calls that the documentation allows ------------------------------------------------------------------
ROWS = [1, 4, 20, 140, 9400]     # dot products, tiles with and without a staged epilogue, clusters of two


def padded(t, pad):
  """t as a view of wider rows, NaN behind each."""
  room = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), dtype=t.dtype, device=t.device)
  room[:, :t.shape[1]] = t
  return room[:, :t.shape[1]]


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("pad", [8, 3])
@pytest.mark.parametrize("k,n", [(72, 600), (1100, 77)])
@pytest.mark.parametrize("rows", ROWS)
def test_strided_rows_of_dy_and_residual(rows, k, n, pad, dtype):
  """The same values in wider rows, which TMA reads (pad 8) or plain loads do: the same bits."""
  x, res = rnd(1, rows, k).to(dtype), rnd(2, rows, n).to(dtype)
  for gated in (False, True):
    wide = 2 * n if gated else n
    w, b, dy = (rnd(3, wide, k) / k ** 0.5).to(dtype), rnd(4, wide), rnd(5, rows, n).to(dtype)
    fw, bw = (ops.gated_linear, ops.gated_linear_backward) if gated else (ops.linear_act, ops.linear_act_backward)
    saved = fw(x, w, b, activation="gelu", save=True)[1]
    for s in {id(saved): saved, 0: None}.values():
      for act in ("gelu", None):      # without an activation dy is itself the products' operand
        want = bw(dy, x, w, b, activation=act, saved=s)
        for u, v in zip(bw(padded(dy, pad), x, w, b, activation=act, saved=s), want):
          assert torch.equal(u, v)
  w, b = w[:n].contiguous(), b[:n].contiguous()
  for act in ("gelu", None):
    want = ops.linear_act(x, w, b, activation=act, residual=res, save=True)
    got = ops.linear_act(x, w, b, activation=act, residual=padded(res, pad), save=True)
    assert torch.equal(got[0], want[0]) and (want[1] is None or torch.equal(got[1], want[1]))
    assert gap(want[0], res.double() + ops.linear_act(x.double().float(), w.float(), b, activation=act).double()) <= 2.0 ** -8


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("n", [600, 77])
@pytest.mark.parametrize("rows", ROWS)
def test_y_in_the_place_of_the_residual(rows, n, dtype):
  """The C ABI allows it; every element of the residual is read before it is written."""
  k = 72
  x, w, b, res = rnd(1, rows, k).to(dtype), (rnd(2, n, k) / k ** 0.5).to(dtype), rnd(3, n), rnd(4, rows, n).to(dtype)
  want = ops.linear_act(x, w, b, activation="silu", residual=res)
  a = N.LinearArgs(dtype=N.SF_BF16 if dtype == BF else N.SF_F32, activation=N.ACTIVATIONS["silu"], rows=rows, k=k, n=n,
                   x=x.data_ptr(), x_sr=k, wt=w.data_ptr(), w_sn=k, w_sk=1, bias=b.data_ptr(), residual=res.data_ptr(),
                   r_sr=n, y=res.data_ptr())
  need = N.load().sf_linear_act_workspace(C.byref(a), N.SF_OP_LINEAR_ACT)
  ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
  N.call("sf_linear_act", C.byref(a), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
  assert torch.equal(res, want)


def test_bf16_activations_with_fp32_parameters():
  """A block that holds fp32 parameters and meets bf16 activations: fp32 gradients of the bf16 weights' products.  Three
  layers forward and back, each with roundings of 2^-9 on average: 2^-7 of each gradient's norm."""
  blk = modules.TransitionBlock(64, 2)
  p = synth.init_params(blk, seed=3)
  modules.prepare(blk)
  blk = blk.cuda()
  params = modules.trainable(blk)
  x, dy = rnd(8, 5, 21, 64).to(BF).requires_grad_(True), rnd(9, 5, 21, 64).to(BF)
  y = blk(x)
  assert y.dtype == BF
  y.backward(dy)
  assert x.grad.dtype == BF and all(q.dtype == q.grad.dtype == F32 for q in params)
  r = {k: v.cuda().double().requires_grad_(True) for k, v in p.items()}
  xr = x.detach().double().requires_grad_(True)
  n = torch.nn.functional.layer_norm(xr, (64,), r["input_layer_norm.weight"], r["input_layer_norm.bias"], 1e-5)
  gate, up = (n @ r["transition1.weight"]).chunk(2, -1)
  (xr + (torch.nn.functional.silu(gate) * up) @ r["transition2.weight"]).backward(dy.double())
  assert gap(x.grad, xr.grad) <= 2.0 ** -7
  for q, name in zip(params, ("input_layer_norm.weight", "input_layer_norm.bias", "transition1.weight", "transition2.weight")):
    assert gap(q.grad, r[name].grad) <= 2.0 ** -7


def test_two_threads():
  """Calls of two threads on streams of their own, interleaved: the bits of the same calls alone."""
  def work(seed, rows, k, n):
    x, w, b, dy = rnd(seed, rows, k).to(BF), rnd(seed + 1, 2 * n, k).to(BF), rnd(seed + 2, 2 * n), rnd(seed + 3, rows, n).to(BF)
    return lambda: (ops.gated_linear(x, w, b), *ops.gated_linear_backward(dy, x, w, b),
                    ops.clip_grad_norm([x.clone(), dy.clone()], 1.0), *ops.layer_norm_backward(x, x))
  jobs = [work(1, 4700, 136, 600), work(11, 9, 1200, 264)]
  want = [job() for job in jobs]
  torch.cuda.synchronize()
  wrong = []

  def run(job, expect):
    try:
      with torch.cuda.stream(torch.cuda.Stream()):
        for _ in range(20):
          for u, v in zip(job(), expect):
            if v is not None and not torch.equal(u, v):
              wrong.append("other bits")
    except Exception as e:          # a failure in a thread would be lost
      wrong.append(repr(e))

  threads = [threading.Thread(target=run, args=a) for a in zip(jobs, want)]
  for t in threads:
    t.start()
  for t in threads:
    t.join()
  assert not wrong


def test_a_captured_training_pass():
  """Warm-up and capture on one side stream, no eager graph of the leaves alive: replays follow their inputs."""
  x, lw, lb = rnd(1, 70, 64).to(BF), 1 + 0.1 * rnd(2, 64), 0.1 * rnd(3, 64)
  w1, w2, dy = (rnd(4, 256, 64) / 8).to(BF), (rnd(5, 64, 128) / 11).to(BF), rnd(6, 70, 64).to(BF)
  leaves = [t.requires_grad_(True) for t in (x, lw, lb, w1, w2)]

  def step():
    y = training.transition(*leaves)
    return (y.detach(), *torch.autograd.grad(y, leaves, dy))

  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    step()
  torch.cuda.current_stream().wait_stream(side)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph, stream=side):
    got = step()
  with torch.no_grad():
    x.copy_(rnd(7, 70, 64))
    w1.mul_(-0.5)
    dy.mul_(2.0)
  graph.replay()
  torch.cuda.synchronize()
  replayed = [t.clone() for t in got]
  for u, v in zip(replayed, step()):
    assert torch.equal(u, v)


class Room:
  """Outputs of the C ABI inside larger buffers of a known byte, at odd offsets: what lies around them stays as it was."""

  def __init__(self):
    self.all = []

  def take(self, rows, cols, dtype, pad=0, offset=1):
    buf = torch.full(((rows * (cols + pad) + 64 + offset) * dtype.itemsize,), 0xA5, dtype=torch.uint8, device="cuda").view(dtype)
    view = buf[32 + offset:32 + offset + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
    self.all.append((buf, buf.clone(), view.storage_offset(), rows, cols, cols + pad))
    return view

  def check(self):
    for buf, before, at, rows, cols, pitch in self.all:
      outside = torch.ones(buf.numel(), dtype=torch.bool, device="cuda")
      outside.as_strided((rows, cols), (pitch, 1), at).fill_(False)
      size = {2: torch.int16, 4: torch.int32, 1: torch.uint8}[buf.element_size()]
      assert torch.equal(buf.view(size)[outside], before.view(size)[outside])


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("kn", [False, True])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("rows,k,n", [(1, 72, 40), (7, 33, 5), (20, 40, 77), (140, 72, 56), (301, 1100, 130), (4700, 136, 601)])
def test_nothing_else_is_written(rows, k, n, offset, kn, gated, dtype):
  """Both directions through the C ABI: outputs without alignment, dwt in rows wider than its own, a workspace of exactly
  the bytes asked for; the values are those of the Python calls, the surroundings stay."""
  wide = 2 * n if gated else n
  x, dy, b = rnd(1, rows, k).to(dtype), rnd(2, rows, n).to(dtype), rnd(3, wide)
  w = (rnd(4, k, wide) / 9).to(dtype).t() if kn else (rnd(4, wide, k) / 9).to(dtype)
  fw, bw = (ops.gated_linear, ops.gated_linear_backward) if gated else (ops.linear_act, ops.linear_act_backward)
  want_y, want_saved = fw(x, w, b, activation="silu", save=True)
  want = bw(dy, x, w, b, activation="silu", saved=None)
  room = Room()
  y, saved, dx = (room.take(rows, c, t, offset=offset) for c, t in ((n, dtype), (wide, F32), (k, dtype)))
  dwt, db = room.take(*((k, wide) if kn else (wide, k)), dtype, pad=3 + 5 * (offset == 0), offset=offset), room.take(1, wide, F32)
  sn, sk = (1, wide) if kn else (k, 1)
  dn, dk = (1, dwt.stride(0)) if kn else (dwt.stride(0), 1)

  def call(name, op, **more):
    a = N.LinearArgs(dtype=N.SF_BF16 if dtype == BF else N.SF_F32, activation=N.ACTIVATIONS["silu"], rows=rows, k=k, n=n,
                     x=x.data_ptr(), x_sr=k, wt=w.data_ptr(), w_sn=sn, w_sk=sk, bias=b.data_ptr(), **more)
    need = N.load().sf_linear_act_workspace(C.byref(a), op)
    ws = torch.full((need + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
    N.call(name, C.byref(a), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    assert bool((ws[need:] == 0x5A).all())

  form = "sf_gated_linear" if gated else "sf_linear_act"
  forward = N.SF_OP_GATED_LINEAR if gated else N.SF_OP_LINEAR_ACT
  keep = want_saved is not None
  call(form, forward, y=y.data_ptr(), saved=saved.data_ptr() if keep else None)
  assert torch.equal(y, want_y) and (not keep or torch.equal(saved, want_saved))
  back = N.SF_OP_GATED_LINEAR_BACKWARD if gated else N.SF_OP_LINEAR_ACT_BACKWARD
  call(form + "_backward", back, dy=dy.data_ptr(), dy_sr=n, dx=dx.data_ptr(), dwt=dwt.data_ptr(), dw_sn=dn, dw_sk=dk,
       dbias=db.data_ptr())
  assert torch.equal(dx, want[0]) and torch.equal(dwt.t() if kn else dwt, want[1]) and torch.equal(db[0], want[2])
  room.check()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("sums", [False, True])
@pytest.mark.parametrize("rows,cols", [(5, 24), (3000, 128), (700, 267), (100, 768), (33, 4096), (40, 9000)])
def test_dx_in_the_place_of_dy(rows, cols, sums, dtype):
  """The C ABI of the LayerNorm gradient allows it."""
  x, dy, w, b = rnd(1, rows, cols).to(dtype), rnd(2, rows, cols).to(dtype), 1 + 0.1 * rnd(3, cols), rnd(4, cols)
  want = ops.layer_norm_backward(dy, x, w, b, need_dweight=sums, need_dbias=sums)
  dw, db = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
  need = N.load().sf_layernorm_backward_workspace(rows, cols)
  ws = torch.full((need + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
  N.call("sf_layernorm_backward", N.SF_BF16 if dtype == BF else N.SF_F32, dy.data_ptr(), x.data_ptr(), w.data_ptr(),
         dy.data_ptr(), dw.data_ptr() if sums else None, db.data_ptr() if sums else None, rows, cols, 1e-5, ws.data_ptr(),
         need, torch.cuda.current_stream().cuda_stream)
  assert torch.equal(dy, want[0]) and bool((ws[need:] == 0x5A).all())
  if sums:
    assert torch.equal(dw, want[1]) and torch.equal(db, want[2])


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,k,n", [(8, 200, 96), (20, 200, 96), (301, 1100, 130), (9400, 72, 600)])
def test_a_row_does_not_depend_on_the_values_of_others(rows, k, n, dtype):
  """y and dx of a row have the same bits whatever the other rows hold, large values among them."""
  w, b, dy = (rnd(1, 2 * n, k) / k ** 0.5).to(dtype), rnd(2, 2 * n), rnd(3, rows, n).to(dtype)
  x, other = rnd(4, rows, k).to(dtype), (1000 * rnd(5, rows, k)).to(dtype)
  mine = torch.arange(rows, device="cuda") % 3 == 1
  mixed, dy2 = torch.where(mine[:, None], x, other), torch.where(mine[:, None], dy, dy.flip(0))
  for save in (False, True):
    a, s = ops.gated_linear(x, w, b, save=True)
    c, t = ops.gated_linear(mixed, w, b, save=True)
    assert torch.equal(a[mine], c[mine])
    u = ops.gated_linear_backward(dy, x, w, b, saved=s if save else None, need_dwt=False)[0]
    v = ops.gated_linear_backward(dy2, mixed, w, b, saved=t if save else None, need_dwt=False)[0]
    assert torch.equal(u[mine], v[mine])
