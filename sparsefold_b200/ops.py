"""Torch-facing wrappers of the C ABI: tensors in, tensors out, current stream.

Each wrapper validates shapes/dtypes, allocates outputs and workspace with the
torch caching allocator, and calls one entry point of libsparsefold_b200.so.
Nothing here computes on the host; a missing library raises NativeError.
"""
from __future__ import annotations

import array
import contextlib
import ctypes as C
import math

import torch

from sparsefold_b200 import _native as N


def _dt(t: torch.Tensor) -> int:
  if t.dtype == torch.float32:
    return N.SF_F32
  if t.dtype == torch.bfloat16:
    return N.SF_BF16
  raise TypeError(f"unsupported dtype {t.dtype}; use float32 or bfloat16")


def _stream() -> int:
  return torch.cuda.current_stream().cuda_stream


def _p(t) -> int | None:
  return None if t is None else t.data_ptr()


def _cuda(*ts):
  for t in ts:
    if t is not None and not t.is_cuda:
      raise ValueError("sparsefold_b200 ops take CUDA tensors only")


def _ws(nbytes: int, device) -> torch.Tensor:
  return torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=device)


def mask_u8(mask: torch.Tensor) -> torch.Tensor:
  return mask.to(torch.uint8).contiguous()


# ---------------------------------------------------------------------------
def layer_norm(x: torch.Tensor, weight, bias, eps: float = 1e-5) -> torch.Tensor:
  _cuda(x, weight, bias)
  cols = x.shape[-1]
  for t in (weight, bias):   # the kernel reads [cols] fp32 of each
    if t is not None and (t.dtype != torch.float32 or t.shape != (cols,) or t.get_device() != x.get_device()):
      raise ValueError(f"layer_norm: weight and bias must be fp32 [{cols}] on {x.device}, got {t.dtype} "
                       f"{tuple(t.shape)} on {t.device}")
  weight, bias = (None if t is None else t.contiguous() for t in (weight, bias))
  x = x.contiguous()
  y = torch.empty_like(x)
  if x.numel() == 0:         # no rows: nothing to launch, and torch gives no address
    return y
  with _on(x.get_device()):
    N.call("sf_layernorm", _dt(x), _p(x), _p(y), _p(weight), _p(bias), x.numel() // cols, cols,
           C.c_float(eps), _stream())
  return y


def linear(x: torch.Tensor, wt: torch.Tensor, bias=None, residual=None, post_op=None) -> torch.Tensor:
  """y = post_op(x @ wt.T + bias + residual); wt is [out, in] in x's dtype."""
  _cuda(x, wt, bias, residual)
  x = x.contiguous()
  k = x.shape[-1]
  n = wt.shape[0]
  assert wt.shape[1] == k and wt.dtype == x.dtype
  rows = x.numel() // k
  y = torch.empty(*x.shape[:-1], n, dtype=x.dtype, device=x.device)
  if residual is not None:
    residual = residual.to(x.dtype).expand_as(y).contiguous()
  N.call("sf_linear", _dt(x), _p(x), _p(wt), _p(bias), _p(residual), _p(y), rows, k, n,
         N.POST_OPS[post_op], _stream())
  return y


def attention(q, k, v, *, scale=None, mask_q=None, mask_k=None, bias=None, gate=None,
              mask_row=None) -> torch.Tensor:
  """Drop-in for backends/torch/attention/sdpa.py:22 dot_product_attention.

  q [..., Q, H, D], k [..., K, H, D], v [..., K, H, Dv] (Dv may differ from D,
  as sdpa.py allows), masks [..., Q] / [..., K] (broadcast), bias broadcastable
  to [..., H, Q, K]; optional gate [..., Q, H, Dv] applies sigmoid(gate) to the
  output.  Returns [..., Q, H, Dv] in q's dtype.
  """
  _cuda(q, k, v)
  batch = q.shape[:-3]
  Q, H, D = q.shape[-3:]
  K = k.shape[-3]
  Dv = v.shape[-1]
  B = math.prod(batch) if batch else 1
  dt = _dt(q)
  q3 = q.reshape(B, Q, H, D)
  k3 = k.expand(*batch, K, H, D).reshape(B, K, H, D)
  v3 = v.expand(*batch, K, H, Dv).reshape(B, K, H, Dv)
  q3, k3, v3 = (t if t.stride(-1) == 1 else t.contiguous() for t in (q3, k3, v3))
  out = torch.empty(B, Q, H, Dv, dtype=q.dtype, device=q.device)
  a = N.AttentionArgs()
  a.dtype = dt
  a.batch, a.heads, a.q_len, a.k_len, a.head_dim = B, H, Q, K, D
  a.value_dim = Dv
  a.q, a.q_sb, a.q_sh, a.q_sq = _p(q3), q3.stride(0), q3.stride(2), q3.stride(1)
  a.k, a.k_sb, a.k_sh, a.k_sk = _p(k3), k3.stride(0), k3.stride(2), k3.stride(1)
  a.v, a.v_sb, a.v_sh, a.v_sk = _p(v3), v3.stride(0), v3.stride(2), v3.stride(1)
  a.out, a.o_sb, a.o_sh, a.o_sq = _p(out), out.stride(0), out.stride(2), out.stride(1)
  keep = [q3, k3, v3, out]
  if bias is not None:
    b4 = bias.to(q.dtype) if bias.dtype not in (torch.float32, q.dtype) else bias
    b4 = b4.expand(*batch, H, Q, K)
    try:
      b4 = b4.view(B, H, Q, K)
    except RuntimeError:
      b4 = b4.reshape(B, H, Q, K)
    if b4.stride(-1) != 1:
      b4 = b4.contiguous()
    a.bias, a.bias_dtype = _p(b4), _dt(b4)
    a.b_sb, a.b_sh, a.b_sq = b4.stride(0), b4.stride(1), b4.stride(2)
    keep.append(b4)
  if mask_q is not None:
    mq = mask_u8(mask_q.expand(*batch, Q).reshape(B, Q))
    a.mask_q, a.mq_sb = _p(mq), mq.stride(0)
    keep.append(mq)
  if mask_k is not None:
    mk = mask_u8(mask_k.expand(*batch, K).reshape(B, K))
    a.mask_k, a.mk_sb = _p(mk), mk.stride(0)
    keep.append(mk)
  if mask_row is not None:
    mr = mask_u8(mask_row.reshape(B))
    a.mask_row = _p(mr)
    keep.append(mr)
  if gate is not None:
    g3 = gate.reshape(B, Q, H, Dv)
    a.gate, a.g_sb, a.g_sh, a.g_sq = _p(g3), g3.stride(0), g3.stride(2), g3.stride(1)
    keep.append(g3)
  a.scale = float(1.0 / math.sqrt(D) if scale is None else scale)
  N.call("sf_attention", C.byref(a), _stream())
  return out.reshape(*batch, Q, H, Dv)


# ---------------------------------------------------------------------------
def tri_mult_weights(glu, ln_w, ln_b, center_w, center_b, w_out, w_gate) -> N.TriMultWeights:
  return N.TriMultWeights(_p(ln_w), _p(ln_b), _p(glu), _p(center_w), _p(center_b), _p(w_out), _p(w_gate))


def tri_mult(z: torch.Tensor, mask_u8_: torch.Tensor, w: N.TriMultWeights, incoming: bool,
             out: torch.Tensor | None = None) -> torch.Tensor:
  """Whole TriangleMultiplication on one device: returns z + update."""
  _cuda(z)
  n, n2, c = z.shape
  assert n == n2 and c == 128 and z.is_contiguous()
  dt = _dt(z)
  lib = N.load()
  pitch = lib.sf_pair_pitch(n)
  a_op = torch.empty(n, c, pitch, dtype=z.dtype, device=z.device)     # [row][channel][pitch]
  b_op = torch.empty_like(a_op)
  p = torch.empty_like(a_op)
  ws = _ws(max(lib.sf_tri_mult_project_workspace(dt, n), lib.sf_tri_mult_output_workspace(dt, n, n)), z.device)
  N.call("sf_tri_mult_project", dt, _p(z), _p(mask_u8_), n, int(incoming), C.byref(w), _p(a_op), _p(b_op),
         _p(ws), ws.numel(), _stream())
  N.call("sf_tri_mult_contract", dt, _p(a_op), _p(b_op), _p(p), c, n, n, n, _stream())
  out = torch.empty_like(z) if out is None else out
  N.call("sf_tri_mult_output", dt, _p(z), _p(p), n, n, C.byref(w), _p(out), _p(ws), ws.numel(), _stream())
  return out


def tri_attention_weights(ln_w, w_qkvg, w_bias, w_out, heads: int) -> N.TriAttentionWeights:
  return N.TriAttentionWeights(_p(ln_w), _p(w_qkvg), _p(w_bias), _p(w_out), heads)


def tri_attention(z: torch.Tensor, mask_u8_: torch.Tensor, w: N.TriAttentionWeights, transpose: bool,
                  out: torch.Tensor | None = None) -> torch.Tensor:
  _cuda(z)
  n, n2, c = z.shape
  assert n == n2 and c == 128 and z.is_contiguous()
  dt = _dt(z)
  ws = _ws(N.load().sf_tri_attention_workspace(dt, n, w.heads), z.device)
  out = torch.empty_like(z) if out is None else out
  N.call("sf_tri_attention", dt, _p(z), _p(mask_u8_), n, int(transpose), C.byref(w), _p(out), _p(ws),
         ws.numel(), _stream())
  return out


def transition(x: torch.Tensor, ln_w, ln_b, w1, w2, out: torch.Tensor | None = None) -> torch.Tensor:
  _cuda(x)
  x = x.contiguous()
  c = x.shape[-1]
  inter = w1.shape[0] // 2
  rows = x.numel() // c
  dt = _dt(x)
  ws = _ws(N.load().sf_transition_workspace(dt, rows, inter), x.device)
  out = torch.empty_like(x) if out is None else out
  N.call("sf_transition", dt, _p(x), _p(ln_w), _p(ln_b), _p(w1), _p(w2), _p(out), rows, c, inter,
         _p(ws), ws.numel(), _stream())
  return out


def pair_logits(z: torch.Tensor, ln_w, ln_b, w, heads: int) -> torch.Tensor:
  """[H, rows, n] logits of LN(z) @ W (SingleActUpdate, blocks.py:745-749)."""
  _cuda(z)
  rows, n, c = z.shape
  dt = _dt(z)
  out = torch.empty(heads, rows, n, dtype=z.dtype, device=z.device)
  ws = _ws(N.load().sf_pair_logits_workspace(dt, rows, n, c), z.device)
  N.call("sf_pair_logits", dt, _p(z.contiguous()), _p(ln_w), _p(ln_b), _p(w), _p(out), rows, n, c, heads,
         _p(ws), ws.numel(), _stream())
  return out


# ---------------------------------------------------------------------------
# diffusion-transformer and MSA helpers
# ---------------------------------------------------------------------------
def _trailing_period(t: torch.Tensor, like: torch.Tensor):
  """(t, period) with t contiguous and like's trailing shape: the elements of t repeat every
  `period` elements of like (t broadcasts over like's leading dims), or t expanded in full."""
  t = t.to(like.dtype)
  lead = like.ndim - t.ndim
  if lead >= 0 and tuple(t.shape) == tuple(like.shape[lead:]):
    t = t.contiguous()
    return t, t.numel()
  t = t.expand_as(like).contiguous()
  return t, t.numel()


def adaln(x: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor) -> torch.Tensor:
  """scale * LN(x) + bias, all [..., C] of x's dtype (AdaptiveLayerNorm with single_cond); scale and
  bias may have fewer leading dims than x (one conditioning for every sample) and are not copied then."""
  _cuda(x, scale, bias)
  x = x.contiguous()
  c = x.shape[-1]
  if scale.shape != bias.shape:
    scale, bias = torch.broadcast_tensors(scale, bias)
  scale, per = _trailing_period(scale, x)
  bias, per_b = _trailing_period(bias, x)
  if per_b != per:
    scale, per = scale.expand_as(x).contiguous(), x.numel()
    bias = bias.expand_as(x).contiguous()
  y = torch.empty_like(x)
  N.call("sf_adaln", _dt(x), _p(x), _p(scale), _p(bias), _p(y), x.numel() // c, c, per // c, _stream())
  return y


def gated_residual(base, u: torch.Tensor, gate: torch.Tensor) -> torch.Tensor:
  """base + u * gate (base may be None); gate broadcasts to u's shape (over leading dims without a copy)."""
  _cuda(u, gate, base)
  u = u.contiguous()
  gate, per = _trailing_period(gate, u)
  if base is not None:
    base = base.to(u.dtype).expand_as(u).contiguous()
  out = torch.empty_like(u)
  N.call("sf_gated_residual", _dt(u), _p(base), _p(u), _p(gate), _p(out), u.numel(), per, _stream())
  return out


def gather_rows(src: torch.Tensor, idx: torch.Tensor, mask: torch.Tensor) -> torch.Tensor:
  """src [B, R, C] -> out [B, n_out, C] with out[b, i] = mask[i] ? src[b, idx[i]] : 0."""
  _cuda(src, idx, mask)
  src = src.contiguous()
  b, r, c = src.shape
  idx = idx.reshape(-1).to(torch.int32).contiguous()
  m = mask_u8(mask.reshape(-1))
  out = torch.empty(b, idx.numel(), c, dtype=src.dtype, device=src.device)
  N.call("sf_gather_rows", _dt(src), _p(src), b, r, _p(idx), _p(m), idx.numel(), c, _p(out), _stream())
  return out


def mask_rows_(x: torch.Tensor, mask: torch.Tensor) -> torch.Tensor:
  """In place: x[..., :] = 0 where !mask[...] (mask has x's leading shape)."""
  _cuda(x, mask)
  assert x.is_contiguous()
  c = x.shape[-1]
  m = mask_u8(mask.expand(x.shape[:-1]).reshape(-1))
  N.call("sf_mask_rows", _dt(x), _p(x), _p(m), x.numel() // c, c, _stream())
  return x


def softmax_rows(x: torch.Tensor, key_bias=None, out=None, ldy=None) -> torch.Tensor:
  _cuda(x, key_bias)
  x = x.contiguous()
  k = x.shape[-1]
  rows = x.numel() // k
  if out is None:
    out = torch.empty_like(x)
  N.call("sf_softmax_rows", _dt(x), _p(x), _p(key_bias), _p(out), rows, k, ldy or k, _stream())
  return out


def transpose_(src: torch.Tensor, dst: torch.Tensor, nb1, nb2, rows, cols, ib1, ib2, is_r, ob1, ob2, os_c) -> None:
  """Batched strided transpose between two CUDA buffers (strides in elements)."""
  _cuda(src, dst)
  N.call("sf_transpose", _dt(src), _p(src), _p(dst), nb1, nb2, rows, cols, ib1, ib2, is_r, ob1, ob2, os_c, _stream())


def pitch(n: int) -> int:
  return int(N.load().sf_pair_pitch(n))


def contract(a_op: torch.Tensor, b_op: torch.Tensor, channels: int, rows: int, cols: int, kdim: int) -> torch.Tensor:
  """P[i][c][j] = sum_k A[i][c][k] B[j][c][k]; A [rows][c][pitch(k)], B [cols][c][pitch(k)] -> [rows][c][pitch(cols)]."""
  _cuda(a_op, b_op)
  p = torch.empty(rows, channels, pitch(cols), dtype=a_op.dtype, device=a_op.device)
  N.call("sf_tri_mult_contract", _dt(a_op), _p(a_op), _p(b_op), _p(p), channels, rows, cols, kdim, _stream())
  return p


def opm_norm(mask: torch.Tensor, dtype) -> torch.Tensor:
  """[n_res, n_res] fp32 = 1/(1e-3 + sum_m mask[m,i] mask[m,j]) (count rounded to dtype)."""
  _cuda(mask)
  m = mask_u8(mask)
  n_seq, n_res = m.shape
  ws = _ws(N.load().sf_opm_norm_workspace(n_seq, n_res), m.device)
  norm = torch.empty(n_res, n_res, dtype=torch.float32, device=m.device)
  dt = N.SF_F32 if dtype == torch.float32 else N.SF_BF16
  N.call("sf_opm_norm", dt, _p(m), n_seq, n_res, _p(norm), _p(ws), ws.numel(), _stream())
  return norm


def opm_repack(o: torch.Tensor, n_res: int, d: int) -> torch.Tensor:
  _cuda(o)
  out = torch.empty(n_res * n_res, d * d, dtype=o.dtype, device=o.device)
  N.call("sf_opm_repack", _dt(o), _p(o), o.shape[-1], n_res, d, _p(out), _stream())
  return out


def scale_rows_(x: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
  _cuda(x, s)
  assert x.is_contiguous() and s.dtype == torch.float32
  c = x.shape[-1]
  N.call("sf_scale_rows", _dt(x), _p(x), _p(s.contiguous()), x.numel() // c, c, _stream())
  return x


def swiglu(h: torch.Tensor) -> torch.Tensor:
  """[..., 2I] -> swish(h[..., :I]) * h[..., I:]."""
  _cuda(h)
  h = h.contiguous()
  i2 = h.shape[-1]
  out = torch.empty(*h.shape[:-1], i2 // 2, dtype=h.dtype, device=h.device)
  N.call("sf_swiglu", _dt(h), _p(h), _p(out), h.numel() // i2, i2 // 2, _stream())
  return out


def pair_outer_sum(left: torch.Tensor, right: torch.Tensor, addend=None) -> torch.Tensor:
  """out[i, j] = left[i] + right[j] (+ addend[i, j]): [B, C] x [N, C] -> [B, N, C] in left's dtype
  (Evoformer._get_seq_pair_embedding, trunk/network.py:195-212)."""
  _cuda(left, right, addend)
  assert left.ndim == 2 and right.ndim == 2 and left.shape[1] == right.shape[1] and left.dtype == right.dtype
  b, c = left.shape
  n = right.shape[0]
  left, right = left.contiguous(), right.contiguous()
  if addend is not None:
    addend = addend.to(left.dtype).expand(b, n, c).contiguous()
  out = torch.empty(b, n, c, dtype=left.dtype, device=left.device)
  N.call("sf_pair_outer_sum", _dt(left), _p(left), _p(right), _p(addend), _p(out), b, n, c, _stream())
  return out


def pair_sparse_linear(x: torch.Tensor, w_kc: torch.Tensor, residual=None) -> torch.Tensor:
  """out[..., :] = sum over the nonzero x[..., k] of x[..., k] * w_kc[k, :] (+ residual): the linear layers
  on one-hot / 0-1 pair features (trunk/network.py:188-193, :214-256).  w_kc is fp32 [K, C]."""
  _cuda(x, w_kc, residual)
  assert w_kc.dtype == torch.float32 and w_kc.ndim == 2 and x.shape[-1] == w_kc.shape[0]
  x = x.contiguous()
  k, c = w_kc.shape
  out = torch.empty(*x.shape[:-1], c, dtype=x.dtype, device=x.device)
  if residual is not None:
    residual = residual.to(x.dtype).expand_as(out).contiguous()
  N.call("sf_pair_sparse_linear", _dt(x), _p(x), _p(w_kc.contiguous()), _p(residual), _p(out), x.numel() // k, k, c,
         _stream())
  return out


# ---------------------------------------------------------------------------
# linear layers with gradients, the LayerNorm gradient, gradient clipping
# ---------------------------------------------------------------------------
# A forward call with save=True keeps the fp32 pre-activations only above this input width.  Up to it the
# backward computes them again: for many bf16 rows 2 k flop at the tensor cores' rate against 8 bytes (written and
# read back) at the memory's meet near k = 1000.  One rule for all: fp32 operands (six products, k = 170) and few rows
# (pre-activations that stay in L2; 3840 x 768 x 768 spends 17 us on the second product) would gain from saving earlier.
SAVE_ABOVE_K = 1024


def _on(index: int):
  """The device as the current one (a no-op where it is already: switching costs more than a small launch)."""
  return contextlib.nullcontext() if index == torch.cuda.current_device() else torch.cuda.device(index)


def _raw_stream(index: int) -> int:
  """The device's current stream as a handle, without the Stream object of ``_stream`` (3 us, as much as the
  launch that follows; these ops are called for single rows too)."""
  return torch._C._cuda_getCurrentRawStream(index)


def _linear_call(name: str, op: int, args: N.LinearArgs, x: torch.Tensor) -> None:
  index = x.get_device()
  if index != torch.cuda.current_device():
    with torch.cuda.device(index):
      return _linear_call(name, op, args, x)
  ref, lib, ws = C.byref(args), N.load(), None
  need = lib.sf_linear_act_workspace(ref, op)
  if need:
    room = torch.empty(need, dtype=torch.uint8, device=x.device)
    ws = room.data_ptr()
  status = getattr(lib, name)(ref, ws, need, _raw_stream(index))
  if status:
    N.check(status, name)


def _rows2d(t: torch.Tensor, cols: int) -> torch.Tensor:
  """[..., cols] as rows with a unit inner stride, without a copy where the strides allow it."""
  if t.ndim != 2:
    t = t.reshape(-1, cols)
  sr, sc = t.stride()
  if sc != 1 or (sr < cols and len(t) > 1):
    t = t.contiguous()
    t = t if t.stride(1) == 1 else t.as_strided(t.shape, (cols, 1))   # one column: torch keeps any stride there
  return t


def _weight2d(wt: torch.Tensor) -> torch.Tensor:
  """A [n, k] weight in either orientation (a transposed view is taken as it is)."""
  n, k = wt.shape
  sn, sk = wt.stride()
  return wt if (sk == 1 and sn >= k) or (sn == 1 and sk >= n) else wt.contiguous().as_strided((n, k), (k, 1))


def _linear_args(what, x, wt, bias, activation, gated, *others) -> tuple:
  """Checks shared by the linear layers with gradients; (args, x rows, weight, bias, features)."""
  act = N.ACTIVATIONS.get(activation)
  if act is None:
    raise ValueError(f"{what}: activation {activation!r} is not one of {sorted(k for k in N.ACTIVATIONS if k)}")
  xs, size = x.shape, wt.shape
  if len(size) != 2 or not xs or size[1] != xs[-1]:
    raise ValueError(f"{what}: x {tuple(xs)} does not fit a weight {tuple(size)}")
  wide, k = size
  if k == 0 or wide == 0 or (gated and wide % 2):
    raise ValueError(f"{what}: weight {tuple(wt.shape)}")
  dtype, index = x.dtype, x.get_device()
  if index < 0:
    raise ValueError("sparsefold_b200 ops take CUDA tensors only")
  if wt.dtype != dtype:
    raise TypeError(f"{what}: weight is {wt.dtype}, x is {dtype}")
  for t in (wt, bias, *others):
    if t is not None and t.get_device() != index:
      raise ValueError(f"{what}: tensors on {t.device} and {x.device}")
  pb = None
  if bias is not None:
    if bias.dtype != torch.float32 or bias.shape != (wide,):
      raise ValueError(f"{what}: bias must be fp32 [{wide}], got {bias.dtype} {tuple(bias.shape)}")
    bias = bias.contiguous()
    pb = bias.data_ptr()
  x2, w2 = _rows2d(x, k), _weight2d(wt)
  n = wide // 2 if gated else wide
  sn, sk = w2.stride()
  a = N.LinearArgs(_dt(x), act, len(x2), k, n, x2.data_ptr(), x2.stride()[0], w2.data_ptr(), sn, sk, pb)
  return a, x2, w2, bias, n


def _saved_for(x: torch.Tensor, rows: int, wide: int, k: int, has_act: bool):
  """Room for the pre-activations that a backward reads, or None where it computes them again."""
  if not has_act or k <= SAVE_ABOVE_K:
    return None
  return torch.empty(rows, wide, dtype=torch.float32, device=x.device)


def linear_act(x: torch.Tensor, wt: torch.Tensor, bias=None, *, activation=None, residual=None, save: bool = False):
  """y = activation(x @ wt.T + bias) + residual in one kernel: x [..., k], wt [n, k] in x's dtype (contiguous or
  a transposed view), bias fp32 [n], residual broadcastable to [..., n]; activation None, "relu", "silu",
  "sigmoid" or "gelu" (the erf form).  (``linear`` adds its residual before post_op, as the reference does.)
  fp32 inputs are computed to fp32 accuracy.  With save=True returns (y, saved); ``saved`` goes to
  ``linear_act_backward`` (a tensor, or None where the backward computes what it needs again).  y is rounded once
  either way, but its last bit may depend on save: pre-activations to keep are summed in shorter runs."""
  a, x2, w2, bias, n = _linear_args("linear_act", x, wt, bias, activation, False, residual)
  y = torch.empty((*x.shape[:-1], n), dtype=x.dtype, device=x.device)
  if residual is not None:
    if residual.dtype != x.dtype or residual.shape != y.shape:
      residual = residual.to(x.dtype).expand(y.shape)
    residual = _rows2d(residual, n)
    a.residual, a.r_sr = residual.data_ptr(), residual.stride(0)
  saved = _saved_for(x, x2.shape[0], n, a.k, a.activation != 0) if save else None
  a.y, a.saved = y.data_ptr(), _p(saved)
  _linear_call("sf_linear_act", N.SF_OP_LINEAR_ACT, a, x)
  return (y, saved) if save else y


def gated_linear(x: torch.Tensor, wt: torch.Tensor, bias=None, *, activation="silu", save: bool = False):
  """y = activation(x @ wt[:i].T + bias[:i]) * (x @ wt[i:].T + bias[i:]) in one kernel: the gated product of a
  transition.  x [..., k], wt [2 i, k] (gate rows first, as ``transition``'s w1; contiguous or a transposed
  view), bias fp32 [2 i]; returns [..., i], with save=True (y, saved) as ``linear_act``."""
  a, x2, w2, bias, n = _linear_args("gated_linear", x, wt, bias, activation, True)
  y = torch.empty((*x.shape[:-1], n), dtype=x.dtype, device=x.device)
  saved = _saved_for(x, x2.shape[0], 2 * n, a.k, True) if save else None
  a.y, a.saved = y.data_ptr(), _p(saved)
  _linear_call("sf_gated_linear", N.SF_OP_GATED_LINEAR, a, x)
  return (y, saved) if save else y


def _linear_backward(what, gated, dy, x, wt, bias, activation, saved, need_dx, need_dwt, need_dbias):
  a, x2, w2, bias, n = _linear_args(what, x, wt, bias, activation, gated, dy, saved)
  wide = wt.shape[0]
  if dy.dtype != x.dtype or dy.shape != (*x.shape[:-1], n):
    raise ValueError(f"{what}: dy must be {x.dtype} {(*x.shape[:-1], n)}, got {dy.dtype} {tuple(dy.shape)}")
  if saved is not None and (saved.dtype != torch.float32 or saved.shape != (x2.shape[0], wide)
                            or not saved.is_contiguous()):
    raise ValueError(f"{what}: saved must be what the forward call returned, fp32 {(x2.shape[0], wide)}")
  dy2 = _rows2d(dy, n)
  a.dy, a.dy_sr = dy2.data_ptr(), dy2.stride()[0]
  dx = dwt = dbias = None
  if saved is not None:
    a.saved = saved.data_ptr()
  if need_dx:
    dx = torch.empty_like(x, memory_format=torch.contiguous_format)
    a.dx = dx.data_ptr()
  if need_dwt:   # in the weight's own orientation
    k = a.k
    if a.w_sk == 1 and a.w_sn >= k:
      dwt = torch.empty_like(wt, memory_format=torch.contiguous_format)
      a.dw_sn, a.dw_sk = k, 1
    else:
      dwt = torch.empty((k, wide), dtype=wt.dtype, device=wt.device).t()
      a.dw_sn, a.dw_sk = 1, wide
    a.dwt = dwt.data_ptr()
  if need_dbias and bias is not None:
    dbias = torch.empty_like(bias)
    a.dbias = dbias.data_ptr()
  _linear_call("sf_" + what, N.SF_OP_GATED_LINEAR_BACKWARD if gated else N.SF_OP_LINEAR_ACT_BACKWARD, a, x)
  return dx, dwt, dbias


def linear_act_backward(dy, x, wt, bias=None, *, activation=None, saved=None, need_dx=True, need_dwt=True,
                        need_dbias=True):
  """(dx, dwt, dbias) of ``linear_act`` from dy [..., n]; the residual's gradient is dy itself.  dbias is fp32 and
  None without a bias, dwt has wt's dtype and orientation; ``saved`` as the forward call returned it (None
  is always right: the pre-activations are then computed again)."""
  return _linear_backward("linear_act_backward", False, dy, x, wt, bias, activation, saved, need_dx, need_dwt,
                          need_dbias)


def gated_linear_backward(dy, x, wt, bias=None, *, activation="silu", saved=None, need_dx=True, need_dwt=True,
                          need_dbias=True):
  """(dx, dwt, dbias) of ``gated_linear`` from dy [..., i]; see ``linear_act_backward``."""
  return _linear_backward("gated_linear_backward", True, dy, x, wt, bias, activation, saved, need_dx, need_dwt,
                          need_dbias)


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight=None, bias=None, eps: float = 1e-5, *,
                        need_dx=True, need_dweight=True, need_dbias=True):
  """(dx, dweight, dbias) of ``layer_norm`` from dy and the forward input x (both [..., c], one dtype); dweight and
  dbias are fp32, None without a weight or bias."""
  index = x.get_device()
  if index < 0:
    raise ValueError("sparsefold_b200 ops take CUDA tensors only")
  xs = x.shape
  if dy.shape != xs or dy.dtype != x.dtype or not xs or xs[-1] == 0:
    raise ValueError(f"layer_norm_backward: dy {dy.dtype} {tuple(dy.shape)}, x {x.dtype} {tuple(xs)}")
  cols = xs[-1]
  for t in (weight, bias):
    if t is not None and (t.dtype != torch.float32 or t.shape != (cols,)):
      raise ValueError(f"layer_norm_backward: weight and bias must be fp32 [{cols}]")
  for t in (dy, weight, bias):
    if t is not None and t.get_device() != index:
      raise ValueError(f"layer_norm_backward: tensors on {t.device} and {x.device}")
  with _on(index):
    dt = _dt(x)
    dy, x = dy.contiguous(), x.contiguous()
    weight = None if weight is None else weight.contiguous()
    rows = x.numel() // cols
    dx = torch.empty_like(x) if need_dx else None
    dw = torch.empty_like(weight) if need_dweight and weight is not None else None
    db = torch.empty_like(bias, memory_format=torch.contiguous_format) if need_dbias and bias is not None else None
    lib = N.load()
    ws = _ws(lib.sf_layernorm_backward_workspace(rows, cols), x.device)
    status = lib.sf_layernorm_backward(dt, dy.data_ptr(), x.data_ptr(), _p(weight), _p(dx), _p(dw), _p(db), rows, cols,
                                       eps, ws.data_ptr(), ws.numel(), _raw_stream(index))
    if status:
      N.check(status, "sf_layernorm_backward")
  return dx, dw, db


def _grad_table(what, grads, out=None, writes=True):
  """Host arrays (addresses, outputs, sizes, dtypes) of a list of gradients.  Each property is read by one map over
  the list: a model has hundreds of gradients and a call should not take longer here than on the device."""
  grads = list(grads)
  if not grads:
    raise ValueError(f"{what}: no gradients")
  outs = grads if out is None else list(out)
  if len(outs) != len(grads):
    raise ValueError(f"{what}: {len(outs)} outputs for {len(grads)} gradients")
  tensor = torch.Tensor
  index = grads[0].get_device()
  dts, numels = [g.dtype for g in grads], list(map(tensor.numel, grads))
  for group in (grads,) if out is None else (grads, outs):
    if index < 0 or set(map(tensor.get_device, group)) != {index}:
      raise ValueError(f"{what}: every gradient must be a CUDA tensor of one device")
    if not all(map(tensor.is_contiguous, group)):
      raise ValueError(f"{what}: gradients must be contiguous")
  if out is not None and (list(map(tensor.numel, outs)) != numels or [o.dtype for o in outs] != dts):
    raise ValueError(f"{what}: an output has another dtype or size than its gradient")
  kinds = set(dts)
  codes = {torch.float32: N.SF_F32, torch.bfloat16: N.SF_BF16}
  if not codes.keys() >= kinds:
    raise TypeError(f"{what}: unsupported dtype in {kinds}; use float32 or bfloat16")
  if len(kinds) == 1:
    dtypes = array.array("i", [codes[dts[0]]]) * len(dts)
  else:
    dtypes = array.array("i", [codes[d] for d in dts])
  ptrs = list(map(tensor.data_ptr, grads))
  optrs = ptrs if out is None else list(map(tensor.data_ptr, outs))
  if writes:   # a tensor that is there twice, or an output that is another entry's gradient, is written by two at once
    once = set(optrs)
    if len(once) != len(optrs):                       # (empty tensors may share an address)
      seen = [p for p, m in zip(optrs, numels) if m]
      if len(set(seen)) != len(seen):
        raise ValueError(f"{what}: the same tensor is in the list twice")
    if out is not None and not once.isdisjoint(ptrs):
      where = {p: i for i, p in enumerate(ptrs) if numels[i]}
      if any(numels[i] and where.get(p, i) != i for i, p in enumerate(optrs)):
        raise ValueError(f"{what}: an output is another entry's gradient")
  ptrs = array.array("Q", ptrs)                       # from lists: an iterator is read item by item
  return index, ptrs, ptrs if out is None else array.array("Q", optrs), array.array("q", numels), dtypes


def _addr(a: array.array) -> int:
  return a.buffer_info()[0]


def _norm_type(what, norm_type) -> int:
  if norm_type not in (2, float("inf")):
    raise ValueError(f"{what}: norm_type {norm_type!r} is not 2 or inf")
  return 2 if norm_type == 2 else 0


def grad_norm(grads, norm_type: float = 2.0) -> torch.Tensor:
  """The global norm (0-dim fp32, on the device) of a list of contiguous fp32 / bf16 gradients: the 2-norm, or with
  norm_type inf the largest magnitude.  Squares are summed in fp64 in a fixed order."""
  t = _norm_type("grad_norm", norm_type)
  index, ptrs, _, numels, dtypes = _grad_table("grad_norm", grads, writes=False)
  with _on(index):
    norm = torch.empty((), dtype=torch.float32, device=index)
    ws = _ws(N.load().sf_grad_norm_workspace(len(ptrs)), index)
    N.call("sf_grad_norm", _addr(ptrs), _addr(numels), _addr(dtypes), len(ptrs), t, _p(norm), _p(ws), ws.numel(),
           _raw_stream(index))
  return norm


def clip_grad_norm(grads, max_norm: float, norm_type: float = 2.0, *, out=None) -> torch.Tensor:
  """Scales the gradients by min(1, max_norm / (norm + 1e-6)) in place, or into the tensors of ``out`` (same dtypes
  and sizes; each its gradient itself or a tensor that overlaps none), and returns the norm that they had (0-dim
  fp32, on the device; nothing waits for it).  A NaN norm makes every gradient NaN.  No two gradients may overlap."""
  t = _norm_type("clip_grad_norm", norm_type)
  if not max_norm >= 0:      # NaN too
    raise ValueError(f"clip_grad_norm: max_norm {max_norm!r}")
  index, ptrs, optrs, numels, dtypes = _grad_table("clip_grad_norm", grads, out)
  with _on(index):
    norm = torch.empty((), dtype=torch.float32, device=index)
    ws = _ws(N.load().sf_grad_norm_workspace(len(ptrs)), index)
    N.call("sf_clip_grad_norm", _addr(ptrs), _addr(optrs), _addr(numels), _addr(dtypes), len(ptrs), t,
           max_norm, _p(norm), _p(ws), ws.numel(), _raw_stream(index))
  return norm
