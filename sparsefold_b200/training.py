"""Differentiable forms of the transition's layers, for fine-tuning and gradient-based design.

Each function runs the kernels of ``ops`` forward and backward inside ``torch.autograd`` (first derivatives
only).  The weights keep either orientation: ``wt`` is [out, in], and a module's reference parameter
([in, out]) is handed over as its transpose without a copy.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from sparsefold_b200 import ops


def _match(g, dtype):
  return None if g is None else g.to(dtype)


def _differentiated(*tensors) -> bool:
  """Whether autograd will ask for a gradient of one of them.  (``ctx.needs_input_grad`` does not say so: it is true for
  parameters under ``torch.no_grad`` too.)"""
  return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


class _LinearAct(torch.autograd.Function):
  @staticmethod
  def forward(ctx, x, wt, bias, activation, gated):
    fn = ops.gated_linear if gated else ops.linear_act
    b32 = None if bias is None else bias.float()
    y, saved = fn(x, wt, b32, activation=activation, save=True)
    ctx.save_for_backward(x, wt, bias, saved)
    ctx.form = (activation, gated)
    return y

  @staticmethod
  @once_differentiable
  def backward(ctx, dy):
    x, wt, bias, saved = ctx.saved_tensors
    activation, gated = ctx.form
    need = ctx.needs_input_grad
    fn = ops.gated_linear_backward if gated else ops.linear_act_backward
    b32 = None if bias is None else bias.float()
    dx, dwt, db = fn(dy, x, wt, b32, activation=activation, saved=saved, need_dx=need[0], need_dwt=need[1],
                     need_dbias=need[2])
    return dx, dwt, _match(db, bias.dtype if bias is not None else None), None, None


class _LayerNorm(torch.autograd.Function):
  @staticmethod
  def forward(ctx, x, weight, bias, eps):
    f32 = lambda t: None if t is None else t.float().contiguous()  # noqa: E731
    ctx.save_for_backward(x, weight, bias)
    ctx.eps = eps
    return ops.layer_norm(x, f32(weight), f32(bias), eps)

  @staticmethod
  @once_differentiable
  def backward(ctx, dy):
    x, weight, bias = ctx.saved_tensors
    f32 = lambda t: None if t is None else t.float()  # noqa: E731
    need = ctx.needs_input_grad
    dx, dw, db = ops.layer_norm_backward(dy, x, f32(weight), f32(bias), ctx.eps, need_dx=need[0], need_dweight=need[1],
                                         need_dbias=need[2])
    return (dx, _match(dw, weight.dtype if weight is not None else None),
            _match(db, bias.dtype if bias is not None else None), None)


def linear_act(x, wt, bias=None, *, activation=None, residual=None):
  """Differentiable ``ops.linear_act``.  Without a gradient to compute, and where the residual is not
  differentiated, the residual is added in the kernel's epilogue; its gradient is dy otherwise too."""
  if not _differentiated(x, wt, bias, residual):
    b32 = None if bias is None else bias.float()
    return ops.linear_act(x, wt, b32, activation=activation, residual=residual)
  if residual is None:
    return _LinearAct.apply(x, wt, bias, activation, False)
  residual = residual.to(x.dtype).expand(*x.shape[:-1], wt.shape[0])
  return _LinearActResidual.apply(x, wt, bias, residual, activation)


class _LinearActResidual(torch.autograd.Function):
  @staticmethod
  def forward(ctx, x, wt, bias, residual, activation):
    b32 = None if bias is None else bias.float()
    ctx.activation = activation
    if not any(ctx.needs_input_grad[:3]):     # the residual's gradient is dy and needs nothing kept
      return ops.linear_act(x, wt, b32, activation=activation, residual=residual)
    y, saved = ops.linear_act(x, wt, b32, activation=activation, residual=residual, save=True)
    ctx.save_for_backward(x, wt, bias, saved)
    return y

  @staticmethod
  @once_differentiable
  def backward(ctx, dy):
    need = ctx.needs_input_grad
    if not any(need[:3]):
      return None, None, None, dy, None
    x, wt, bias, saved = ctx.saved_tensors
    b32 = None if bias is None else bias.float()
    dx, dwt, db = ops.linear_act_backward(dy, x, wt, b32, activation=ctx.activation, saved=saved, need_dx=need[0],
                                          need_dwt=need[1], need_dbias=need[2])
    return dx, dwt, _match(db, bias.dtype if bias is not None else None), dy if need[3] else None, None


def gated_linear(x, wt, bias=None, *, activation="silu"):
  """Differentiable ``ops.gated_linear``."""
  if not _differentiated(x, wt, bias):
    return ops.gated_linear(x, wt, None if bias is None else bias.float(), activation=activation)
  return _LinearAct.apply(x, wt, bias, activation, True)


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5):
  """Differentiable ``ops.layer_norm``; weight and bias of any float dtype (computed in fp32)."""
  return _LayerNorm.apply(x, weight, bias, eps)


def transition(x, ln_w, ln_b, w1, w2):
  """Differentiable TransitionBlock (trunk/blocks.py:79-96): x + (silu(n w1a^T) * (n w1b^T)) w2^T with
  n = LayerNorm(x); w1 [2 i, c] (gate rows first) and w2 [c, i] as ``ops.transition``, in x's dtype."""
  n = layer_norm(x, ln_w, ln_b)
  return linear_act(gated_linear(n, w1), w2, residual=x)
