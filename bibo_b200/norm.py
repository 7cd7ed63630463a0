"""Layer norm on the kernels of ``bibo_moe_layernorm_fwd`` / ``_bwd``.

``BiBoLayerNorm`` is ``torch.nn.LayerNorm`` over the last dimension (same constructor, parameters, state dict and type under
autocast: fp32) with its forward and backward on those kernels; ``layer_norm`` keeps its input's type under autocast too.
``bibo_b200.moe.ffn_forward`` takes a decoder layer whose norm is a layer norm.
"""
from __future__ import annotations

import torch
import torch.nn as nn
from torch.autograd.forward_ad import unpack_dual
from torch.autograd.function import once_differentiable

from . import functional as Fn

__all__ = ["BiBoLayerNorm", "layer_norm"]


class _LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        out, saved = Fn.layernorm_forward(x, weight, bias, eps, keep=True)
        ctx.save_for_backward(x, weight, saved[0])
        ctx.wtype, ctx.has_bias = saved[1], bias is not None
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        # the weight itself is read either way; its gradient and the bias's cost a pass of their own only when asked for
        dx, dw, db = Fn.layernorm_backward(dy.contiguous(), x, weight, (stats, ctx.wtype), ctx.has_bias and need_b, need_w)
        return dx if need_x else None, dw, db, None


def layer_norm(x: torch.Tensor, weight=None, bias=None, eps: float = 1e-5) -> torch.Tensor:
    """Differentiable layer norm of x [..., H] over H; ``weight`` / ``bias`` [H] are optional, fp32 or of x's dtype.  Reverse mode
    only: inputs with a forward-mode tangent are refused."""
    if x.dim() < 1:
        raise RuntimeError("layer_norm takes a tensor of at least one dimension")
    # without a reverse-mode gradient no autograd function stands between the tangent and the kernel, which would drop it
    if any(t is not None and unpack_dual(t).tangent is not None for t in (x, weight, bias)):
        raise NotImplementedError("bibo_b200: layer_norm has no forward-mode derivative")
    rows = x.reshape(-1, x.shape[-1])
    if rows.shape[1] > 1 and rows.stride(1) != 1 or rows.shape[0] > 1 and rows.stride(0) < rows.shape[1]:
        rows = rows.contiguous()
    grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias))
    out = _LayerNormFunction.apply(rows, weight, bias, eps) if grad else Fn.layernorm_forward(rows, weight, bias, eps)
    return out.view(x.shape)


def layer_norm_module_forward(norm: nn.LayerNorm, x: torch.Tensor) -> torch.Tensor:
    """``torch.nn.LayerNorm.forward`` over the last dimension on the kernels."""
    if len(norm.normalized_shape) != 1 or norm.normalized_shape[0] != x.shape[-1]:
        raise RuntimeError(f"the layer norm kernels normalise the last dimension: normalized_shape {norm.normalized_shape} "
                           f"for an input of {tuple(x.shape)}")
    weight, bias = norm.weight, norm.bias
    if torch.is_autocast_enabled("cuda"):           # as torch's: computed and returned in fp32
        x, weight, bias = (t if t is None or t.dtype == torch.float64 else t.float() for t in (x, weight, bias))
    return layer_norm(x, weight, bias, norm.eps)


class BiBoLayerNorm(nn.LayerNorm):
    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm_module_forward(self, x)
