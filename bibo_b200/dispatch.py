"""Differentiable token dispatch and combine for experts that are not this package's own.

    with torch.no_grad():                                  # x [N,H]; the choice of experts has no gradient ...
        idx = router(x[None])[0][0]                        # a BiBoMoERouter; its weights, the second result, have none either
    score = torch.sigmoid(x.float() @ router.gate_proj.weight.float().T).gather(1, idx)
    w = score / score.sum(1, keepdim=True)                 # ... so the weights [N,k] are formed again where the router trains
    plan = functional.dispatch_plan(idx, n_experts)        # rows of expert e: [plan.offsets[e], plan.offsets[e+1])
    xs = dispatch_tokens(x, plan)                          # [plan.rows, H] in expert order
    ys = my_experts(xs, plan.offsets)                      # any row-wise function of xs
    out = combine_tokens(ys, w, plan)                      # [N,H], gradients to ys and w

Gradients end at the ``w`` that is passed: the routers of this package return weights without a gradient (``BiBoMoELayer`` trains its
router inside the block's own backward), so a router trains through ``combine_tokens`` only if its weights are computed
differentiably, as above.  An index beyond the experts counts as an empty slot, in both directions, and is reported by
``plan.raise_if_failed()`` alone, which waits for the plan.

The gradients are the kernels of ``bibo_b200.functional``: sums over a token's slots run in a fixed order.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import functional as Fn

__all__ = ["dispatch_tokens", "combine_tokens"]


class _DispatchFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, plan):
        ctx.plan = plan
        return Fn.dispatch_forward(x, plan)

    @staticmethod
    @once_differentiable
    def backward(ctx, dxs):
        return Fn.dispatch_backward(dxs.contiguous(), ctx.plan), None


class _CombineFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ys, topk_w, plan):
        ctx.plan = plan
        ctx.save_for_backward(ys, topk_w)
        return Fn.combine_forward(ys, topk_w, plan)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        ys, topk_w = ctx.saved_tensors
        dys, dw = Fn.combine_backward(dout.contiguous(), ys, topk_w, ctx.plan, need_dw=ctx.needs_input_grad[1])
        return dys, dw, None


def dispatch_tokens(x: torch.Tensor, plan: Fn.DispatchPlan) -> torch.Tensor:
    """xs [plan.rows, H]: the rows of x [N,H] in the plan's expert order, zero where a row has no slot."""
    return _DispatchFunction.apply(x, plan)


def combine_tokens(ys: torch.Tensor, topk_w: Optional[torch.Tensor], plan: Fn.DispatchPlan) -> torch.Tensor:
    """out [N,H]: each token's rows of ys [plan.rows, H] summed with its weights topk_w [N,k] (None: plain sum).  The gradient of
    ``topk_w`` goes where autograd finds its history; weights straight from ``BiBoMoERouter`` have none."""
    return _CombineFunction.apply(ys, topk_w, plan)
