"""The weights' gradients of combine on terms whose roundings all point the same way."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_long_sums_of_the_weights_gradient_are_cut_into_parts():
    """16384 equal positive terms per slot, a warp per token, so 512 a lane.  Added one by one, a term of 1 + 2^-16 - 2^-23 loses
    nearly half a step in each of the last 256 additions: 128 * 2^-24 of the sum.  In parts of an access (4 terms), with u = 2^-24: an
    addition rounds by at most u times its result, the 128 partial sums of a lane average half of its sum, so 64.5 u of it, 4 u
    for the parts, 5 u for the lanes: 74 u."""
    from bibo_b200 import functional as Fn
    n, h = 32 * torch.cuda.get_device_properties(0).multi_processor_count, 16384
    c = 1.0 + 2.0 ** -16 - 2.0 ** -23
    plan = Fn.dispatch_plan(torch.zeros(n, 1, dtype=torch.int32, device=DEV), 1)
    dout = torch.ones(n, h, device=DEV)
    ys = torch.full((plan.rows, h), c, device=DEV)
    dys, dw = Fn.combine_backward(dout, ys, torch.ones(n, 1, device=DEV), plan)
    assert float((dw.double() - h * c).abs().max()) <= 74 * 2.0 ** -24 * h * c
    assert torch.equal(dys, dout)
