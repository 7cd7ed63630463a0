"""Where the operators beside the block meet torch's modules, modes and the framework's own router."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layer_norm_module_under_autocast_is_torchs(dtype):
    """Types and values of result and gradients.  Both compute in fp32 from the same values: sums of 72 (of 5 rows for the
    parameters) order-1 terms, 1e-5 of the largest entry; gradients arrive in the inputs' types, half a step of which is added."""
    import bibo_b200
    torch.manual_seed(0)
    mine, theirs = bibo_b200.BiBoLayerNorm(72).to(DEV, dtype), torch.nn.LayerNorm(72).to(DEV, dtype)
    with torch.no_grad():
        for a, b in zip(mine.parameters(), theirs.parameters()):
            a.copy_(torch.randn(72))
            b.copy_(a)
    x, dy = torch.randn(5, 72, device=DEV, dtype=dtype), torch.randn(5, 72, device=DEV)
    results = []
    for norm in (mine, theirs):
        leaf = x.clone().requires_grad_()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            out = norm(leaf)
            with torch.no_grad():
                assert norm(leaf).dtype == torch.float32
        out.backward(dy)
        results.append((out.detach(), leaf.grad, norm.weight.grad, norm.bias.grad))
    for got, want in zip(*results):
        assert got.dtype == want.dtype
        tol = 1e-5 * float(want.abs().max()) + torch.finfo(want.dtype).eps * want.double().abs()     # two roundings, half a step each
        assert bool(((got.double() - want.double()).abs() <= tol).all())
    assert results[0][0].dtype == torch.float32 and results[0][1].dtype == dtype
