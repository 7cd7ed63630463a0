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


def _decoder(norm, block="mlp", dtype=torch.bfloat16):
    from bibo_b200 import BiBoMLP, BiBoMoELayer, MoEConfig
    dl = torch.nn.Module()
    cfg = MoEConfig(hidden_size=256, moe_intermediate_size=128, num_routed_experts=64)
    dl.mlp = BiBoMoELayer(cfg) if block == "moe" else BiBoMLP(cfg, is_expert=True, intermediate_size=256)
    dl = dl.to(DEV).to(dtype).eval()
    dl.post_attention_layernorm = norm.to(DEV)
    return dl


@pytest.mark.parametrize("grad", [True, False])
def test_feed_forward_fires_the_hooks_of_a_layer_norm(grad):
    from bibo_b200.moe import ffn_forward
    torch.manual_seed(2)
    dl = _decoder(torch.nn.LayerNorm(256, dtype=torch.bfloat16))
    h, seen = torch.randn(2, 33, 256, device=DEV, dtype=torch.bfloat16), []
    with torch.set_grad_enabled(grad):
        want = ffn_forward(dl, h)
        dl.post_attention_layernorm.register_forward_hook(lambda m, args, out: seen.append(out.detach()))
        got = ffn_forward(dl, h)
    # the norm's results may round apart (half a step each of bf16) and pass through the same block: as in the test of the two paths
    assert len(seen) == 1 and seen[0].shape == h.shape
    got, want = got.detach().float(), want.detach().float()
    assert float((got - want).abs().max()) <= 2.0 ** -7 * float(want.abs().max())


@pytest.mark.parametrize("block", ["moe", "mlp"])
def test_feed_forward_of_a_bf16_stream_under_autocast(block):
    """The norm returns fp32 there; with and without gradients the fp32 block runs and the sum is fp32.  Both run the same kernels
    or fp32 sums of at most 256 terms in another order: 1e-4 of the largest entry."""
    from bibo_b200 import BiBoLayerNorm
    from bibo_b200.moe import ffn_forward
    torch.manual_seed(3)
    h = torch.randn(2, 33, 256, device=DEV, dtype=torch.bfloat16)
    for norm in (BiBoLayerNorm(256), torch.nn.LayerNorm(256)):
        dl = _decoder(norm, block, torch.float32)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            with torch.no_grad():
                got = ffn_forward(dl, h)
            want = ffn_forward(dl, h.clone().requires_grad_()).detach()
        assert got.dtype == want.dtype == torch.float32
        assert float((got - want).abs().max()) <= 1e-4 * float(want.abs().max())


def test_the_frameworks_router_trains_through_combine_tokens():
    """The steps at the top of bibo_b200/dispatch.py: the choice from BiBoMoERouter, its weights formed again so that they carry a
    gradient, against the same in 64 bits.  fp32 throughout: sums of at most 90 x 64 order-1 terms, 1e-4 of the largest entry."""
    import bibo_b200
    from bibo_b200 import functional
    torch.manual_seed(4)
    n, h, e, k = 90, 64, 16, 3
    router = bibo_b200.BiBoMoERouter(bibo_b200.MoEConfig(hidden_size=h, num_routed_experts=e, num_experts_per_tok=k)).to(DEV)
    torch.nn.init.normal_(router.gate_proj.weight, std=0.3)
    experts = torch.randn(e, h, h, device=DEV) / 8
    x, c = torch.randn(n, h, device=DEV), torch.randn(n, h, device=DEV)
    with torch.no_grad():
        idx, given = (t[0] for t in router(x[None]))
    score = torch.sigmoid(x.float() @ router.gate_proj.weight.float().T).gather(1, idx)
    w = score / score.sum(1, keepdim=True)
    assert float((w.detach() - given).abs().max()) <= 1e-5
    plan = functional.dispatch_plan(idx, e)
    xs = bibo_b200.dispatch_tokens(x, plan)
    off = plan.offsets.tolist()
    ys = torch.cat([xs[off[i]:off[i + 1]] @ experts[i] for i in range(e)])
    out = bibo_b200.combine_tokens(ys, w, plan)
    (out * c).sum().backward()
    plan.raise_if_failed()

    wr = router.gate_proj.weight.detach().double().requires_grad_()
    s64 = torch.sigmoid(x.double() @ wr.T).gather(1, idx)
    w64 = s64 / s64.sum(1, keepdim=True)
    out64 = sum(w64[:, j:j + 1] * torch.einsum("nh,nhi->ni", x.double(), experts.double()[idx[:, j]]) for j in range(k))
    (out64 * c.double()).sum().backward()
    for got, want in ((out.detach(), out64.detach()), (router.gate_proj.weight.grad, wr.grad)):
        assert float((got.double() - want).abs().max()) <= 1e-4 * float(want.abs().max())
    assert float(wr.grad.abs().max()) > 0


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_steps_parameters_of_every_real_type(dtype, nesterov):
    """The first step: the momentum is the gradient, u = 1.95 g or g in fp32, and the same kernel call gives the same bits."""
    import bibo_b200
    from bibo_b200 import functional
    torch.manual_seed(5)
    p = torch.nn.Parameter(torch.randn(40, 24, device=DEV).to(dtype))
    before = p.detach().clone()
    p.grad = torch.randn(40, 24, device=DEV).to(dtype)
    bibo_b200.Muon([p], lr=0.5, nesterov=nesterov).step()
    u = torch.add(p.grad, p.grad.float(), alpha=0.95).float() if nesterov else p.grad.float()
    want = before.double() - 0.5 * (40 / 24) ** 0.5 * functional.orthogonalize(u).double()
    # one sum in the parameter's type, or in fp32 on the way to it: half a step of each
    tol = (torch.finfo(dtype).eps + 2.0 ** -22) * want.abs() + 2.0 ** -20
    assert bool(((p.detach().double() - want).abs() <= tol).all())
