"""Newton-Schulz orthogonalisation against the same steps in 64 bits.

Tolerance.  The result is a bf16 rounding (half a step: 2^-8 relative) of a value computed with f16 operands.  f16 rounds to
nearest with at most 2^-11 relative per element; with d = 2^-11 / sqrt(3) the root mean square of it, rounding a matrix M
moves it by d |M|_F in the Frobenius norm.  With F = b G + c G^2, single roundings of independent sign (so the terms add as
squares) and |.| the spectral norm, a step x' = a x + F x has
    dG = d |G|_F,   dF = d |F|_F + (|b| + 2 |c| |G|) dG,   dx' = L dx + |x| dF + d |x'|_F
where L is the slope of a s + b s^3 + c s^5 over the singular values present (at least a).  Where two steps are joined
(x'' = a1 a2 x + R x; no x' is rounded, x'' is kept in two halves):
    dT = d |T|_F + 2 (a1 + |F1|) dF1,   dG' = d |G'|_F + |T| dG + |G| dT,   dF2 = d |F2|_F + (|b2| + 2 |c2| |G'|) dG',
    dR = d |R|_F + (a1 + |F1|) dF2 + (a2 + |F2|) dF1,   dx'' = L1 L2 dx + |x| dR
dx starts at 0: a bf16 update is held exactly, an fp32 one in two halves (2^-22) in the terms "a x", while the rounding of the
other factor, d |x|_F, enters through |F| or |R|, which is added.  A factor 4 covers the tail of the distribution."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
NS = (3.4445, -4.7750, 2.0315)
D = 2.0 ** -11 / math.sqrt(3)


def _steps64(u, steps, coefficients, eps=1e-7):
    """Exact result and the root-mean-square bound on the Frobenius error of each matrix (before the bf16 rounding)."""
    x = u.double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / (x.flatten(-2).norm(dim=-1)[..., None, None] + eps)
    fro = lambda a: a.flatten(-2).norm(dim=-1)
    top = lambda a: torch.linalg.matrix_norm(a.cpu(), 2).to(DEV)
    co = [coefficients] * steps if not hasattr(coefficients[0], "__len__") else coefficients
    one = torch.eye(x.shape[-2], dtype=x.dtype, device=DEV)
    err2 = torch.zeros_like(fro(x))
    first = (D * fro(x)) ** 2 if u.dtype == torch.float32 else 0 * err2       # the rounded operand of the first product

    def polynomial(g, c):
        f = c[1] * g + c[2] * (g @ g)
        s = torch.linalg.eigvalsh(g.cpu()).to(DEV).clamp_min(0)
        return f, (c[0] + 3 * c[1] * s + 5 * c[2] * s ** 2).abs().amax(-1).clamp_min(abs(c[0]))

    k = 0
    if steps >= 3:
        (a1, b1, c1), (a2, b2, c2) = co[:2]
        g = x @ x.mT
        f1, l1 = polynomial(g, co[0])
        t = f1 @ f1 + 2 * a1 * f1
        g2 = a1 * a1 * g + t @ g
        f2, l2 = polynomial(g2, co[1])
        r = f2 @ f1 + a1 * f2 + a2 * f1
        new = (a2 * one + f2) @ ((a1 * one + f1) @ x)
        dg = (D * fro(g)) ** 2
        df1 = (D * fro(f1)) ** 2 + (abs(b1) + 2 * abs(c1) * top(g)) ** 2 * dg
        dt = (D * fro(t)) ** 2 + 4 * (a1 + top(f1)) ** 2 * df1
        dg2 = (D * fro(g2)) ** 2 + top(t) ** 2 * dg + top(g) ** 2 * dt
        df2 = (D * fro(f2)) ** 2 + (abs(b2) + 2 * abs(c2) * top(g2)) ** 2 * dg2
        dr = (D * fro(r)) ** 2 + (a1 + top(f1)) ** 2 * df2 + (a2 + top(f2)) ** 2 * df1
        err2 = top(x) ** 2 * dr + top(r) ** 2 * first
        first, x, k = (D * fro(new)) ** 2, new, 2
    for k in range(k, steps):
        g = x @ x.mT
        f, slope = polynomial(g, co[k])
        new = co[k][0] * x + f @ x
        df = (D * fro(f)) ** 2 + (abs(co[k][1]) + 2 * abs(co[k][2]) * top(g)) ** 2 * (D * fro(g)) ** 2
        err2 = slope ** 2 * err2 + top(x) ** 2 * df + top(f) ** 2 * first + (D * fro(new)) ** 2
        first, x = 0 * err2, new
    return (x.mT if tall else x), err2.sqrt()


def _check(u, steps=5, coefficients=NS, **kw):
    from bibo_b200 import functional as Fn
    got = Fn.orthogonalize(u, steps, coefficients, **kw)
    again = Fn.orthogonalize(u, steps, coefficients, **kw)
    torch.cuda.synchronize()
    assert got.dtype == torch.bfloat16 and got.shape == u.shape and got.is_contiguous() and torch.equal(got, again)
    _near(got, u, steps, coefficients, **kw)
    return got


def _near(got, u, steps=5, coefficients=NS, **kw):
    want, bound = _steps64(u, steps, coefficients, **kw)
    diff = (got.double() - want).flatten(-2).norm(dim=-1)
    tol = 4 * bound + 2.0 ** -8 * want.flatten(-2).norm(dim=-1)
    assert bool((diff <= tol).all()), (diff / want.flatten(-2).norm(dim=-1), tol / want.flatten(-2).norm(dim=-1))


def _momentum(shape, dtype, seed, rank=8, floor=0.1, scale=1e-3):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    *lead, m, n = shape
    k = min(rank, m, n)
    u = (r(*lead, m, k) / torch.arange(1, k + 1, device=DEV)) @ r(*lead, k, n) + floor * r(*lead, m, n)
    return (scale * u).to(dtype)


SHAPES = [(1, 1), (1, 7), (5, 1), (2, 3), (64, 64), (64, 2048), (2048, 64), (128, 128), (127, 129), (130, 257), (200, 72),
          (3, 65, 300), (2, 3, 100, 40), (4, 256, 512), (5, 512, 128), (2, 300, 900), (1, 640, 640), (2, 1030, 777),
          (100, 384), (100, 385), (20, 100, 500), (128, 1536), (1537, 96), (7, 3000), (2500, 128), (150, 33, 129),
          (12, 4000), (129, 4100), (4100, 140), (1, 256, 6000), (6, 700, 1100)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_matches_the_steps_in_64_bits(shape, dtype):
    _check(_momentum(shape, dtype, sum(shape)))


@pytest.mark.parametrize("steps", [1, 2, 6])
def test_step_counts_and_coefficients(steps):
    u = _momentum((3, 96, 160), torch.bfloat16, steps)
    _check(u, steps)
    _check(u, steps, (1.5, -0.5, 0.0))
    _check(u, steps, [(3.4445, -4.7750, 2.0315)] * (steps - 1) + [(1.875, -1.25, 0.375)])


@pytest.mark.parametrize("scale", [1e-12, 1.0, 1e12])
def test_scale_of_the_update_does_not_matter_beyond_eps(scale):
    u = _momentum((2, 150, 130), torch.float32, 1, scale=1.0)
    _check(scale * u, eps=0.0)
    _check(scale * u)


def test_spectra_from_orthogonal_to_rank_one():
    q = torch.linalg.qr(torch.randn(256, 192, dtype=torch.float64))[0].float().to(DEV)
    got = _check(q)
    # an orthogonal matrix: all singular values are 1/sqrt(192), so the steps leave one common value behind
    s = torch.linalg.svdvals(got.double())
    assert float(s.max() / s.min()) < 1.02
    one = torch.outer(torch.randn(300), torch.randn(200)).to(DEV)
    _check(one.bfloat16().float())
    _check(torch.ones(70, 90, device=DEV, dtype=torch.bfloat16))


def test_rows_and_matrices_of_larger_tensors():
    from bibo_b200 import functional as Fn
    for dtype in (torch.bfloat16, torch.float32):
        wide = torch.full((3, 90, 131), float("nan"), dtype=dtype, device=DEV)
        wide[:, :80, 1:126] = _momentum((3, 80, 125), dtype, 4)
        u = wide[:, :80, 1:126]
        assert torch.equal(_check(u), Fn.orthogonalize(u.contiguous()))
        assert torch.equal(Fn.orthogonalize(u[1]), Fn.orthogonalize(u.contiguous())[1])
        tall = torch.full((3, 131, 90), float("nan"), dtype=dtype, device=DEV)
        tall[:, 1:126, 3:83] = _momentum((3, 125, 80), dtype, 5)
        assert torch.equal(_check(tall[:, 1:126, 3:83]), Fn.orthogonalize(tall[:, 1:126, 3:83].contiguous()))
        large = torch.full((2, 300, 520), float("nan"), dtype=dtype, device=DEV)
        large[:, :280, 8:408] = _momentum((2, 280, 400), dtype, 6)
        _check(large[:, :280, 8:408])             # the squares are summed in another order than contiguous ones: not the same bits
        # orders that the kernels do not read: laid out first
        assert torch.equal(Fn.orthogonalize(u.mT), Fn.orthogonalize(u.mT.contiguous()))
        assert torch.equal(Fn.orthogonalize(u[0].expand(2, -1, -1)), Fn.orthogonalize(u[:1].repeat(2, 1, 1)))


def test_zero_matrices_and_empty_stacks():
    from bibo_b200 import functional as Fn
    u = _momentum((3, 100, 140), torch.float32, 9)
    u[1] = 0                                          # an expert without tokens
    got = _check(u)
    assert not bool(got[1].any())
    for shape in ((0, 5), (5, 0), (0, 4, 4), (3, 0, 4)):
        assert Fn.orthogonalize(torch.empty(shape, device=DEV)).shape == shape
    u[2, 0, 0] = float("nan")
    got = Fn.orthogonalize(u)
    assert bool(got[2].isnan().all()) and bool(got[0].isfinite().all()) and not bool(got[1].any())


def test_many_matrices():
    """Many small ones, and more larger ones than a workspace holds at once."""
    from bibo_b200 import _lib
    from bibo_b200 import functional as Fn
    u = _momentum((33000, 8, 16), torch.bfloat16, 2)
    got = Fn.orthogonalize(u)
    for i in (0, 1, 16383, 16384, 32767, 32768, 32999):
        assert torch.equal(got[i], Fn.orthogonalize(u[i]))
    _check(u[32760:32776].clone())
    size = _lib.load().bibo_moe_orthogonalize_workspace
    assert size(320, 640, 1024) == size(10000, 640, 1024) > 1 << 30       # a group of fewer than 320
    u = _momentum((320, 640, 1024), torch.bfloat16, 3)
    got = Fn.orthogonalize(u)
    which = [0, 150, 297, 298, 299, 300, 319]
    _near(got[which], u[which])                       # one matrix alone is summed in another order: not the same bits


def test_two_graphs_and_streams_do_not_share_a_workspace():
    from bibo_b200 import functional as Fn
    a, b = _momentum((2, 200, 260), torch.bfloat16, 1), _momentum((2, 200, 260), torch.bfloat16, 2)
    want = [Fn.orthogonalize(a), Fn.orthogonalize(b)]
    graphs = []
    for u in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = Fn.orthogonalize(u)
        graphs.append((graph, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    for s, (graph, _) in zip(streams, graphs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, w) for (_, out), w in zip(graphs, want))
    new = _momentum((2, 200, 260), torch.bfloat16, 3)
    a.copy_(new)
    graphs[0][0].replay()
    assert torch.equal(graphs[0][1], Fn.orthogonalize(new))


def test_calls_on_two_streams_at_once():
    from bibo_b200 import functional as Fn
    us = [_momentum(shape, torch.bfloat16, 7 + i) for i, shape in enumerate([(1, 520, 600), (4, 300, 700), (3, 64, 900), (1, 200, 3400)])]
    want = [Fn.orthogonalize(u) for u in us]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for s, out in zip(streams, got):
            with torch.cuda.stream(s):
                out.append([Fn.orthogonalize(u) for u in us])
    torch.cuda.synchronize()
    for out in got:
        for run in out:
            assert all(torch.equal(a, b) for a, b in zip(run, want))


def test_muon_step_on_the_blocks_parameters():
    """The optimiser's step against its formula in 64 bits, on the gradients that the block's own backward produced."""
    import bibo_b200
    from bibo_b200 import functional as Fn
    torch.manual_seed(0)
    layer = bibo_b200.BiBoMoELayer(bibo_b200.MoEConfig(hidden_size=128, moe_intermediate_size=64, num_routed_experts=8,
                                                       num_experts_per_tok=2)).to(DEV).train()
    matrices = [p for p in layer.parameters() if p.requires_grad and p.dim() >= 2]
    assert len(matrices) == 3
    opt = bibo_b200.Muon(matrices, lr=0.03, weight_decay=0.1)
    buf = [torch.zeros_like(p, dtype=torch.float64) for p in matrices]
    for _ in range(2):
        opt.zero_grad()
        layer(torch.randn(2, 64, 128, device=DEV)).square().mean().backward()
        before = [p.detach().double().clone() for p in matrices]
        opt.step()
        for p, w, v in zip(matrices, before, buf):
            g = p.grad.double()
            v.mul_(0.95).add_(g)
            u = (g + 0.95 * v).float()
            scale = 0.03 * max(1.0, p.shape[-2] / p.shape[-1]) ** 0.5
            want = w * (1 - 0.03 * 0.1) - scale * Fn.orthogonalize(u).double()
            # The optimiser's momentum is fp32 and may differ from v by a rounding, so that f16 values near a tie round the
            # other way: elements cannot be compared, matrices can.  Both results are within 4 bound + 2^-8 |x|_F of the
            # exact steps of their inputs (see above), the inputs are at most 3 * 2^-24 apart, relative to their norm, which
            # five steps of slope a stretch to 3.4445^5 * 3 * 2^-24 < 1e-4, and the parameter takes three fp32 roundings.
            exact, bound = _steps64(u, 5, NS)
            fro = lambda t: t.flatten(-2).norm(dim=-1)
            tol = scale * (2 * (4 * bound + 2.0 ** -8 * fro(exact)) + 1e-4) + 4 * 2.0 ** -24 * fro(w)
            assert bool((fro(p.detach().double() - want) <= tol).all())


def test_training_step_with_the_callers_own_experts():
    """Layer norm -> router -> dispatch -> the caller's experts -> combine, backward and the orthogonalised update, against
    the same step in plain 64-bit torch on the same routing."""
    import bibo_b200
    from bibo_b200 import functional as Fn
    torch.manual_seed(5)
    n, h, e, k, inter = 150, 64, 8, 2, 48
    norm = bibo_b200.BiBoLayerNorm(h).to(DEV)
    router = bibo_b200.BiBoMoERouter(bibo_b200.MoEConfig(hidden_size=h, num_routed_experts=e, num_experts_per_tok=k)).to(DEV)
    w1 = torch.nn.Parameter(0.1 * torch.randn(e, inter, h, device=DEV))
    w2 = torch.nn.Parameter(0.1 * torch.randn(e, h, inter, device=DEV))
    x = torch.randn(1, n, h, device=DEV)
    c = torch.randn(n, h, device=DEV)

    z = norm(x)
    with torch.no_grad():
        idx, weight = router(z.detach())
    weight = weight[0].clone().requires_grad_()
    plan = Fn.dispatch_plan(idx[0], e)
    xs = bibo_b200.dispatch_tokens(z[0], plan)
    off = plan.offsets.tolist()
    ys = torch.cat([torch.relu(xs[off[i]:off[i + 1]] @ w1[i].T) @ w2[i].T for i in range(e)])
    out = bibo_b200.combine_tokens(ys, weight, plan)
    (out * c).sum().backward()

    p = {name: t.detach().double().requires_grad_() for name, t in
         dict(nw=norm.weight, nb=norm.bias, w1=w1, w2=w2, weight=weight).items()}
    xd = x[0].double()
    mu = xd.mean(1, keepdim=True)
    zd = (xd - mu) / torch.sqrt(((xd - mu) ** 2).mean(1, keepdim=True) + norm.eps) * p["nw"] + p["nb"]
    outd = torch.zeros(n, h, dtype=torch.float64, device=DEV)
    for j in range(k):
        y = torch.relu(torch.einsum("nh,nih->ni", zd, p["w1"][idx[0, :, j]]))
        outd = outd + p["weight"][:, j:j + 1] * torch.einsum("ni,nhi->nh", y, p["w2"][idx[0, :, j]])
    (outd * c.double()).sum().backward()
    # fp32 throughout (the experts' products are torch's): sums of at most 150 x 64 order-1 terms, 1e-4 of the largest entry
    for got, want in ((norm.weight.grad, p["nw"].grad), (norm.bias.grad, p["nb"].grad), (w1.grad, p["w1"].grad),
                      (w2.grad, p["w2"].grad), (weight.grad, p["weight"].grad), (out.detach(), outd.detach())):
        assert float((got.double() - want).abs().max()) <= 1e-4 * float(want.abs().max())
    for q in (w1, w2):
        _check(q.grad)
    opt = bibo_b200.Muon([w1, w2], lr=0.1)
    before = w1.detach().clone()
    opt.step()
    # the first step's update is (1 + momentum) g, whose orthogonal factor is g's; m = 48 < n = 64: no extra scale
    step = (before - w1.detach()).double() / 0.1
    want, bound = _steps64(w1.grad.float(), 5, NS)
    size = want.flatten(-2).norm(dim=-1)
    assert bool(((step - want).flatten(-2).norm(dim=-1) <= 4 * bound + (2.0 ** -8 + 1e-4) * size).all())


def test_muon_refuses_to_capture_its_first_step():
    import bibo_b200
    p = torch.nn.Parameter(torch.randn(64, 96, device=DEV))
    p.grad = torch.randn_like(p)
    opt = bibo_b200.Muon([p])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="before a step is captured"):
            opt.step()
        unused = p.detach() + 1                                        # the capture itself is whole
    opt.step()
    start, buf = p.detach().clone(), opt.state[p]["momentum_buffer"].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(2):
        graph.replay()
    got, got_buf = p.detach().clone(), opt.state[p]["momentum_buffer"].clone()
    with torch.no_grad():
        p.copy_(start)
        opt.state[p]["momentum_buffer"].copy_(buf)
    for _ in range(2):
        opt.step()
    assert torch.equal(got, p.detach()) and torch.equal(got_buf, opt.state[p]["momentum_buffer"])
