"""Expert-order dispatch and combine against plain indexing in 64 bits.

Tolerances: u = 2^-24; a sum of n products in fp32 is off by at most (n + 1) u times the sum of the absolute values (for the
dot products no chain is longer than H/32 + 16); a stored value by half a step of its type more.  Copies are exact."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
BF, FP = torch.bfloat16, torch.float32


def _half(t):
    return torch.finfo(t).eps / 2


def _plan_reference(idx, experts, align):
    """slot_row, offsets and counts by counting, slot by slot."""
    flat = idx.reshape(-1).tolist()
    counts = [0] * experts
    for e in flat:
        if 0 <= e < experts:
            counts[e] += 1
    offsets = [0]
    for c in counts:
        offsets.append(offsets[-1] + -(-c // align) * align)
    at, rows = list(offsets), []
    for e in flat:
        if 0 <= e < experts:
            rows.append(at[e])
            at[e] += 1
        else:
            rows.append(-1)
    return torch.tensor(rows).view(idx.shape), torch.tensor(offsets), torch.tensor(counts)


def _idx(n, k, experts, empty, seed, dtype=torch.int32, skew=0.0):
    g = torch.Generator().manual_seed(seed)
    p = 1.0 / (1 + torch.arange(experts).float()) ** skew
    idx = torch.multinomial(p.expand(max(n, 1), -1), k, replacement=k > experts, generator=g)[:n]
    idx = torch.where(torch.rand(n, k, generator=g) < empty, -1 - torch.randint(0, 5, (n, k), generator=g), idx)
    return idx.to(dtype)


def _check_plan(plan, idx, experts, align):
    rows, offsets, counts = _plan_reference(idx, experts, align)
    assert torch.equal(plan.slot_row.cpu().long(), rows)
    assert torch.equal(plan.offsets.cpu().long(), offsets) and torch.equal(plan.counts.cpu().long(), counts)
    inverse = torch.full((plan.rows,), -1)
    used = rows.reshape(-1) >= 0
    inverse[rows.reshape(-1)[used]] = used.nonzero()[:, 0]
    assert torch.equal(plan.row_slot.cpu().long(), inverse)
    plan.raise_if_failed()
    return rows.to(DEV)


CASES = [  # tokens, hidden, k, experts, empty, align, skew
    (1, 2048, 6, 64, 0.0, 1, 0.0), (1, 1, 1, 1, 0.0, 1, 0.0), (2, 5, 3, 2, 0.0, 4, 0.0), (8, 2048, 6, 64, 0.0, 128, 0.0),
    (33, 96, 8, 256, 0.5, 1, 1.0), (129, 1153, 3, 40, 0.3, 1, 1.0), (700, 258, 4, 64, 1.0, 16, 0.0),
    (1000, 640, 6, 64, 0.875, 128, 2.0), (2500, 72, 12, 9, 0.1, 7, 0.5), (65, 4100, 32, 1024, 0.0, 1, 0.0),
    (30000, 24, 6, 64, 0.0, 1, 0.0), (9001, 40, 1, 3, 0.2, 1024, 1.0)]


@pytest.mark.parametrize("n,h,k,e,empty,align,skew", CASES)
@pytest.mark.parametrize("dtype", [BF, FP])
def test_all_four_directions(n, h, k, e, empty, align, skew, dtype):
    from bibo_b200 import functional as Fn
    g = torch.Generator(device=DEV).manual_seed(n + h)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    idx = _idx(n, k, e, empty, n * 3 + k, torch.int64 if n % 2 else torch.int32, skew)
    plan = Fn.dispatch_plan(idx.to(DEV), e, align)
    rows = _check_plan(plan, idx, e, align)
    flat = rows.reshape(-1)
    used = flat >= 0
    token = torch.arange(n, device=DEV).repeat_interleave(k)
    x = r(n, h).to(dtype)
    xs = Fn.dispatch_forward(x, plan)
    want = torch.zeros(plan.rows, h, dtype=dtype, device=DEV)
    want[flat[used]] = x[token[used]]
    assert torch.equal(xs, want)

    ys, dout, dxs = r(plan.rows, h).to(dtype), r(n, h).to(dtype), r(plan.rows, h).to(dtype)
    free = torch.ones(plan.rows, dtype=torch.bool, device=DEV)
    free[flat[used]] = False
    ys[free], dxs[free] = float("nan"), float("inf")            # rows without a slot and weights of empty slots are not read
    for wtype in (FP, BF):
        w = torch.rand(n, k, generator=g, device=DEV).to(wtype)
        w[rows < 0] = float("nan")
        out = Fn.combine_forward(ys, w, plan)
        dys, dw = Fn.combine_backward(dout, ys, w, plan)
        assert torch.equal(out, Fn.combine_forward(ys, w, plan))
        W = torch.where(rows >= 0, w.double(), 0.0)
        Y = torch.where((rows >= 0)[:, :, None], ys.double()[rows.clamp_min(0)], 0.0)
        want = (W[:, :, None] * Y).sum(1)
        tol = (k + 1) * U * (W[:, :, None] * Y).abs().sum(1) + 1.01 * _half(dtype) * want.abs()
        assert bool(((out.double() - want).abs() <= tol).all())
        G = dout.double()
        want = (Y * G[:, None]).sum(2)
        tol = (h / 32 + 16) * U * (Y * G[:, None]).abs().sum(2) + 1.01 * _half(wtype) * want.abs()
        assert dw.dtype == wtype and bool(((dw.double() - want).abs() <= tol).all()) and not bool(dw[rows < 0].any())
        want = torch.zeros(plan.rows, h, dtype=torch.float64, device=DEV)
        want[flat[used]] = (W[:, :, None] * G[:, None]).reshape(-1, h)[used]
        assert bool(((dys.double() - want).abs() <= 1.01 * (_half(dtype) + U) * want.abs()).all())
        assert not bool(dys[free].any())
    dx = Fn.dispatch_backward(dxs, plan)
    D = torch.where((rows >= 0)[:, :, None], dxs.double()[rows.clamp_min(0)], 0.0)
    want = D.sum(1)
    assert bool(((dx.double() - want).abs() <= (k + 1) * U * D.abs().sum(1) + 1.01 * _half(dtype) * want.abs()).all())


@pytest.mark.parametrize("n,k,e", [(1024, 8, 64), (1025, 8, 64), (32768, 6, 64), (16384, 8, 256), (70000, 2, 1000)])
def test_plan_at_the_block_and_cluster_sizes(n, k, e):
    from bibo_b200 import functional as Fn
    idx = _idx(n, k, e, 0.1, n, skew=1.0)
    _check_plan(Fn.dispatch_plan(idx.to(DEV), e, 1), idx, e, 1)
    same = torch.full((n, k), e - 1, dtype=torch.int64)              # every slot on one expert, the same one k times a token
    _check_plan(Fn.dispatch_plan(same.to(DEV), e, 128), same, e, 128)


def test_offsets_beyond_32_bits():
    """Expert-ordered rows of more than 2^31 elements (and 2^32 bytes): the last rows are where they should be."""
    from bibo_b200 import functional as Fn
    n, k, e, h = 34000, 8, 16, 8192
    idx = torch.arange(k, device=DEV, dtype=torch.int32).expand(n, k) * 2
    plan = Fn.dispatch_plan(idx.contiguous(), e)
    assert plan.rows * h > 1 << 31
    x = torch.randn(n, h, device=DEV).to(BF)
    xs = Fn.dispatch_forward(x, plan)
    for j in (0, k - 1):                                           # expert 2j holds all tokens in order
        assert torch.equal(xs[j * n:(j + 1) * n], x)
    w = torch.rand(n, k, device=DEV)
    out = Fn.combine_forward(xs, w, plan)
    t = torch.tensor([0, 1, n // 2, n - 1], device=DEV)
    want = x[t].double() * w[t].double().sum(1, keepdim=True)
    assert bool(((out[t].double() - want).abs() <= ((k + 1) * U + 1.01 * _half(BF)) * want.abs()).all())
    dys, dw = Fn.combine_backward(x, xs, w, plan)
    want = w[t, k - 1].double()[:, None] * x[t].double()
    assert bool(((dys[(k - 1) * n + t].double() - want).abs() <= 1.01 * (_half(BF) + U) * want.abs()).all())
    sq = x[t].double().square().sum(1)
    assert bool(((dw[t, k - 1].double() - sq).abs() <= (h / 32 + 16) * U * sq).all())


def test_no_tokens_and_out_of_range_indices():
    from bibo_b200 import functional as Fn
    plan = Fn.dispatch_plan(torch.empty(0, 4, dtype=torch.int64, device=DEV), 8, 16)
    assert plan.rows == 0 and plan.offsets.tolist() == [0] * 9
    x = torch.empty(0, 32, device=DEV)
    assert Fn.dispatch_forward(x, plan).shape == (0, 32) and Fn.combine_forward(x, None, plan).shape == (0, 32)
    dys, dw = Fn.combine_backward(x, x, torch.empty(0, 4, device=DEV), plan)
    assert dys.shape == (0, 32) and dw.shape == (0, 4)
    # an index of 8 or 2^32 + 1 is out of range for 8 experts: an empty slot, and a status
    idx = torch.tensor([[0, 7], [8, 1], [2 ** 32 + 1, -2 ** 40]], device=DEV)
    plan = Fn.dispatch_plan(idx, 8)
    assert plan.slot_row.tolist() == [[0, 2], [-1, 1], [-1, -1]]
    with pytest.raises(RuntimeError, match="out of range"):
        plan.raise_if_failed()


def test_strided_rows_and_gradients():
    """x and dout as slices of wider tensors, at every alignment."""
    from bibo_b200 import functional as Fn
    idx = _idx(50, 3, 8, 0.2, 1).to(DEV)
    plan = Fn.dispatch_plan(idx, 8)
    for dtype in (BF, FP):
        for h, pad in ((64, 8), (64, 3), (33, 1), (62, 2)):
            wide = torch.randn(50, h + pad, device=DEV).to(dtype)
            x = wide[:, :h]
            assert torch.equal(Fn.dispatch_forward(x, plan), Fn.dispatch_forward(x.contiguous(), plan))
            ys, w = torch.randn(plan.rows, h, device=DEV).to(dtype), torch.rand(50, 3, device=DEV)
            a, b = Fn.combine_backward(x, ys, w, plan), Fn.combine_backward(x.contiguous(), ys, w, plan)
            # the access width changes the order of the dot product's sum, nothing else
            assert torch.equal(a[0], b[0]) and torch.allclose(a[1], b[1], rtol=0, atol=4 * (h + 16) * U * 16)


def test_autograd_matches_the_formula_and_differences():
    import bibo_b200
    from bibo_b200 import functional as Fn
    torch.manual_seed(0)
    n, k, e, h = 19, 3, 5, 12
    idx = _idx(n, k, e, 0.2, 4).to(DEV)
    plan = Fn.dispatch_plan(idx, e, 4)
    x = torch.randn(n, h, device=DEV, requires_grad=True)
    w = torch.rand(n, k, device=DEV, requires_grad=True)
    scale = torch.randn(e, h, device=DEV)
    c = torch.randn(n, h, device=DEV)
    expert = torch.zeros(plan.rows, dtype=torch.long, device=DEV)
    off = plan.offsets.tolist()
    for i in range(e):
        expert[off[i]:off[i + 1]] = i
    xs = bibo_b200.dispatch_tokens(x, plan)
    out = bibo_b200.combine_tokens(torch.tanh(xs * scale[expert]), w, plan)
    (out * c).sum().backward()

    def f(xx, ww):
        total = torch.zeros((), dtype=torch.float64, device=DEV)
        for j in range(k):
            ok = (idx[:, j] >= 0).double()[:, None]
            y = torch.tanh(xx * scale.double()[idx[:, j].clamp_min(0)])
            total = total + (ok * ww[:, j:j + 1] * y * c.double()).sum()
        return total

    args = [x.detach().double().requires_grad_(), w.detach().double().requires_grad_()]
    f(*args).backward()
    # fp32 against 64 bits: three roundings and a tanh on order-1 values, summed over k
    assert torch.allclose(x.grad.double(), args[0].grad, rtol=1e-5, atol=1e-5)
    assert torch.allclose(w.grad.double(), args[1].grad, rtol=1e-5, atol=1e-5)
    for i, grad in enumerate((x.grad, w.grad)):
        d = torch.randn_like(args[i])
        step = [a.detach() for a in args]
        lo, hi = list(step), list(step)
        lo[i], hi[i] = step[i] - 1e-5 * d, step[i] + 1e-5 * d
        slope = float((f(*hi) - f(*lo)) / 2e-5)
        assert abs(float((grad.double() * d).sum()) - slope) < 1e-4 * max(1.0, abs(slope))
    # weights that need no gradient, and a gradient that arrives expanded
    xs = bibo_b200.dispatch_tokens(x, plan)
    x.grad = None
    bibo_b200.combine_tokens(xs, None, plan).sum().backward()
    assert torch.equal(x.grad, (idx >= 0).sum(1, keepdim=True).float().expand(n, h))


def test_router_to_combine_equals_the_blocks_own_permute_and_combine():
    """The same routing through this pair and through the block's stages: rows of an expert hold the same tokens in the
    same order."""
    from bibo_b200 import BiBoMoERouter, MoEConfig
    from bibo_b200 import functional as Fn
    torch.manual_seed(3)
    router = BiBoMoERouter(MoEConfig(hidden_size=256)).to(DEV).to(BF)
    router.bias.data = router.bias.data.float()
    x = torch.randn(1, 300, 256, device=DEV).to(BF)
    idx, w = router(x)
    plan = Fn.dispatch_plan(idx[0], 64, align=128)
    xs = Fn.dispatch_forward(x[0], plan)
    wr = torch.randn(64, 256, 256, device=DEV).to(BF)
    gate_up, down, theta = wr, torch.randn(64, 256, 128, device=DEV).to(BF), torch.zeros(64, device=DEV)
    out, ws = Fn.experts_forward(x[0], idx[0], w[0], gate_up, down, theta, 64)
    torch.cuda.synchronize()
    assert torch.equal(ws.counts(), plan.counts)
    assert torch.equal(ws.slot_row, plan.slot_row)                # the block pads to 128 rows as well
    used = (plan.row_slot >= 0).nonzero()[:, 0]
    assert torch.equal(xs[used], ws.xp[used])
    ys = torch.zeros(plan.rows, 256, dtype=BF, device=DEV)
    ys[used] = ws.y[used]
    assert torch.equal(Fn.combine_forward(ys, w[0].contiguous(), plan), out)


def test_capture_replays_a_new_routing_and_streams():
    from bibo_b200 import functional as Fn
    n, h, k, e = 200, 128, 4, 16
    idx = _idx(n, k, e, 0.1, 1).to(DEV)
    x, w = torch.randn(n, h, device=DEV), torch.rand(n, k, device=DEV)
    Fn.combine_forward(Fn.dispatch_forward(x, Fn.dispatch_plan(idx, e)), w, Fn.dispatch_plan(idx, e))
    graphs = []
    for _ in range(2):                                            # two captured graphs over the same inputs
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan = Fn.dispatch_plan(idx, e)
            xs = Fn.dispatch_forward(x, plan)
            out = Fn.combine_forward(xs, w, plan)
        graphs.append((graph, plan, xs, out))
    new = _idx(n, k, e, 0.3, 2).to(DEV)
    idx.copy_(new)
    for graph, *_ in graphs:
        graph.replay()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        p2 = Fn.dispatch_plan(new, e)
        xs2 = Fn.dispatch_forward(x, p2)
        out2 = Fn.combine_forward(xs2, w, p2)
    torch.cuda.synchronize()
    for _, plan, xs, out in graphs:
        assert torch.equal(plan.slot_row, p2.slot_row) and torch.equal(xs, xs2) and torch.equal(out, out2)
