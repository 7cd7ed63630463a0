"""Layer norm kernels against the formula in 64 bits, element by element.

Tolerances: u = 2^-24 is half a step of fp32.  A sum of H terms of which no chain is longer than H/32 + 32 additions is off
by at most (H/32 + 32) u times the sum of the absolute values; the rest follows the formula term by term; the last rounding
adds half a step of the output's type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def _inputs(n, h, dtype, wtype, bias, pad, seed, offset=0.5):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    wide = torch.full((n, h + pad), float("nan"), dtype=dtype)
    wide[:, :h] = (r(n, h) + offset * r(h)).to(dtype)
    gwide = torch.full((n, h + pad), float("nan"), dtype=dtype)
    gwide[:, :h] = r(n, h).to(dtype)
    w = (1 + 0.3 * r(h)).to(wtype).to(DEV) if wtype is not None else None
    b = (0.3 * r(h)).to(wtype or dtype).to(DEV) if bias else None
    return wide.to(DEV)[:, :h], gwide.to(DEV)[:, :h], w, b


def _half(t):
    return torch.finfo(t).eps / 2


def _check(got, want, tol, what):
    got = got.double()
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), (what, int(bad.sum()), float((got - want).abs().max()), float((got - want).abs().max() / tol.max()))


def _compare(x, dy, w, b, eps):
    from bibo_b200 import functional as Fn
    n, h = x.shape
    y, saved = Fn.layernorm_forward(x, w, b, eps, keep=True)
    plain = Fn.layernorm_forward(x, w, b, eps)
    dx, dw, db = Fn.layernorm_backward(dy, x, w, saved, has_bias=b is not None)
    again = Fn.layernorm_backward(dy, x, w, saved, has_bias=b is not None)
    torch.cuda.synchronize()
    assert torch.equal(y, plain) and torch.equal(dx, again[0])
    assert y.dtype == dx.dtype == x.dtype and (dw is None) == (w is None) and (db is None) == (b is None)
    X, G = x.double(), dy.double()
    W = w.double() if w is not None else torch.ones(h, dtype=torch.float64, device=DEV)
    B = b.double() if b is not None else torch.zeros(h, dtype=torch.float64, device=DEV)
    ops = (h / 32 + 32) * U
    mean = X.mean(1, keepdim=True)
    var = ((X - mean) ** 2).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    z = (X - mean) * rstd
    d_mean = ops * X.abs().mean(1, keepdim=True)
    # var is off by its sum's rounding and by the square of the mean's error; half of that, relatively, reaches rstd
    # (rsqrtf itself: 2 steps of fp32); eps is fp32
    d_rstd = rstd * (0.5 * (2 * ops * var + d_mean ** 2 + U * eps) / (var + eps) + 6 * U)
    d_z = rstd * (d_mean + 2 * U * (X.abs() + mean.abs())) + (X - mean).abs() * d_rstd + 2 * U * z.abs()
    want = z * W + B
    _check(y, want, W.abs() * d_z + 3 * U * ((z * W).abs() + B.abs()) + _half(x.dtype) * 1.01 * want.abs(), "y")
    g = G * W
    m0, m1 = g.mean(1, keepdim=True), (g * z).mean(1, keepdim=True)
    d_m0 = (ops + 2 * U) * g.abs().mean(1, keepdim=True)
    d_m1 = (ops + 4 * U) * (g * z).abs().mean(1, keepdim=True) + (g.abs() * d_z).mean(1, keepdim=True)
    inner = g - m0 - z * m1
    d_inner = d_m0 + z.abs() * d_m1 + m1.abs() * d_z + 4 * U * (g.abs() + m0.abs() + (z * m1).abs())
    want = rstd * inner
    _check(dx, want, rstd * d_inner + inner.abs() * d_rstd + _half(x.dtype) * 1.01 * want.abs(), "dx")
    rows = (n + 32) * U                                # no chain over the rows is longer than the rows themselves
    if dw is not None:
        assert torch.equal(dw, again[1]) and dw.dtype == w.dtype
        want = (G * z).sum(0)
        _check(dw, want, rows * (G * z).abs().sum(0) + (G.abs() * d_z).sum(0) + _half(dw.dtype) * 1.01 * want.abs(), "dweight")
    if db is not None:
        assert torch.equal(db, again[2]) and db.dtype == b.dtype
        want = G.sum(0)
        _check(db, want, rows * G.abs().sum(0) + _half(db.dtype) * 1.01 * want.abs(), "dbias")


BF, FP = torch.bfloat16, torch.float32
SIZES = [(1, 1), (1, 2048), (3, 7), (2, 64), (33, 513), (17, 1000), (300, 256), (1025, 1531), (5, 4096), (9, 5000),
         (7, 16384), (3, 20001), (2, 70000), (5000, 96)]


@pytest.mark.parametrize("n,h", SIZES)
@pytest.mark.parametrize("dtype,wtype", [(BF, BF), (BF, FP), (FP, FP)])
def test_forward_and_backward_match_the_formula(n, h, dtype, wtype):
    x, dy, w, b = _inputs(n, h, dtype, wtype, True, 0, n * 7 + h)
    _compare(x, dy, w, b, 1e-5)


@pytest.mark.parametrize("n,h", [(1185, 520), (2500, 640), (1300, 1000), (1201, 1024), (1190, 2040), (3001, 2048), (1187, 2056),
                                 (1300, 4096), (1200, 4104), (1186, 8192), (1188, 8200)])
@pytest.mark.parametrize("dtype,wtype,pad", [(BF, FP, 0), (BF, BF, 8), (FP, FP, 0), (FP, FP, 4)])
def test_many_aligned_rows(n, h, dtype, wtype, pad):
    """Rows that stream through shared memory: every width of it, the sizes around their limits, rows of a wider tensor, and
    row counts that leave the last group short."""
    x, dy, w, b = _inputs(n, h, dtype, wtype, True, pad, n + h)
    _compare(x, dy, w, b, 1e-5)


@pytest.mark.parametrize("n,h", [(1190, 768), (1203, 776), (1185, 1280), (1201, 1536), (1188, 1544), (1300, 2560), (1187, 2880), (1190, 3584),
                                 (1186, 5120), (1189, 6144), (1200, 6152), (1185, 7168)])
@pytest.mark.parametrize("dtype,wtype,pad", [(BF, FP, 0), (BF, BF, 8), (FP, FP, 4)])
def test_widths_between_the_powers_of_two(n, h, dtype, wtype, pad):
    x, dy, w, b = _inputs(n, h, dtype, wtype, True, pad, n + h)
    _compare(x, dy, w, b, 1e-5)


@pytest.mark.parametrize("n", [1, 16, 17, 1031, 40003])
@pytest.mark.parametrize("h", [2, 8, 12, 40, 64, 66, 100, 128, 131, 200, 256, 260, 392, 512])
@pytest.mark.parametrize("dtype,wtype,pad", [(BF, FP, 0), (BF, BF, 3), (FP, FP, 0), (FP, FP, 1)])
def test_short_rows(n, h, dtype, wtype, pad):
    """Several rows a warp: every number of lanes and accesses, row counts that leave the last turn short, one block and many."""
    x, dy, w, b = _inputs(n, h, dtype, wtype, True, pad, n + h)
    _compare(x, dy, w, b, 1e-5)


@pytest.mark.parametrize("n,h", [(60001, 640), (50002, 1000), (50003, 1280), (30002, 2048), (20011, 2560), (20003, 3584), (12001, 5120),
                                 (9002, 8192)])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_rows_that_go_round_the_ring_many_times(n, h, dtype):
    x, dy, w, b = _inputs(n, h, dtype, FP, True, 0, n + h)
    _compare(x, dy, w, b, 1e-5)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("pad", [1, 3, 4, 8, 24])
@pytest.mark.parametrize("h", [64, 2048, 321])
def test_rows_of_a_wider_tensor(dtype, pad, h):
    """The rows are a slice: their stride and alignment vary, and the elements between them are NaN."""
    x, dy, w, b = _inputs(37, h, dtype, dtype, True, pad, pad)
    assert x.stride(0) == h + pad
    _compare(x, dy, w, b, 1e-5)
    flat = torch.zeros(37 * h + 1, dtype=dtype, device=DEV)        # contiguous rows that start off every alignment
    odd = flat[1:].view(37, h)
    odd.copy_(x)
    _compare(odd, dy, w, b, 1e-5)


@pytest.mark.parametrize("wtype,bias", [(None, False), (None, True), (BF, False)])
def test_weight_and_bias_are_optional(wtype, bias):
    x, dy, w, b = _inputs(65, 768, BF, wtype, bias, 0, 3)
    _compare(x, dy, w, b, 1e-6)


def test_offset_channels_and_constant_rows():
    """A mean a thousand times the spread, and rows without any spread: y = bias, finite gradients."""
    x, dy, w, b = _inputs(50, 2048, FP, FP, True, 0, 5)
    _compare(x + 1000.0, dy, w, b, 1e-5)
    from bibo_b200 import functional as Fn
    const = torch.full((4, 2048), 3.25, device=DEV)
    y, saved = Fn.layernorm_forward(const, w, b, 1e-5, keep=True)
    dx, dw, db = Fn.layernorm_backward(dy[:4].contiguous(), const, w, saved)
    assert torch.equal(y, b.expand(4, -1)) and bool(dx.isfinite().all()) and float(dw.abs().max()) == 0.0
    bad = x.clone()
    bad[7, 100] = float("nan")
    bad[9, 3] = float("inf")
    y = Fn.layernorm_forward(bad, w, b, 1e-5)
    clean = Fn.layernorm_forward(x, w, b, 1e-5)
    keep = [i for i in range(50) if i not in (7, 9)]
    assert bool(y[7].isnan().all()) and bool(y[9].isnan().any()) and torch.equal(y[keep], clean[keep])


def test_offsets_beyond_32_bits():
    from bibo_b200 import functional as Fn
    n, h = 270000, 8192
    x = torch.randn(n, h, device=DEV, dtype=torch.bfloat16)
    assert x.numel() > 1 << 31
    w, b = torch.rand(h, device=DEV), torch.rand(h, device=DEV)
    y, saved = Fn.layernorm_forward(x, w, b, keep=True)
    dx, _, _ = Fn.layernorm_backward(x, x, w, saved)
    last = x[-2000:].contiguous()
    yl, sl = Fn.layernorm_forward(last, w, b, keep=True)
    assert torch.equal(y[-2000:], yl) and torch.equal(saved[0][:, -2000:], sl[0])
    assert torch.equal(dx[-2000:], Fn.layernorm_backward(last, last, w, sl)[0])


def test_no_rows():
    from bibo_b200 import functional as Fn
    w, b = torch.ones(64, device=DEV), torch.zeros(64, device=DEV)
    x = torch.empty(0, 64, device=DEV)
    y, saved = Fn.layernorm_forward(x, w, b, keep=True)
    dx, dw, db = Fn.layernorm_backward(x, x, w, saved)
    assert y.shape == dx.shape == (0, 64) and float(dw.abs().sum()) == 0 and float(db.abs().sum()) == 0


def test_module_is_a_layer_norm_and_gradient_matches_differences():
    import bibo_b200
    torch.manual_seed(0)
    m = bibo_b200.BiBoLayerNorm(40).to(DEV)
    m.load_state_dict(torch.nn.LayerNorm(40).state_dict())
    with torch.no_grad():
        m.weight.add_(0.3 * torch.randn(40, device=DEV))
        m.bias.add_(0.3 * torch.randn(40, device=DEV))
    x = torch.randn(2, 5, 40, device=DEV, requires_grad=True)
    c = torch.randn(2, 5, 40, device=DEV)
    (m(x) * c).sum().backward()

    def f(xx, ww, bb):
        mu = xx.mean(-1, keepdim=True)
        v = ((xx - mu) ** 2).mean(-1, keepdim=True)
        return (((xx - mu) / torch.sqrt(v + m.eps) * ww + bb) * c.double()).sum()

    args = [x.detach().double(), m.weight.detach().double(), m.bias.detach().double()]
    for i, grad in enumerate((x.grad, m.weight.grad, m.bias.grad)):
        d = torch.randn_like(args[i])
        lo, hi = list(args), list(args)
        h = 1e-5
        lo[i], hi[i] = args[i] - h * d, args[i] + h * d
        slope = float((f(*hi) - f(*lo)) / (2 * h))
        # differences: h^2 ~ 1e-10 of the third derivative; the kernel: a few hundred roundings of 2^-24 of order-1 terms
        assert abs(float((grad.double() * d).sum()) - slope) < 1e-3 * max(1.0, abs(slope))
    # a transposed input is not rows: it is laid out first, a gradient that is expanded too
    xt = torch.randn(40, 6, device=DEV).t().requires_grad_()
    m(xt).sum().backward()
    assert xt.grad.shape == (6, 40)
    with torch.no_grad():
        assert torch.equal(m(xt), m(xt.contiguous()))


def test_capture_and_side_stream():
    from bibo_b200 import functional as Fn
    x, dy, w, b = _inputs(64, 512, BF, BF, True, 0, 11)
    want = Fn.layernorm_forward(x, w, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = Fn.layernorm_forward(x, w, b)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, saved = Fn.layernorm_forward(x, w, b, keep=True)
        grads = Fn.layernorm_backward(dy, x, w, saved)
    x2 = torch.randn_like(x)
    x.copy_(x2)
    graph.replay()
    y_now, s_now = Fn.layernorm_forward(x2, w, b, keep=True)
    g_now = Fn.layernorm_backward(dy, x2, w, s_now)
    torch.cuda.synchronize()
    assert torch.equal(y, y_now) and all(torch.equal(a, c) for a, c in zip(grads, g_now))


def test_decoder_feed_forward_with_a_layer_norm():
    """moe.ffn_forward: h + block(layer_norm(h)), both with and without gradients."""
    from bibo_b200 import BiBoLayerNorm, BiBoMLP, BiBoMoELayer, MoEConfig
    from bibo_b200.moe import ffn_forward
    torch.manual_seed(1)
    for block in ("moe", "mlp"):
        dl = torch.nn.Module()
        cfg = MoEConfig(hidden_size=256, moe_intermediate_size=128, num_routed_experts=64)
        dl.mlp = BiBoMoELayer(cfg) if block == "moe" else BiBoMLP(cfg, is_expert=True, intermediate_size=256)
        dl.post_attention_layernorm = BiBoLayerNorm(256)
        dl = dl.to(DEV).to(torch.bfloat16).eval()
        h = torch.randn(2, 33, 256, device=DEV, dtype=torch.bfloat16)
        with torch.no_grad():
            got = ffn_forward(dl, h)
            x = dl.post_attention_layernorm(h)
            want = h + dl.mlp(x)
        # the residual is added to the block's rounded output inside its last kernel
        assert float((got.float() - want.float()).abs().max()) <= 2.0 ** -7 * float(want.float().abs().max())
        hg = h.clone().requires_grad_()
        out = ffn_forward(dl, hg)
        out.float().sum().backward()
        assert hg.grad.isfinite().all() and dl.post_attention_layernorm.weight.grad.isfinite().all()
        assert float((out.detach().float() - want.float()).abs().max()) <= 2.0 ** -7 * float(want.float().abs().max())
