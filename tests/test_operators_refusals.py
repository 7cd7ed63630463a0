"""Calls of the operators beside the block that have to be refused, or answered otherwise, before anything is launched."""
import pytest
import torch


class _FakeCuda(torch.Tensor):
    """A tensor that says it is on a GPU, for the checks that come before any launch."""

    @property
    def is_cuda(self):
        return True


def _fake(t):
    return t.as_subclass(_FakeCuda)


def _zeros(*shape, **kw):
    return _fake(torch.zeros(*shape, **kw))


@pytest.fixture
def launches(monkeypatch):
    """The names of the kernels' entry points that a test's calls would have launched."""
    from bibo_b200 import functional as Fn
    names = []
    monkeypatch.setattr(Fn, "_launch", lambda name, dev, *args: names.append(name))
    return names


def test_layernorm_backward_refuses_a_weight_that_is_not_the_forwards(launches):
    """The kernel reads [H] elements of the forward's parameter type behind the weight's address."""
    from bibo_b200 import functional as Fn
    x, dy = _zeros(4, 64), _zeros(4, 64)
    stats = _zeros(2, 4)
    bad = [_zeros(64, dtype=torch.bfloat16), _zeros(8), _zeros(65), _zeros(1, 64), _zeros(128)[::2], torch.zeros(64)]
    for weight in bad:
        with pytest.raises(RuntimeError, match="weight"):
            Fn.layernorm_backward(dy, x, weight, (stats, torch.float32))
    half = _zeros(4, 64, dtype=torch.bfloat16)
    for wtype, other in ((torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)):
        with pytest.raises(RuntimeError, match="weight must be the forward's"):
            Fn.layernorm_backward(half, half, _zeros(64, dtype=other), (stats, wtype))
    for saved in ((stats.double(), torch.float32), (_zeros(4, 2).t(), torch.float32), (stats, torch.bfloat16)):
        with pytest.raises(RuntimeError, match="not what layernorm_forward kept"):
            Fn.layernorm_backward(dy, x, None, saved)
    assert launches == []
    Fn.layernorm_backward(dy, x, _zeros(64), (stats, torch.float32))
    Fn.layernorm_backward(half, half, _zeros(64, dtype=torch.bfloat16), (stats, torch.bfloat16))
    assert launches == ["bibo_moe_layernorm_bwd"] * 2


def test_layer_norm_refuses_forward_mode_tangents(launches):
    """The kernel fills a fresh tensor: a tangent would be lost without a word."""
    import bibo_b200
    from torch.autograd import forward_ad
    frozen = bibo_b200.BiBoLayerNorm(8).requires_grad_(False)
    value, tangent = torch.randn(3, 8), torch.randn(3, 8)
    with forward_ad.dual_level():
        x = forward_ad.make_dual(value, tangent)
        w = forward_ad.make_dual(torch.ones(8), torch.randn(8))
        for call in (lambda: bibo_b200.layer_norm(x), lambda: frozen(x), lambda: bibo_b200.layer_norm(value, w),
                     lambda: bibo_b200.layer_norm(value, torch.ones(8), w), lambda: bibo_b200.BiBoLayerNorm(8)(x)):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="forward-mode"):
                    call()
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(frozen, (value,), (tangent,))
    assert launches == []


def test_orthogonalize_refuses_polynomials_that_leave_the_range():
    """x, G and b G + c G^2 are kept as f16 times 2^12, so singular values that start in [0, 1] have to stay below 4 and the factor
    below 16 in every step that sees them, not in the first one alone."""
    import ctypes
    from bibo_b200 import _lib
    from bibo_b200 import functional as Fn
    lib = _lib.load()

    def call(*steps, eps=1e-7):
        flat = (ctypes.c_float * (3 * len(steps)))(*[v for c in steps for v in c])
        return lib.bibo_moe_orthogonalize(None, 0, 0, 4, 4, 4, _lib.F32, len(steps), flat, eps, None, None, None)   # no matrices

    ns, half = Fn.NEWTON_SCHULZ, (0.5, 0.0, 0.0)
    assert call(*[ns] * 64) == 0 and call((1.5, -0.5, 0.0)) == 0 and call((1.875, -1.25, 0.375), ns) == 0
    assert call((1.0, 16.0, -16.0), (0.25, 0.0, 0.0), (1.5, -0.5, 0.0)) == 0            # up to 3.76, factor up to 4
    assert call((8.25, -23.5, 17.25), (4.0, -3.0, 0.5), (4.0, -3.0, 0.5)) == 0
    assert call((15.0, 0.0, 0.0)) == 0 and call((15.0, 0.0, 0.0), half) == -4              # the last result need not be squared
    assert call((16.0, 0.0, 0.0)) == -4
    assert call((3.9, 0.0, 0.0), ns) == -4 and b"step 1" in lib.bibo_moe_last_error_string()     # factor near 400 at 3.9
    assert call((1.0, 0.0, -15.9)) == -4 and call((1.0, 64.0, -64.0)) == -4                 # at the end and inside of [0, 1]
    assert call((0.1, 4.0, 0.0), half) == -4 and call((0.1, 3.8, 0.0), half) == 0
    assert call((4.0, 16.0, -17.0), half) == -4                                          # 5.8 inside, 3 at s = 1
    for bad in (float("nan"), float("inf"), -float("inf")):
        for at in range(3):
            assert call(ns, tuple(bad if i == at else v for i, v in enumerate(ns))) == -4
    assert call(ns, eps=-1e-7) == -1 and call(ns, eps=float("nan")) == -1 and call(ns, eps=0.0) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layer_norm_module_returns_fp32_under_autocast(launches, monkeypatch, dtype):
    import bibo_b200
    norm, x = bibo_b200.BiBoLayerNorm(8, dtype=dtype), _zeros(3, 8, dtype=dtype)
    norm.weight, norm.bias = (torch.nn.Parameter(_fake(p.detach())) for p in (norm.weight, norm.bias))
    assert norm(x).dtype == dtype
    monkeypatch.setattr(torch, "is_autocast_enabled", lambda *a: True)
    with torch.no_grad():
        assert norm(x).dtype == torch.float32
    assert norm(x).dtype == torch.float32 and len(launches) == 3


def _decoder(norm):
    dl = torch.nn.Module()
    dl.mlp, dl.post_attention_layernorm = torch.nn.Module(), norm
    return dl


def test_feed_forward_fires_the_hooks_of_a_layer_norm(monkeypatch):
    """The kernels are called around the module, so a module with hooks, or with a forward set on it, is called itself."""
    from bibo_b200 import mlp, norm
    from bibo_b200.moe import ffn_forward
    monkeypatch.setattr(mlp, "mlp_module_forward", lambda m, x, residual=None: x if residual is None else x + residual)
    monkeypatch.setattr(norm, "layer_norm_module_forward", lambda m, x: torch.full_like(x, 7))
    h, seen = torch.randn(3, 8), []
    hooks = {
        "forward": lambda m: m.register_forward_hook(lambda *a: seen.append(1)),
        "with kwargs": lambda m: m.register_forward_hook(lambda *a: seen.append(1), with_kwargs=True),
        "pre": lambda m: m.register_forward_pre_hook(lambda *a: seen.append(1)),
        "backward": lambda m: m.register_full_backward_hook(lambda *a: seen.append(1)),
        "pre-backward": lambda m: m.register_full_backward_pre_hook(lambda *a: seen.append(1)),
        "global": lambda m: torch.nn.modules.module.register_module_forward_hook(lambda *a: seen.append(1)),
    }
    for kind, register in hooks.items():
        for grad in (True, False):
            if "backward" in kind and not grad:
                continue
            m = torch.nn.LayerNorm(8)
            want = h + m(h)
            handle = register(m)
            seen.clear()
            with torch.set_grad_enabled(grad):
                out = ffn_forward(_decoder(m), h.clone().requires_grad_(grad))
            if grad:
                out.sum().backward()
            handle.remove()
            assert torch.equal(out, want) and len(seen) >= 1, kind
            with torch.no_grad():
                assert torch.equal(ffn_forward(_decoder(m), h), h + 7)          # nobody listens any more
    m = torch.nn.LayerNorm(8)
    m.forward = lambda x: 3 * x
    with torch.no_grad():
        assert torch.equal(ffn_forward(_decoder(m), h), h + 3 * h)


def test_feed_forward_adds_a_residual_of_another_type_itself(monkeypatch):
    """A norm that is called as it is may return another type than the stream's: the blocks' kernels refuse such a residual."""
    from bibo_b200 import mlp, moe
    from bibo_b200.moe import ffn_forward

    def block(m, x, residual=None):
        if residual is not None and residual.dtype != x.dtype:
            raise RuntimeError(f"residual dtype {residual.dtype} != {x.dtype}")
        return x if residual is None else x + residual

    class Wide(torch.nn.LayerNorm):
        def forward(self, x):
            return super().forward(x.float())

    monkeypatch.setattr(mlp, "mlp_module_forward", block)
    monkeypatch.setattr(moe, "layer_forward", block)
    h = torch.randn(3, 8, dtype=torch.bfloat16)
    for is_moe in (False, True):
        dl = _decoder(Wide(8))
        if is_moe:
            dl.mlp.gate = dl.mlp.experts = None
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                got = ffn_forward(dl, h)
            assert got.dtype == torch.float32 and torch.equal(got, h + dl.post_attention_layernorm(h))


def test_muon_refuses_before_it_changes_anything():
    import bibo_b200
    from bibo_b200 import functional as Fn
    make = lambda **kw: bibo_b200.Muon([torch.nn.Parameter(torch.zeros(4, 6))], **kw)
    opt = make()
    for bad, match in ((dict(params=[torch.nn.Parameter(torch.zeros(4))]), "matrices"),
                       (dict(params=[torch.nn.Parameter(torch.zeros(2, 2))], momentum=1.0), "momentum"),
                       (dict(params=[torch.nn.Parameter(torch.zeros(2, 2))], steps=65), "steps=65"),
                       (dict(params=[torch.nn.Parameter(torch.zeros(2, 2))], coefficients=(9.0, 0.0, 0.0)), "out of range")):
        with pytest.raises(ValueError, match=match):
            opt.add_param_group(bad)
        assert len(opt.param_groups) == 1
    for bad in (dict(steps=0), dict(steps=1 << 40), dict(steps=2, coefficients=[Fn.NEWTON_SCHULZ]), dict(eps=-1.0),
                dict(coefficients=(1.0, float("nan"), 0.0))):
        with pytest.raises(ValueError, match="Muon"):
            make(**bad)
    # a parameter that is not on a GPU, beside one that says it is: neither has moved afterwards
    near, far = torch.nn.Parameter(_zeros(4, 6)), torch.nn.Parameter(torch.zeros(4, 6))
    for p in (near, far):
        p.grad = torch.ones(4, 6)
    opt = bibo_b200.Muon([near, far])
    momentum = torch.full((4, 6), 3.0)
    opt.state[near]["momentum_buffer"] = momentum
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        opt.step()
    assert bool((momentum == 3).all()) and not opt.state[far]


def test_orthogonalize_refuses_step_counts_without_building_them():
    from bibo_b200 import functional as Fn
    with pytest.raises(RuntimeError, match="steps=65"):
        Fn.check_polynomials(1 << 40, Fn.NEWTON_SCHULZ, 1e-7)
    with pytest.raises(RuntimeError, match="steps need"):
        Fn.check_polynomials(1 << 40, [Fn.NEWTON_SCHULZ] * 3, 1e-7)
    Fn.check_polynomials(64, Fn.NEWTON_SCHULZ, 0.0)


def test_sizes_beyond_32_bits_are_refused_and_not_cut(launches):
    """The C ABI takes them as 32-bit integers: 2^32 + 8 columns would be eight."""
    from bibo_b200 import _lib
    from bibo_b200 import functional as Fn
    lib = _lib.load()
    wide = _fake(torch.empty(1, 2 ** 32 + 8, device="meta"))
    with pytest.raises(RuntimeError, match="up to 2\\^30"):
        Fn.layernorm_forward(wide)
    plan = Fn.DispatchPlan(1, 1, 8, 1, "meta")
    for call in (lambda: Fn.dispatch_forward(wide, plan), lambda: Fn.combine_forward(wide, None, plan),
                 lambda: Fn.combine_backward(wide, wide, None, plan)):
        with pytest.raises(RuntimeError, match="up to 2\\^30"):
            call()
    for shape in ((2 ** 32 + 4, 8), (8, 2 ** 32 + 4)):
        with pytest.raises(RuntimeError, match="rows and columns"):
            Fn.orthogonalize(_fake(torch.empty(shape, device="meta")))
    for k, e, a in ((2, 2 ** 32 + 8, 1), (2, 8, 2 ** 32 + 1), (2 ** 32 + 2, 8, 1)):
        with pytest.raises(RuntimeError, match="dispatch plan"):
            Fn.dispatch_plan(_fake(torch.empty(0, k, dtype=torch.int32, device="meta")), e, a)
    assert launches == []
    p = 4096                                                    # never read: refused before the first launch
    assert lib.bibo_moe_layernorm_fwd(p, 1 << 31, p, p, 1e-5, 4, (1 << 30) + 1, _lib.F32, _lib.F32, p, None, None, None) == -4
    wide = 65535 * 256 + 1
    assert lib.bibo_moe_layernorm_bwd(p, wide, p, wide, p, p, p, 4, wide, _lib.F32, _lib.F32, p, p, p, p, None) == -4
