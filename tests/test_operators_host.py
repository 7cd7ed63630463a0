"""Argument checks and host logic of layer norm and expert-order dispatch: everything here fails, or is decided, before the
first CUDA call."""
import ctypes

import pytest
import torch


def _dummy():
    one = ctypes.c_int(0)
    return ctypes.addressof(one) & ~15 | 16            # non-null, 16-byte aligned, never dereferenced


def test_c_entry_points_refuse_bad_arguments():
    from bibo_b200 import _lib
    lib, p = _lib.load(), _dummy()
    err = lambda: lib.bibo_moe_last_error_string()
    F, B = _lib.F32, _lib.BF16
    assert lib.bibo_moe_layernorm_fwd(p, 64, p, p, 1e-5, 4, 64, 7, F, p, None, None, None) == -1 and b"dtype=7" in err()
    assert lib.bibo_moe_layernorm_fwd(p, 64, p, p, 1e-5, 4, 64, F, B, p, None, None, None) == -1 and b"weight dtype" in err()
    assert lib.bibo_moe_layernorm_fwd(p, 64, p, p, 1e-5, 4, 0, F, F, p, None, None, None) == -1
    assert lib.bibo_moe_layernorm_fwd(p, 63, p, p, 1e-5, 4, 64, F, F, p, None, None, None) == -1 and b"stride" in err()
    assert lib.bibo_moe_layernorm_fwd(p, 64, p, p, 1e-5, 4, 64, F, F, p, p, None, None) == -1 and b"null" in err()
    assert lib.bibo_moe_layernorm_fwd(None, 64, p, p, 1e-5, 4, 64, F, F, p, None, None, None) == -1
    assert lib.bibo_moe_layernorm_fwd(p, 64, p, p, 1e-5, 1 << 31, 64, F, F, p, None, None, None) == -4
    assert lib.bibo_moe_layernorm_fwd(None, 64, None, None, 1e-5, 0, 64, F, F, None, None, None, None) == 0
    assert lib.bibo_moe_layernorm_bwd(p, 64, p, 32, p, p, p, 4, 64, F, F, p, p, p, p, None) == -1 and b"stride" in err()
    assert lib.bibo_moe_layernorm_bwd(p, 64, p, 64, p, p, p, 400, 64, F, F, p, None, p, p, None) == -1 and b"null" in err()
    assert lib.bibo_moe_layernorm_bwd_parts(0) == 0 and lib.bibo_moe_layernorm_bwd_parts(400) == 400
    assert lib.bibo_moe_dispatch_plan(None, 4, 10, 6, 64, 1, p, None) == -1 and b"null" in err()
    assert lib.bibo_moe_dispatch_plan(p, 2, 10, 6, 64, 1, p, None) == -1 and b"indices of 2" in err()
    for n, k, e, a in ((-1, 6, 64, 1), (10, 0, 64, 1), (10, 33, 64, 1), (10, 6, 0, 1), (10, 6, 1025, 1), (10, 6, 64, 0),
                       (10, 6, 64, 1025), (1 << 28, 6, 64, 1), (1 << 59, 32, 64, 1)):
        assert lib.bibo_moe_dispatch_plan(p, 4, n, k, e, a, p, None) == -4
        assert lib.bibo_moe_dispatch_rows_cap(n, k, e, a) == -1 and lib.bibo_moe_dispatch_plan_words(n, k, e, a) == -1
        assert lib.bibo_moe_dispatch_fwd(p, 64, p, n, 64, k, e, a, F, p, None) == -4
        assert lib.bibo_moe_dispatch_combine_fwd(p, p, F, p, n, 64, k, e, a, F, p, None) == -4
        assert lib.bibo_moe_dispatch_combine_bwd(p, 64, p, p, F, p, n, 64, k, e, a, F, p, p, None) == -4
    assert lib.bibo_moe_dispatch_fwd(p, 64, p, 4, 0, 6, 64, 1, F, p, None) == -4
    assert lib.bibo_moe_dispatch_fwd(p, 32, p, 4, 64, 6, 64, 1, F, p, None) == -1 and b"stride" in err()
    assert lib.bibo_moe_dispatch_fwd(p, 64, None, 4, 64, 6, 64, 1, F, p, None) == -1
    assert lib.bibo_moe_dispatch_combine_fwd(p, p, 5, p, 4, 64, 6, 64, 1, F, p, None) == -1 and b"weight dtype" in err()
    assert lib.bibo_moe_dispatch_combine_bwd(p, 64, None, p, F, p, 4, 64, 6, 64, 1, F, p, p, None) == -1


def test_row_bounds_of_a_plan():
    from bibo_b200 import _lib
    lib = _lib.load()
    cap = lib.bibo_moe_dispatch_rows_cap
    assert cap(100, 6, 64, 1) == 600 and cap(0, 6, 64, 128) == 0
    assert cap(1, 6, 64, 128) == 6 * 128                            # at most six groups have a row
    assert cap(100, 6, 64, 16) == (600 + 64 * 15 + 15) // 16 * 16
    for n, k, e, a in ((100, 6, 64, 16), (3, 2, 7, 128), (1, 1, 1, 1)):
        row_slot = lib.bibo_moe_dispatch_off_row_slot(n, k, e)
        assert lib.bibo_moe_dispatch_off_slot_row(e) >= 2 * e + 2 and lib.bibo_moe_dispatch_off_slot_row(e) % 4 == 0
        assert row_slot >= lib.bibo_moe_dispatch_off_slot_row(e) + n * k
        assert lib.bibo_moe_dispatch_plan_words(n, k, e, a) >= row_slot + cap(n, k, e, a)


def test_python_entry_points_refuse_cpu_tensors():
    import bibo_b200
    from bibo_b200 import functional as Fn
    x = torch.randn(4, 64)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        Fn.layernorm_forward(x)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        bibo_b200.BiBoLayerNorm(64)(x)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        bibo_b200.layer_norm(x.requires_grad_())
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        Fn.dispatch_plan(torch.zeros(4, 2, dtype=torch.int32), 8)
    with pytest.raises(RuntimeError, match="normalise the last dimension"):
        bibo_b200.BiBoLayerNorm((4, 64))(x)


def test_layer_norm_module_has_the_state_dict_of_torchs():
    import bibo_b200
    mine, theirs = bibo_b200.BiBoLayerNorm(48, eps=1e-6, bias=False), torch.nn.LayerNorm(48, eps=1e-6, bias=False)
    assert list(mine.state_dict()) == list(theirs.state_dict()) == ["weight"] and mine.eps == 1e-6
    assert bibo_b200.BiBoLayerNorm(48, elementwise_affine=False).weight is None


class _FakeCuda(torch.Tensor):
    """A tensor that says it is on a GPU, for the checks that come before any launch."""

    @property
    def is_cuda(self):
        return True


def _fake(t):
    return t.as_subclass(_FakeCuda)


def test_shape_stride_and_dtype_checks():
    from bibo_b200 import functional as Fn
    rows = lambda *s, **k: _fake(torch.zeros(*s, **k))
    with pytest.raises(RuntimeError, match="rows"):
        Fn.layernorm_forward(rows(4))
    with pytest.raises(RuntimeError, match="H >= 1"):
        Fn.layernorm_forward(rows(4, 0))
    with pytest.raises(RuntimeError, match="contiguous within its rows"):
        Fn.layernorm_forward(rows(64, 4).t())
    with pytest.raises(RuntimeError, match="contiguous within its rows"):
        Fn.layernorm_forward(_fake(torch.zeros(1, 64).expand(4, 64)))
    x = rows(4, 64)
    with pytest.raises(RuntimeError, match=r"weight must be \[64\]"):
        Fn.layernorm_forward(x, rows(63))
    with pytest.raises(RuntimeError, match="both float32"):
        Fn.layernorm_forward(x, rows(64, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="both float32"):
        Fn.layernorm_forward(rows(4, 64, dtype=torch.bfloat16), rows(64), rows(64, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        Fn.layernorm_forward(rows(4, 64, dtype=torch.float16))
    saved = (torch.zeros(2, 4), torch.float32)
    with pytest.raises(RuntimeError, match="expected 64"):
        Fn.layernorm_backward(rows(4, 63), x, None, saved)
    with pytest.raises(RuntimeError, match="dtype"):
        Fn.layernorm_backward(rows(4, 64, dtype=torch.bfloat16), x, None, saved)
    with pytest.raises(RuntimeError, match="kept 4"):
        Fn.layernorm_backward(rows(3, 64), rows(3, 64), None, saved)
    with pytest.raises(RuntimeError, match="dy has 3 rows"):
        Fn.layernorm_backward(rows(3, 64), x, None, saved)
    with pytest.raises(RuntimeError, match="int32 or int64"):
        Fn.dispatch_plan(rows(4, 2), 8)
    with pytest.raises(RuntimeError, match="int32 or int64"):
        Fn.dispatch_plan(rows(4, dtype=torch.int32), 8)
    with pytest.raises(RuntimeError, match="n_experts=1025"):
        Fn.dispatch_plan(rows(4, 2, dtype=torch.int32), 1025)
    plan = Fn.DispatchPlan(4, 2, 8, 1, "cpu")
    assert (plan.rows, plan.buf.numel(), plan._slot_row, plan._row_slot) == Fn._plan_layout(4, 2, 8, 1)
    assert plan.rows == 8 and plan.slot_row.shape == (4, 2) and plan.offsets.shape == (9,) and plan.row_slot.shape == (8,)
    with pytest.raises(RuntimeError, match="needs 4"):
        Fn.dispatch_forward(rows(5, 64), plan)
    with pytest.raises(RuntimeError, match="needs 8"):
        Fn.combine_forward(rows(7, 64), None, plan)
    with pytest.raises(RuntimeError, match=r"topk_w must be \[4, 2\]"):
        Fn.combine_forward(rows(8, 64), rows(4, 3), plan)
    with pytest.raises(RuntimeError, match="ys must be contiguous"):
        Fn.combine_forward(rows(8, 65)[:, :64], None, plan)
    with pytest.raises(RuntimeError, match="expected 64"):
        Fn.combine_backward(rows(4, 32), rows(8, 64), None, plan)
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        Fn.combine_forward(rows(8, 64), rows(4, 2, dtype=torch.float16), plan)


def test_orthogonalize_refusals_and_workspace():
    import bibo_b200
    from bibo_b200 import _lib
    from bibo_b200 import functional as Fn
    lib, p = _lib.load(), _dummy()
    co = (ctypes.c_float * 3)(1.5, -0.5, 0.0)
    aligned = (p + 127) & ~127
    call = lambda batch=2, bs=640 * 320, r=640, c=320, rs=320, dt=_lib.F32, steps=1, u=p, ws=aligned, out=p: lib.bibo_moe_orthogonalize(
        u, batch, bs, r, c, rs, dt, steps, co, 1e-7, ws, out, None)
    err = lambda: lib.bibo_moe_last_error_string()
    assert call(dt=3) == -1 and call(steps=0) == -1 and call(steps=65) == -1 and b"steps=65" in err()
    assert call(rs=319) == -1 and call(bs=640 * 320 - 1) == -1 and b"overlapping" in err()
    assert call(u=None) == -1 and call(ws=None) == -1 and call(out=None) == -1
    assert call(ws=aligned + 16) == -2 and call(r=-1) == -1
    assert call(batch=0) == 0 and call(r=0) == 0
    size = lib.bibo_moe_orthogonalize_workspace
    assert size(0, 5, 5) == 0 and size(7, 128, 300) == size(7, 300, 128) == 0 and size(7, 129, 300) > 0
    assert size(64, 1024, 2048) == size(64, 2048, 1024) <= 1 << 31
    assert size(10000, 1024, 2048) <= 1 << 31 and size(1, 20000, 20000) > 1 << 31
    fake = lambda *s, **k: _fake(torch.zeros(*s, **k))
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        Fn.orthogonalize(torch.zeros(4, 4))
    with pytest.raises(RuntimeError, match="a matrix or a stack"):
        Fn.orthogonalize(fake(4))
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        Fn.orthogonalize(fake(4, 4, dtype=torch.float16))
    for steps, c in ((0, Fn.NEWTON_SCHULZ), (2, [Fn.NEWTON_SCHULZ]), (1, (1.0, 2.0))):
        with pytest.raises(RuntimeError, match="steps need"):
            Fn.orthogonalize(fake(4, 4), steps, c)
    with pytest.raises(ValueError, match="matrices"):
        bibo_b200.Muon([torch.nn.Parameter(torch.zeros(4))])
    with pytest.raises(ValueError, match="momentum"):
        bibo_b200.Muon([torch.nn.Parameter(torch.zeros(4, 4))], momentum=1.0)


def test_muon_state_loads_in_fp32():
    import bibo_b200
    make = lambda: bibo_b200.Muon([torch.nn.Parameter(torch.zeros(4, 6, dtype=t)) for t in (torch.bfloat16, torch.float32)])
    a, b = make(), make()
    for p in a.param_groups[0]["params"]:
        a.state[p]["momentum_buffer"] = torch.randn(4, 6)
    b.load_state_dict(a.state_dict())
    for p, q in zip(a.param_groups[0]["params"], b.param_groups[0]["params"]):
        got, want = b.state[q]["momentum_buffer"], a.state[p]["momentum_buffer"]
        assert got.dtype == torch.float32 and torch.equal(got, want) and got.data_ptr() != want.data_ptr()
    make().load_state_dict(make().state_dict())                        # no step taken yet


def test_muon_skips_empty_parameters():
    import bibo_b200
    p = torch.nn.Parameter(torch.zeros(4, 0))
    p.grad = torch.zeros(4, 0)
    bibo_b200.Muon([p]).step()


def test_feed_forward_calls_a_layer_norm_with_a_forward_of_its_own(monkeypatch):
    from bibo_b200 import mlp, norm
    from bibo_b200.moe import ffn_forward
    monkeypatch.setattr(mlp, "mlp_module_forward", lambda m, x, residual=None: x if residual is None else x + residual)
    monkeypatch.setattr(norm, "layer_norm_module_forward", lambda m, x: torch.full_like(x, 7))

    class Doubled(torch.nn.LayerNorm):
        def forward(self, x):
            return 2 * super().forward(x)

    h = torch.randn(3, 8)
    for grad in (True, False):
        for cls, want in ((torch.nn.LayerNorm, lambda m: torch.full_like(h, 7)), (Doubled, lambda m: m(h))):
            dl = torch.nn.Module()
            dl.mlp, dl.post_attention_layernorm = torch.nn.Module(), cls(8)
            with torch.set_grad_enabled(grad):
                assert torch.equal(ffn_forward(dl, h), h + want(dl.post_attention_layernorm))
            if cls is torch.nn.LayerNorm:
                with monkeypatch.context() as m, torch.set_grad_enabled(grad):
                    m.setattr(torch, "is_autocast_enabled", lambda *a: True)
                    assert torch.equal(ffn_forward(dl, h), h + dl.post_attention_layernorm(h))
