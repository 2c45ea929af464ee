"""CPU checks of the norm, quantizer, product and linear layer: refusals of the Python calls and of the C entry points (no GPU is
touched), shape functions."""
import pytest
import torch

P = 1 << 20   # an aligned address that is never dereferenced


def test_python_calls_refuse():
    import mok
    x, w = torch.zeros(4, 256, dtype=torch.bfloat16), torch.zeros(256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        mok.rms_norm(x, w)
    with pytest.raises(ValueError, match="two-dimensional"):
        mok.rms_norm(x[0], w)
    with pytest.raises(ValueError, match="CUDA"):
        mok.quantize_blocks(x)
    with pytest.raises(ValueError, match="three dimensions"):
        mok.quantize_blocks(x[None])
    with pytest.raises(ValueError, match="two-dimensional CUDA"):
        mok.block_matmul((x, x), (x, x))
    with pytest.raises(ValueError, match="shapes"):
        mok.fp8_linear(x, torch.zeros(8, 128, dtype=torch.bfloat16))
    with pytest.raises(TypeError):
        mok.fp8_linear(x, torch.zeros(8, 256))


def test_norm_entry_points_refuse():
    from mok import _native as nat
    L = nat.lib()

    def forward(x=P, xs=256, r=None, rs=0, w=P, rows=4, hidden=256, hid=None, y=P, q=None, qs=0, s=None):
        return L.mok_rms_norm_forward(x, xs, r, rs, w, 0, rows, hidden, 1e-6, hid, y, q, qs, s, 1, 1, None, None)
    assert forward(rows=0) == 0
    for bad in (dict(x=None), dict(w=None), dict(y=None), dict(rows=-1), dict(hidden=0), dict(hidden=12), dict(x=P + 8), dict(xs=250),
                dict(r=P + 2, rs=256), dict(q=P, qs=256), dict(q=P, qs=128, s=P), dict(q=P + 4, qs=256, s=P), dict(xs=-256)):
        assert forward(**bad) == -1, bad
    assert forward(hidden=16392, xs=16392) == -4

    def backward(dy=P, z=P, zs=256, rows=4, hidden=256, dx=P, dw=P, scratch=P):
        return L.mok_rms_norm_backward(dy, None, z, zs, P, 0, P, rows, hidden, dx, dw, scratch, None)
    for bad in (dict(dy=None), dict(z=None), dict(dx=None), dict(dw=None), dict(scratch=None), dict(rows=0), dict(hidden=4), dict(dy=P + 4), dict(zs=4)):
        assert backward(**bad) == -1, bad
    assert L.mok_rms_norm_scratch_bytes(3, 256) == 3 * 256 * 4 and L.mok_rms_norm_scratch_bytes(0, 256) == 0


def test_quantizer_entry_point_refuses():
    from mok import _native as nat
    L = nat.lib()

    def call(x=P, xs=256, rows=4, cols=256, tile=1, q=P, qs=256, s=P, qt=None, qts=0, st=None):
        return L.mok_block_quantize(x, xs, rows, cols, tile, q, qs, s, 1, 1, qt, qts, st, 1, 1, None)
    assert call(rows=0) == 0
    for bad in (dict(x=None), dict(x=P + 4), dict(xs=3), dict(cols=12), dict(tile=2), dict(q=None), dict(q=None, s=None), dict(qs=128), dict(qs=260),
                dict(qt=P, qts=16), dict(qt=P, qts=2, st=P), dict(qt=P + 1, qts=16, st=P)):
        assert call(**bad) == -1, bad
    assert call(rows=65536 * 128) == -4


def test_product_entry_point_refuses():
    from mok import _native as nat
    L = nat.lib()

    def call(a=P, ast=256, sa=P, b=P, bst=256, sb=P, tile=128, rows=4, cols=256, depth=256, out=P, ost=256, scratch=P):
        return L.mok_block_matmul(a, ast, sa, 1, 1, b, bst, sb, 1, 1, tile, rows, cols, depth, out, ost, scratch, None, None)
    assert call(rows=0) == 0
    for bad in (dict(a=None), dict(sa=None), dict(b=None), dict(sb=None), dict(out=None), dict(tile=64), dict(rows=-1), dict(cols=0), dict(depth=0),
                dict(a=P + 8), dict(b=P + 4), dict(ast=250), dict(bst=240), dict(ost=128)):
        assert call(**bad) == -1, bad
    assert call(rows=(1 << 24) + 1) == -4
    assert L.mok_block_matmul_scratch_bytes(0, 128, 128) == 0 and L.mok_block_matmul_scratch_bytes(8192, 7168, 2048) == 0


def test_shape_functions():
    import mok  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x, w = torch.empty(24, 264, dtype=torch.bfloat16), torch.empty(264, dtype=torch.float32)
        y, hidden, rms = torch.ops.mok.rms_norm_fwd(x, w, None, 1e-6)
        assert (y.shape, hidden.shape, rms.shape, rms.dtype) == ((24, 264), (0,), (24,), torch.float32)
        q, s, hidden = torch.ops.mok.rms_norm_fp8_fwd(x, w, x, 1e-6)
        assert q.stride() == (272, 1) and q.shape == hidden.shape == (24, 264) and s.shape == (24, 3) and s.stride() == (1, 24)
        d_x, d_w = torch.ops.mok.rms_norm_bwd(x, None, x, w, rms)
        assert d_x.shape == x.shape and (d_w.shape, d_w.dtype) == (w.shape, torch.float32)
        q, s, qt, st = torch.ops.mok.block_quantize(x, 128, True)
        assert s.shape == (1, 3) and qt.shape == (264, 24) and qt.stride() == (32, 1) and st.shape == (3, 1)
        q1, s1, _, _ = torch.ops.mok.block_quantize(x, 1, False)
        out = torch.ops.mok.block_matmul(q1, s1, q, s)
        assert (out.shape, out.dtype) == ((24, 24), torch.bfloat16)


def test_linear_refuses_another_weights_codes():
    import mok
    x, w = torch.zeros(4, 256, dtype=torch.bfloat16), torch.zeros(128, 256, dtype=torch.bfloat16)

    def codes(rows, cols):
        return torch.zeros(rows, cols).to(torch.float8_e4m3fn), torch.ones(-(-rows // 128), -(-cols // 128))
    for bad in ((codes(64, 256), (None, None)), (codes(256, 128), codes(128, 256)), (codes(128, 256), codes(128, 256))):
        with pytest.raises(ValueError, match="must be that of weight"):
            mok.fp8_linear(x, w, quantized_weight=bad)
    # the transposed half is missed by the call that asks for it, not by its backward
    half = (codes(128, 256), (None, None))
    leaf = x.clone().requires_grad_()
    with pytest.raises(ValueError, match="transpose"):
        mok.fp8_linear(leaf, w, quantized_weight=half)
    for call in (lambda: mok.fp8_linear(x, w, quantized_weight=half), lambda: torch.no_grad()(mok.fp8_linear)(leaf, w, quantized_weight=half)):
        with pytest.raises(ValueError, match="CUDA"):   # got as far as the kernels' own checks
            call()


@pytest.mark.parametrize("x_grad", [False, True])
@pytest.mark.parametrize("w_grad", [False, True])
@pytest.mark.parametrize("kept", [False, True])
def test_linear_makes_what_its_gradients_need(monkeypatch, x_grad, w_grad, kept):
    """Which matrices are quantized, and which of them in both orientations, with and without gradients: requires_grad alone asks
    for nothing."""
    import mok
    from mok import block_ops
    x, w = torch.randn(4, 256).to(torch.bfloat16), torch.randn(128, 256).to(torch.bfloat16)
    calls = []

    def quantize(m, tile_rows, normal, transpose):
        calls.append(("x" if tile_rows == 1 else "w", transpose))
        one = torch.ones(1, 1)
        return m, one, (m.t() if transpose else None), (one if transpose else None)
    monkeypatch.setattr(block_ops, "_quantize", quantize)
    monkeypatch.setattr(block_ops, "_matmul", lambda a, a_scales, b, b_scales: a @ b.t())
    weight = ((w, torch.ones(1, 2)), (w.t(), torch.ones(2, 1))) if kept else None
    leaves = x.clone().requires_grad_(x_grad), w.clone().requires_grad_(w_grad)
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            out = mok.fp8_linear(*leaves, quantized_weight=weight)
        assert calls == ([] if kept else [("w", False)]) + [("x", False)] and not out.requires_grad
        calls.clear()
    out = mok.fp8_linear(*leaves, quantized_weight=weight)
    assert calls == ([] if kept else [("w", x_grad)]) + [("x", w_grad)] and out.requires_grad == (x_grad or w_grad)
    if out.requires_grad:
        out.sum().backward()
        assert [t.grad is not None for t in leaves] == [x_grad, w_grad]
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for mode in (torch.no_grad, torch.enable_grad):
            with mode(), pytest.raises(RuntimeError, match="forward mode AD"):
                mok.fp8_linear(dual, leaves[1], quantized_weight=weight)


def test_norm_refuses_tangents(monkeypatch):
    """Forward-mode tangents of any input, with and without gradients: there is no rule for them, and none may be lost."""
    import mok
    from mok import block_ops
    from torch.autograd import forward_ad
    x, w, r = torch.randn(4, 256).to(torch.bfloat16), torch.ones(256), torch.randn(4, 256).to(torch.bfloat16)
    monkeypatch.setattr(block_ops, "_norm_forward", lambda x, w, r, *rest: (x + r, None, None, x + r, w[:4] + 0.0))
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        for inputs in ((dual(x), w, r), (x, dual(w), r), (x, w, dual(r))):
            for mode in (torch.no_grad, torch.enable_grad):
                with mode(), pytest.raises(RuntimeError, match="forward mode AD"):
                    mok.rms_norm(*inputs)
        assert not mok.rms_norm(x, w, r)[0].requires_grad       # nothing with a tangent: as ever
