"""The norm, the quantizer, the 8-bit product and the linear layer against plain formulas in 64 bits.

Tolerances: a rounding to bf16 is off by at most 2^-8 of the value (half a step), one to e4m3 by 2^-4 (below the normal range by
2^-10 of the scale); fp32 sums of n terms by n 2^-23 of the sum of magnitudes, whatever their order."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, E4M3 = 2.0 ** -8, 2.0 ** -4


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import mok  # noqa: F401
    return torch.device("cuda", 0)


def _normal(dev, *shape, std=1.0, seed=0, dtype=torch.bfloat16):
    return torch.empty(shape, device=dev).normal_(0.0, std, generator=torch.Generator(device=dev).manual_seed(seed)).to(dtype)


def _within(got, want, tol):
    off = (got.double() - want).abs()
    assert got.shape == want.shape and bool((off <= tol).all()), f"{(off - tol).max().item():.3e} above the bound"


def _scales(x, rows):
    """Smallest power of two per rows x 128 that brings the block to 448, at least 2^-126, in 64 bits."""
    x = torch.nn.functional.pad(x.double(), (0, -x.shape[1] % 128, 0, -x.shape[0] % rows))
    big = x.view(x.shape[0] // rows, rows, -1, 128).abs().amax(dim=(1, 3))
    fraction, exponent = torch.frexp(big / 448.0)   # fraction in [0.5, 1), 0 for 0; log2 is not exact on every device
    exponent = torch.where(fraction == 0.5, exponent - 1, exponent)
    return torch.ldexp(torch.ones_like(big), torch.where(big > 0, exponent, -126).clamp_min(-126))


def _spread(scales, shape, rows):
    return scales.double().repeat_interleave(rows, 0)[: shape[0]].repeat_interleave(128, 1)[:, : shape[1]]


def _quantized(x, rows):
    s = _scales(x, rows)
    every = _spread(s, x.shape, rows)
    return (x.double() / every).to(torch.float32).to(torch.float8_e4m3fn), s


def _values(q, s, rows):
    return q.double() * _spread(s, q.shape, rows)


# ---- norm -----------------------------------------------------------------------------------------------------------
NORM_SHAPES = [(1, 8), (1, 2048), (3, 264), (5, 128), (7, 1000), (65, 2056), (333, 7168), (300, 8192), (4, 8200), (2, 16384)]


def _norm_inputs(dev, T, H, residual, w32=False, seed=0):
    x = _normal(dev, T, H, seed=seed)
    r = _normal(dev, T, H, std=2.0, seed=seed + 1) if residual else None
    w = (1.0 + 0.2 * _normal(dev, H, seed=seed + 2, dtype=torch.float32)).to(torch.float32 if w32 else torch.bfloat16)
    return x, r, w


def _norm_reference(x, r, w, eps):
    z = x.double() + (r.double() if r is not None else 0.0)
    rho = (z.square().mean(1, keepdim=True) + eps).rsqrt()
    return z, rho, z * rho * w.double()


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("T,H", NORM_SHAPES)
def test_norm_forward(dev, T, H, residual):
    import mok
    x, r, w = _norm_inputs(dev, T, H, residual, w32=H % 16 == 0)
    z, rho, want = _norm_reference(x, r, w, 1e-6)
    got = mok.rms_norm(x, w, r)
    y, hidden = got if residual else (got, None)
    _within(y, want, (BF16 + 2.0 ** -18) * want.abs())
    if residual:
        _within(hidden, z, BF16 * z.abs())
    (q, s), hidden8 = mok.rms_norm_quantized(x, w, r)
    big = torch.nn.functional.pad(want, (0, -H % 128)).view(T, -1, 128).abs().amax(2)
    near = (torch.log2(big / 448.0) - torch.log2(big / 448.0).round()).abs() < 1e-5   # the fp32 value may lie on the other side
    assert bool(((s.double() == _scales(want, 1)) | near).all()) and s.shape == (T, -(-H // 128))
    _within(_values(q, s, 1), want, (E4M3 + 2.0 ** -18) * want.abs() + 2.0 ** -10 * _spread(s, want.shape, 1))
    assert (hidden8 is None) == (not residual) and (not residual or torch.equal(hidden8, hidden))


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("T,H", NORM_SHAPES)
def test_norm_backward(dev, T, H, residual):
    import mok
    x, r, w = _norm_inputs(dev, T, H, residual, w32=H % 16 == 0)
    d_y, d_h = _normal(dev, T, H, seed=7), _normal(dev, T, H, seed=8)
    leaves = [t.requires_grad_() for t in (x, w, r) if t is not None]
    y = mok.rms_norm(x, w, r)
    ends, grads = (y, (d_y, d_h)) if residual else ((y,), (d_y,))
    got = torch.autograd.grad(ends, leaves, grads)
    z, rho, _ = _norm_reference(x.detach(), r.detach() if residual else None, w.detach(), 1e-6)
    g = d_y.double() * w.detach().double()
    c = rho.square() * (g * z).mean(1, keepdim=True)
    want = rho * (g - z * c) + (d_h.double() if residual else 0.0)
    # z is read back from its rounding to bf16, which moves z c and the mean of g z by 2^-8 of their magnitudes at most
    moved = rho * z.abs() * (c.abs() + rho.square() * (g * z).abs().mean(1, keepdim=True)) if residual else 0.0
    fine = rho * (g.abs() + 2 * z.abs() * rho.square() * (g * z).abs().mean(1, keepdim=True))
    tol = BF16 * (want.abs() + moved) * (1 + BF16) + H * 2.0 ** -23 * fine + 2.0 ** -20 * (d_h.double().abs() if residual else 0.0)
    _within(got[0], want, tol)
    if residual:
        assert torch.equal(got[0], got[2])
    terms = d_y.double() * z * rho
    sum_tol = (BF16 if residual else 0.0) + (T + 16) * 2.0 ** -23
    want_w = terms.sum(0)
    _within(got[1], want_w, (BF16 if got[1].dtype == torch.bfloat16 else 2.0 ** -24) * want_w.abs() * 1.01 + sum_tol * 1.01 * terms.abs().sum(0))
    assert got[1].dtype == w.dtype


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("T,H", [(4000, 1032), (3100, 2048), (2400, 2056), (1700, 4104), (900, 8200), (450, 16384)])
def test_norm_backward_many_rows_a_block(dev, T, H, residual):
    test_norm_backward(dev, T, H, residual)


@pytest.mark.parametrize("T,H", [(1, 8), (40, 1000), (333, 7168), (64, 16384)])
def test_norm_codes_are_those_of_the_exact_norm(dev, T, H):
    """A code is another one than the exact norm's only where the exact value lies next to the middle between two codes: the sum of
    squares is off by 2^-21 at most (eights of squares in fp32, then 64 bits), its root by half of that, and rho, two products and
    the value that is rounded to a code by 2^-24 each: 2^-21 in all."""
    import mok
    x, r, w = _norm_inputs(dev, T, H, True)
    want = _norm_reference(x, r, w, 1e-6)[2]
    (q, s), _ = mok.rms_norm_quantized(x, w, r)
    exact = want / _spread(s, q.shape, 1)
    codes = torch.arange(256, device=dev, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    codes = codes[codes.isfinite()].unique()            # in order
    above = torch.searchsorted(codes, exact).clamp(1, codes.numel() - 1)
    nearest = torch.minimum((exact - codes[above - 1]).abs(), (exact - codes[above]).abs())
    # within d of the middle either neighbour is at most 2 d further away than the nearest
    assert bool(((exact - q.double()).abs() <= nearest + 2 * 2.0 ** -21 * exact.abs()).all())


def test_norm_gradient_against_differences(dev):
    import mok
    T, H, h = 6, 520, 1e-5
    x, r, w = _norm_inputs(dev, T, H, True, w32=True)
    d_y, d_h = _normal(dev, T, H, seed=7).double(), _normal(dev, T, H, seed=8).double()
    leaves = [t.requires_grad_() for t in (x, r, w)]
    got = torch.autograd.grad(mok.rms_norm(x, w, r), leaves, (d_y.bfloat16(), d_h.bfloat16()))

    def f(x, r, w):
        z, _, y = _norm_reference(x, r, w, 1e-6)
        return (y * d_y + z * d_h).sum()
    base = [t.detach().double() for t in leaves]
    for i in range(3):
        step = _normal(dev, *base[i].shape, seed=20 + i, dtype=torch.float64)
        up, down = [list(base), list(base)]
        up[i], down[i] = base[i] + h * step, base[i] - h * step
        slope = (f(*up) - f(*down)) / (2 * h)
        # every entry of the gradient is off by 2^-8 of it, and by as much through z, at most (see test_norm_backward)
        tol = 4 * BF16 * (got[i].double() * step).abs().sum()
        assert abs((got[i].double() * step).sum() - slope) <= tol
        assert tol < 0.2 * (got[i].double().norm() * step.norm())   # the bound says something


def test_norm_unused_outputs_and_frozen_inputs(dev):
    import mok
    x, r, w = _norm_inputs(dev, 9, 256, True)
    x.requires_grad_()
    y, hidden = mok.rms_norm(x, w, r)
    d = _normal(dev, 9, 256, seed=3)
    assert torch.equal(torch.autograd.grad(hidden, x, d, retain_graph=True)[0], d)       # y unused
    only_y = torch.autograd.grad(y, x, d, retain_graph=True)[0]
    both = torch.autograd.grad((y, hidden), x, (d, torch.zeros_like(d)))[0]
    assert torch.equal(only_y, both)
    w.requires_grad_()
    y = mok.rms_norm(x.detach(), w)
    d_w, = torch.autograd.grad(y, w, d)
    assert d_w.shape == w.shape


def test_norm_shared_leaf_gets_both_gradients(dev):
    import mok
    x, _, w = _norm_inputs(dev, 5, 256, False)
    x.requires_grad_()
    y, hidden = mok.rms_norm(x, w, x)                     # the same tensor as input and residual: z = 2 x
    (y.float().sum() + hidden.float().sum()).backward()
    z = (2 * x.detach()).requires_grad_()
    y1 = mok.rms_norm(z, w)
    d_z, = torch.autograd.grad(y1, z, torch.ones_like(y1))
    want = 2 * (d_z.double() + 1)
    _within(x.grad, want, 4 * BF16 * (want.abs() + 2))


def test_norm_extreme_rows(dev):
    import mok
    H = 512
    x = _normal(dev, 6, H)
    x[0] = 0
    x[1, 3] = float("nan")
    x[2, 5] = float("inf")
    x[3] *= 1e-18
    x[4] *= 1e15
    w = torch.ones(H, device=dev, dtype=torch.bfloat16)
    y = mok.rms_norm(x, w)
    assert bool((y[0] == 0).all()) and bool(y[1].isnan().all()) and bool(y[2, 5].isnan())
    want = _norm_reference(x, None, w, 1e-6)[2]
    _within(y[3:], want[3:], (BF16 + 2.0 ** -18) * want[3:].abs())
    (q, s), _ = mok.rms_norm_quantized(x, w)
    assert bool((q[0].float() == 0).all()) and bool((s[0] == 2.0 ** -126).all())
    assert bool(s[1].isnan().all()) and bool(q[1].float().isnan().all())


# ---- quantizer ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("tile_rows", [1, 128])
@pytest.mark.parametrize("M,N", [(1, 8), (1, 128), (7, 136), (128, 128), (129, 264), (200, 1000), (1000, 1544), (65, 2048)])
def test_quantizer_is_exact(dev, M, N, tile_rows):
    import mok
    x = _normal(dev, M, N, std=3.0)
    x[0, :8] = torch.tensor([0, 448.0, 448.0 * 2 ** -6, 449.0 * 2, 2.0 ** -126, -3.0, 1e30, -1e-30], device=dev).bfloat16()
    if M > 5:
        x[5] = 0
    (q, s), (qt, st) = mok.quantize_blocks(x, tile_rows=tile_rows, transpose=True)
    one_q, one_s = mok.quantize_blocks(x, tile_rows=tile_rows)
    for got_q, got_s, m in ((q, s, x), (qt, st, x.t()), (one_q, one_s, x)):
        want_q, want_s = _quantized(m, tile_rows)
        assert got_s.shape == want_s.shape and torch.equal(got_s.double(), want_s)
        assert got_q.shape == m.shape and torch.equal(got_q.contiguous().view(torch.uint8) & 0x7F, want_q.view(torch.uint8) & 0x7F)
        assert torch.equal(got_q.double(), want_q.double())


@pytest.mark.parametrize("tile_rows", [1, 128])
def test_quantizer_not_finite(dev, tile_rows):
    import mok
    x = _normal(dev, 256, 384)
    x[3, 5], x[200, 300] = float("nan"), float("-inf")
    (q, s), (qt, st) = mok.quantize_blocks(x, tile_rows=tile_rows, transpose=True)
    for v in (_values(q, s, tile_rows), _values(qt, st, tile_rows).t()):
        bad = v.isnan()
        assert bool(bad[3, 5]) and bool(bad[200, 300])
        hit = torch.zeros_like(bad)
        if tile_rows == 128:
            hit[:128, :128] = hit[128:, 256:] = True
            assert torch.equal(bad, hit)
        else:
            assert int(bad.sum()) == 2 * 128     # one block of the matrix concerned each


def test_quantizer_of_experts(dev):
    import mok
    for I in (256, 192):
        w = _normal(dev, 3, I, 320, std=0.1)
        q, s = mok.quantize_blocks(w, tile_rows=128)
        assert q.shape == w.shape and s.shape == (3, -(-I // 128), 3) and q.is_contiguous()
        for e in range(3):
            want_q, want_s = _quantized(w[e], 128)
            assert torch.equal(q[e].double(), want_q.double()) and torch.equal(s[e].double(), want_s)


# ---- product --------------------------------------------------------------------------------------------------------
def _operands(dev, M, N, K, b_rows, seed=0):
    a = _normal(dev, M, K, std=100.0, seed=seed, dtype=torch.float32).clamp(-448, 448).to(torch.float8_e4m3fn)
    b = _normal(dev, N, K, std=100.0, seed=seed + 1, dtype=torch.float32).clamp(-448, 448).to(torch.float8_e4m3fn)
    kb = -(-K // 128)
    sa = torch.rand(kb, M, device=dev, generator=torch.Generator(device=dev).manual_seed(seed + 2)).add_(0.5).t()
    sb = torch.rand(-(-N // 128) if b_rows == 128 else N, kb, device=dev, generator=torch.Generator(device=dev).manual_seed(seed + 3)).add_(0.5)
    return a, sa, b, sb


def _check_product(got, a, sa, b, sb, b_rows):
    av, bv = _values(a, sa, 1), _values(b, sb, b_rows)
    want = av @ bv.t()
    # one rounding to bf16; 128 products and their scaled sums in fp32
    _within(got, want, BF16 * want.abs() * 1.01 + (256 + a.shape[1] / 128) * 2.0 ** -23 * (av.abs() @ bv.abs().t()))


PRODUCTS = [(1, 1, 16), (1, 128, 128), (1, 2048, 2048), (5, 264, 304), (16, 4096, 1024), (17, 130, 4096), (31, 129, 144), (32, 768, 2048),
            (33, 640, 1040), (64, 2048, 512), (65, 300, 8192), (128, 256, 256), (200, 257, 400), (255, 512, 128), (256, 256, 2048), (257, 1100, 640),
            (1000, 1544, 1808), (2304, 2048, 384), (20, 4096, 7168), (5000, 1032, 272), (4900, 1500, 400)]


@pytest.mark.parametrize("b_rows", [1, 128])
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_product(dev, M, N, K, b_rows):
    import mok
    a, sa, b, sb = _operands(dev, M, N, K, b_rows)
    got = mok.block_matmul((a, sa), (b, sb))
    torch.cuda.synchronize()
    mok.ops.check_status(dev)
    _check_product(got, a, sa, b, sb, b_rows)
    assert torch.equal(got, mok.block_matmul((a, sa), (b, sb)))


def test_product_strides_and_depth_that_is_no_multiple_of_16(dev):
    import mok
    M, N, K = 100, 200, 333
    a, sa, b, sb = _operands(dev, M, N, K, 128)
    got = mok.block_matmul((a, sa), (b, sb))                                   # rows of 333 bytes: copied to aligned rows
    _check_product(got, a, sa, b, sb, 128)
    wide_a, wide_b = torch.zeros(M, 512, device=dev).to(a.dtype), torch.zeros(N, 400, device=dev).to(a.dtype)
    wide_a.view(torch.uint8).fill_(0x7F)                                       # NaN codes around the operands are not read
    wide_b.view(torch.uint8).fill_(0x7F)
    va, vb = wide_a[:, 64:64 + K], wide_b[:, 16:16 + K]
    va.copy_(a), vb.copy_(b)
    assert torch.equal(got, mok.block_matmul((va, sa.contiguous()), (vb, sb.t().contiguous().t())))


def test_product_passes_nan_on(dev):
    import mok
    for M in (4, 300):
        a, sa, b, sb = _operands(dev, M, 256, 512, 128)
        clean = mok.block_matmul((a, sa), (b, sb))
        a.view(torch.uint8)[2, 100] = 0x7F
        b.view(torch.uint8)[130, 7] = 0xFF
        sa = sa.clone()
        sa[1, 3] = float("inf")
        got = mok.block_matmul((a, sa), (b, sb))
        bad = torch.zeros_like(got, dtype=torch.bool)
        bad[2], bad[:, 130] = True, True
        assert bool(got[bad].isnan().all()) and bool((got[1].isinf() | got[1].isnan()).all())
        bad[1] = True
        assert torch.equal(got[~bad], clean[~bad])


def test_product_beyond_31_bits(dev):
    import mok
    M, N, K = 70000, 32768, 128
    a, sa, b, sb = _operands(dev, M, N, K, 128)
    got = mok.block_matmul((a, sa), (b, sb))
    for rows in (slice(0, 3), slice(M - 3, M)):
        _check_product(got[rows], a[rows], sa[rows], b, sb, 128)


def test_norm_and_quantizer_beyond_31_bits(dev):
    import mok
    T, H = 140000, 16384
    x = _normal(dev, 8, H).repeat(T // 8, 1)
    w = torch.ones(H, device=dev, dtype=torch.bfloat16)
    y = mok.rms_norm(x, w)
    assert torch.equal(y[-8:], y[:8]) and torch.equal(y[:8], mok.rms_norm(x[:8], w))
    del y
    q, s = mok.quantize_blocks(x)
    want = mok.quantize_blocks(x[:8])
    assert torch.equal(q[-8:].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(s[-8:], want[1])


# ---- linear layer ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T,N,K", [(1, 128, 256), (37, 264, 136), (300, 512, 640), (130, 2048, 1000)])
def test_linear_and_its_gradients(dev, T, N, K):
    import mok
    x, w, d_y = _normal(dev, T, K).requires_grad_(), _normal(dev, N, K, std=K ** -0.5, seed=1).requires_grad_(), _normal(dev, T, N, seed=2)
    y = mok.fp8_linear(x, w)
    d_x, d_w = torch.autograd.grad(y, (x, w), d_y)
    xd, wd = x.detach(), w.detach()
    qx, qw, qd = (_values(*_quantized(m, r), r) for m, r in ((xd, 1), (wd, 128), (d_y, 1)))
    qxt, qdt = (_values(*_quantized(m.t(), 1), 1) for m in (xd, d_y))
    for got, a, b in ((y, qx, qw), (d_x, qd, qw.t()), (d_w, qdt, qxt)):
        want = a @ b.t()
        _within(got, want, BF16 * want.abs() * 1.01 + (256 + a.shape[1] / 128) * 2.0 ** -23 * (a.abs() @ b.abs().t()))
    kept = mok.quantize_weight(wd)
    y2 = mok.fp8_linear(x, w, quantized_weight=kept)
    assert torch.equal(y, y2) and torch.equal(torch.autograd.grad(y2, x, d_y)[0], d_x)
    with torch.no_grad():
        assert torch.equal(mok.fp8_linear(x, w), y)
        assert torch.equal(mok.block_matmul(mok.quantize_blocks(x), kept[0]), y)
    y3 = mok.fp8_linear(x, wd)
    assert torch.equal(torch.autograd.grad(y3, x, d_y.t().contiguous().t())[0], d_x)      # a gradient of other strides


# ---- all of them: strides, streams, graphs, empty batches --------------------------------------------------------------
def test_strided_rows(dev):
    import mok
    wide = _normal(dev, 50, 1024)
    w = _normal(dev, 512, seed=1)
    view = wide[::2, 256:768]
    assert torch.equal(mok.rms_norm(view, w), mok.rms_norm(view.contiguous(), w))
    odd = wide[:, 3:515]                                   # rows begin between 16-byte boundaries
    assert torch.equal(mok.rms_norm(odd, w, odd)[0], mok.rms_norm(odd.contiguous(), w, odd.contiguous())[0])
    turned = _normal(dev, 512, 64).t()
    for a, b in zip(mok.quantize_blocks(turned), mok.quantize_blocks(turned.contiguous())):
        assert torch.equal(a.float(), b.float())
    x = wide[:, :512].requires_grad_()
    one_row = x[:1].expand(50, 512)                        # row stride zero
    y = mok.rms_norm(one_row, w)
    d = torch.autograd.grad(y, x, torch.ones((), device=dev, dtype=torch.bfloat16).expand(50, 512))[0]
    assert bool(torch.isfinite(d).all()) and torch.equal(y[0], y[49])


def test_empty_batches(dev):
    import mok
    x, w = torch.empty(0, 256, device=dev, dtype=torch.bfloat16, requires_grad=True), _normal(dev, 256).requires_grad_()
    y = mok.rms_norm(x, w)
    d_x, d_w = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert y.shape == (0, 256) and d_x.shape == (0, 256) and bool((d_w == 0).all())
    (q, s), _ = mok.rms_norm_quantized(x.detach(), w.detach())
    assert q.shape == (0, 256) and s.shape == (0, 2)
    assert mok.block_matmul((q, s), mok.quantize_blocks(_normal(dev, 128, 256), tile_rows=128)).shape == (0, 128)
    m = _normal(dev, 128, 256).requires_grad_()
    y = mok.fp8_linear(x, m)
    assert y.shape == (0, 128) and bool((torch.autograd.grad(y.sum(), m)[0] == 0).all())


def test_side_stream_and_captured_graph(dev):
    """norm -> 8-bit product -> norm, on another stream and captured; two graphs replayed in turn do not disturb each other."""
    import mok
    T, H, N = 20, 1024, 2048
    w, w2 = _normal(dev, H, seed=1), _normal(dev, N, seed=2)
    weight = mok.quantize_weight(_normal(dev, N, H, std=0.03, seed=3), transpose=False)[0]

    def chain(x, r):
        q, hidden = mok.rms_norm_quantized(x, w, r)
        return mok.rms_norm(mok.block_matmul(q, weight), w2), hidden
    inputs = [(_normal(dev, T, H, seed=10 + i), _normal(dev, T, H, seed=20 + i)) for i in range(4)]
    want = [chain(*i) for i in inputs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = chain(*inputs[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, want[0]))
    graphs = []
    for x, r in inputs[:2]:
        x, r = x.clone(), r.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = chain(x, r)
        graphs.append((g, x, r, out))
    for i, (g, x, r, _) in enumerate(graphs):
        x.copy_(inputs[2 + i][0]), r.copy_(inputs[2 + i][1])
    for g, *_ in graphs + graphs[::-1]:
        g.replay()
    torch.cuda.synchronize()
    for i, (_, _, _, out) in enumerate(graphs):
        assert all(torch.equal(a, b) for a, b in zip(out, want[2 + i]))


def test_captured_training_step(dev):
    import mok
    x, w, m = _normal(dev, 64, 512).requires_grad_(), _normal(dev, 512, seed=1).requires_grad_(), _normal(dev, 256, 512, std=0.05, seed=2).requires_grad_()
    d = _normal(dev, 64, 256, seed=3)

    def step():
        return torch.autograd.grad(mok.fp8_linear(mok.rms_norm(x, w), m), (x, w, m), d)
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_traced_calls_match(dev):
    import mok
    x, r, w = _norm_inputs(dev, 16, 256, True)
    weight = mok.quantize_blocks(_normal(dev, 128, 256, std=0.05), tile_rows=128)

    @torch.compile(fullgraph=True, backend="aot_eager")
    def f(x, r):
        (q, s), hidden = mok.rms_norm_quantized(x, w, r)
        y, _ = mok.rms_norm(x, w, r)
        return mok.block_matmul((q, s), weight), hidden, y
    got = f(x, r)
    (q, s), hidden = mok.rms_norm_quantized(x, w, r)
    want = mok.block_matmul((q, s), weight), hidden, mok.rms_norm(x, w, r)[0]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("residual", [False, True])
def test_traced_training_step_matches(dev, residual):
    """Norm and linear layer under torch.compile, forward and both gradients: the eager call's to the bit."""
    import mok
    x, r = (_normal(dev, 40, 256, seed=i).requires_grad_() for i in range(2))
    w, a = _normal(dev, 256, seed=3).requires_grad_(), _normal(dev, 64, 256, std=0.06, seed=4).requires_grad_()
    kept = mok.quantize_weight(a.detach())

    def step(x, r, w, a):
        y, hidden = mok.rms_norm(x, w, r) if residual else (mok.rms_norm(x, w), x * 2)
        return mok.fp8_linear(y, a), mok.fp8_linear(hidden, a, quantized_weight=kept)
    args = (x, r, w, a)
    leaves = args if residual else (x, w, a)
    want = step(*args)
    ends = [_normal(dev, *t.shape, seed=5 + i) for i, t in enumerate(want)]
    grads = torch.autograd.grad(want, leaves, ends)
    got = torch.compile(step, fullgraph=True, backend="aot_eager")(*args)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(got, leaves, ends), grads))
    with torch.no_grad():
        again = torch.compile(step, fullgraph=True, backend="aot_eager")(*args)
    assert all(torch.equal(p, q) for p, q in zip(again, want)) and not again[0].requires_grad
