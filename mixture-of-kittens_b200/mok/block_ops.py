"""Operators around the MoE layer: the root-mean-square norm with the residual's addition and 8-bit floating point products with
a scale per block of 128.  The reference has none of them: its operators begin with the activations and end with the layer's
output.

A matrix in 8 bits is a pair (codes, scales): e4m3 codes [M, N] and fp32 scales, value = scale * code.  Scales are per 1 x 128
([M, ceil(N / 128)], activations) or per 128 x 128 ([ceil(M / 128), ceil(N / 128)], weights).  The quantizers take the smallest
power of two that brings a block to 448; the product takes any scales.  Scales of 1 x 128 come back as a transposed view (block
index major), which is how the product reads them.

`rms_norm`, `rms_norm_quantized`, `quantize_blocks`, `block_matmul` and `fp8_linear` are what a model calls; the `mok::*` ops below
are what `torch.compile` sees.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad as _forward_ad

from ._native import entry as _entry
from ._native import launch, status_word
from .ops import _require

E4M3 = torch.float8_e4m3fn
_BF16, _F32 = torch.bfloat16, torch.float32
BLOCK = 128


_traced_impl = None


def _traced() -> bool:
    global _traced_impl
    if _traced_impl is None:
        from .functional import _traced as _traced_impl
    return _traced_impl()


def _differentiated(*tensors: torch.Tensor | None) -> bool:
    """Whether autograd has to see a call on these tensors: a gradient may be asked for, or they may have tangents (which the autograd
    functions here refuse)."""
    return ((torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors))
            or _forward_ad._current_level >= 0)


class _NoDerivative(torch.autograd.Function):
    @staticmethod
    def forward(ctx, what, call, *tensors):
        ctx.what = what
        return call()

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(ctx.what + " has no derivatives: no autograd formula was written for it")


def _without_derivative(what: str, call, *tensors: torch.Tensor | None):
    """call(), which reads these tensors: where one of them requires a gradient the outputs ask for it in a backward that raises (as
    those of the ops do; 7 to 14 us of host time instead of 20 to 34), and tangents are refused."""
    if _forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and _forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(what + " has no derivatives: its inputs must not have tangents")
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return _NoDerivative.apply(what, call, *tensors)
    return call()


def _round_up(n: int, m: int) -> int:
    return -(-n // m) * m


def _address(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _check_matrix(name: str, x: torch.Tensor, multiple: int) -> None:
    _require(x.ndim == 2, name + " must be two-dimensional")
    _require(x.is_cuda, name + " must be a CUDA tensor")
    _require(x.dtype is _BF16, name + " must be bfloat16", TypeError)
    if x.shape[1] <= 0 or x.shape[1] % multiple:
        raise ValueError(f"{name}'s last dimension must be a positive multiple of {multiple}")


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x, or a copy where the kernels cannot address its rows (16-byte aligned, neighbours in memory, rows 16 bytes apart or more)."""
    if x.stride(1) == 1 and x.stride(0) % 8 == 0 and x.stride(0) >= 0 and x.data_ptr() % 16 == 0:
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _like(x: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of x's shape and type."""
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


def _new_codes(like: torch.Tensor, rows: int, cols: int) -> torch.Tensor:
    """[rows, cols] codes whose rows begin at multiples of 16 bytes."""
    ld = _round_up(cols, 16)
    q = like.new_empty((rows, ld), dtype=E4M3)
    return q if ld == cols else q[:, :cols]


def _new_scales(like: torch.Tensor, rows: int, cols: int, tile_rows: int) -> torch.Tensor:
    blocks = -(-cols // BLOCK)
    if tile_rows == 1:
        return torch.empty_strided((rows, blocks), (1, rows), dtype=_F32, device=like.device)
    return like.new_empty((-(-rows // BLOCK), blocks), dtype=_F32)


# ------------------------------------------------------------------------------------------------------------
# norm
# ------------------------------------------------------------------------------------------------------------
def _check_norm(x, weight, residual, eps) -> None:
    _check_matrix("x", x, 8)
    _require(x.shape[1] <= 16384, "x's last dimension must be at most 16384")
    _require(weight.shape == x.shape[1:], "weight must have shape (hidden_size,)")
    _require(weight.device == x.device, "weight must be on the device of x")
    _require(weight.dtype is _BF16 or weight.dtype is _F32, "weight must be bfloat16 or float32", TypeError)
    if residual is not None:
        _require(residual.shape == x.shape and residual.device == x.device, "residual must have the shape and device of x")
        _require(residual.dtype is _BF16, "residual must be bfloat16", TypeError)
    _require(isinstance(eps, float) and eps >= 0.0, "eps must be a non-negative float", TypeError)


def _norm_forward(x, weight, residual, eps, want_y, want_codes, want_rms):
    _check_norm(x, weight, residual, eps)
    x = _rows(x)
    T, H = x.shape
    weight = weight.contiguous()
    if weight.data_ptr() % 16:
        weight = weight.clone()
    hidden = None
    if residual is not None:
        residual = _rows(residual)
        hidden = _like(x)
    y = _like(x) if want_y else None
    codes = _new_codes(x, T, H) if want_codes else None
    scales = _new_scales(x, T, H, 1) if want_codes else None
    rms = x.new_empty((T,), dtype=_F32) if want_rms else None
    if T:
        launch("rms_norm", _entry("mok_rms_norm_forward"), x.device, x.data_ptr(), x.stride(0), _address(residual),
               0 if residual is None else residual.stride(0), weight.data_ptr(), weight.dtype is _F32, T, H, eps, _address(hidden),
               _address(y), _address(codes), codes.stride(0) if want_codes else 0, _address(scales),
               scales.stride(0) if want_codes else 0, scales.stride(1) if want_codes else 0, _address(rms))
    return y, codes, scales, hidden, rms


@torch.library.custom_op("mok::rms_norm_fwd", mutates_args=())
def rms_norm_fwd(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None, eps: float
                 ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """z = x + residual in fp32; inv_rms = (mean z^2 + eps)^-1/2; y = z * inv_rms * weight.

    Inputs:  x bf16 [T, H] (H % 8 == 0); weight bf16 | f32 [H]; residual bf16 [T, H] | None; eps float
    Outputs: y bf16 [T, H]; hidden = z rounded to bf16 [T, H] (empty without a residual); inv_rms f32 [T]
    """
    y, _, _, hidden, rms = _norm_forward(x, weight, residual, eps, True, False, True)
    return y, hidden if hidden is not None else x.new_empty((0,)), rms


@torch.library.custom_op("mok::rms_norm_fp8_fwd", mutates_args=())
def rms_norm_fp8_fwd(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None, eps: float
                     ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """rms_norm_fwd with y quantized from its fp32 values.

    Outputs: codes e4m3 [T, H]; scales f32 [T, ceil(H / 128)]; hidden bf16 [T, H] (empty without a residual)
    """
    _, codes, scales, hidden, _ = _norm_forward(x, weight, residual, eps, False, True, False)
    return codes, scales, hidden if hidden is not None else x.new_empty((0,))


def _norm_backward(d_y, d_hidden, z, weight, rms):
    _check_matrix("z", z, 8)
    T, H = z.shape
    _require(weight.shape == z.shape[1:] and rms.shape == z.shape[:1], "weight and inv_rms must have shapes (hidden_size,) and (num_tokens,)")
    _require(weight.dtype is _BF16 or weight.dtype is _F32, "weight must be bfloat16 or float32", TypeError)
    _require(rms.dtype is _F32, "inv_rms must be float32", TypeError)
    for name, t in (("d_y", d_y), ("d_hidden", d_hidden)):
        if t is not None:
            _require(t.shape == z.shape and t.device == z.device, name + " must have the shape and device of z")
            _require(t.dtype is _BF16, name + " must be bfloat16", TypeError)
    _require(weight.device == z.device and rms.device == z.device, "weight and inv_rms must be on the device of z")
    d_x, d_weight = z.new_empty((T, H)), torch.empty_like(weight, memory_format=torch.contiguous_format)
    if T == 0:
        return d_x, d_weight.zero_()
    z, weight, rms = _rows(z), weight.contiguous(), rms.contiguous()
    if weight.data_ptr() % 16:
        weight = weight.clone()
    d_y = _rows(d_y.contiguous())
    d_hidden = None if d_hidden is None else _rows(d_hidden.contiguous())
    scratch = z.new_empty((_entry("mok_rms_norm_scratch_bytes")(T, H) // 4,), dtype=_F32)
    launch("rms_norm backward", _entry("mok_rms_norm_backward"), z.device, d_y.data_ptr(), _address(d_hidden), z.data_ptr(), z.stride(0),
           weight.data_ptr(), weight.dtype is _F32, rms.data_ptr(), T, H, d_x.data_ptr(), d_weight.data_ptr(), scratch.data_ptr())
    return d_x, d_weight


@torch.library.custom_op("mok::rms_norm_bwd", mutates_args=())
def rms_norm_bwd(d_y: torch.Tensor, d_hidden: torch.Tensor | None, z: torch.Tensor, weight: torch.Tensor, inv_rms: torch.Tensor
                 ) -> tuple[torch.Tensor, torch.Tensor]:
    """Gradients of rms_norm_fwd.

    Inputs:  d_y bf16 [T, H]; d_hidden bf16 [T, H] | None; z bf16 [T, H] (hidden, or x without a residual); weight; inv_rms f32 [T]
    Outputs: d_x bf16 [T, H] (also the residual's); d_weight [H] in the weight's type, summed in a fixed order
    """
    return _norm_backward(d_y, d_hidden, z, weight, inv_rms)


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        ctx.set_materialize_grads(False)
        if _traced():
            y, hidden, rms = rms_norm_fwd(x, weight, residual, eps)
            hidden = None if residual is None else hidden
        else:
            y, _, _, hidden, rms = _norm_forward(x, weight, residual, eps, True, False, True)
        ctx.save_for_backward(x if hidden is None else hidden, weight, rms)
        ctx.has_residual = residual is not None
        return y if hidden is None else (y, hidden)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_y, d_hidden=None):
        z, weight, rms = ctx.saved_tensors
        if d_y is None:   # only the residual stream went on
            return d_hidden, None, d_hidden if ctx.has_residual else None, None
        d_x, d_weight = (rms_norm_bwd if _traced() else _norm_backward)(d_y, d_hidden, z, weight, rms)
        return d_x, d_weight, d_x if ctx.has_residual else None, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *, eps: float = 1e-6):
    """Root-mean-square norm of x + residual, differentiable: y bf16 [T, H], or (y, hidden) with a residual, where hidden =
    x + residual (rounded to bf16) is the stream that the next block adds to.  The norm is taken of the unrounded sum; the backward
    reads the sum from `hidden`, so that one tensor is kept for it instead of two."""
    if _differentiated(x, weight, residual):
        return _RmsNorm.apply(x, weight, residual, eps)
    if _traced():
        y, hidden, _ = rms_norm_fwd(x, weight, residual, eps)
        return y if residual is None else (y, hidden)
    y, _, _, hidden, _ = _norm_forward(x, weight, residual, eps, True, False, False)
    return y if residual is None else (y, hidden)


def rms_norm_quantized(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *, eps: float = 1e-6):
    """The norm's output in 8 bits, ready for `block_matmul`: ((codes, scales), hidden), hidden None without a residual.  Not
    differentiable, a backward through it raises: `fp8_linear` quantizes inside and has one."""
    if _traced():
        codes, scales, hidden = rms_norm_fp8_fwd(x, weight, residual, eps)
        return (codes, scales), hidden if residual is not None else None
    _, codes, scales, hidden, _ = _without_derivative(
        "rms_norm_quantized", lambda: _norm_forward(x, weight, residual, eps, False, True, False), x, weight, residual)
    return (codes, scales), hidden


# ------------------------------------------------------------------------------------------------------------
# quantizer
# ------------------------------------------------------------------------------------------------------------
def _quantize(x, tile_rows, normal, transpose):
    _check_matrix("x", x, 8)
    _require(tile_rows in (1, BLOCK), "tile_rows must be 1 or 128")
    _require(normal or transpose, "at least one quantized layout must be requested")
    x = _rows(x)
    M, N = x.shape
    across, down = -(-N // BLOCK), -(-M // BLOCK)
    q = s = qt = st = None
    s_strides, st_strides = ((1, M), (1, N)) if tile_rows == 1 else ((across, 1), (down, 1))
    if normal:
        q, s = _new_codes(x, M, N), _new_scales(x, M, N, tile_rows)
    if transpose:
        qt, st = _new_codes(x, N, M), _new_scales(x, N, M, tile_rows)
    if M:
        launch("block_quantize", _entry("mok_block_quantize"), x.device, x.data_ptr(), x.stride(0), M, N, tile_rows,
               _address(q), _round_up(N, 16), _address(s), *s_strides, _address(qt), _round_up(M, 16), _address(st), *st_strides)
    return q, s, qt, st


@torch.library.custom_op("mok::block_quantize", mutates_args=())
def block_quantize(x: torch.Tensor, tile_rows: int, transpose: bool
                   ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """bf16 [M, N] (N % 8 == 0) -> codes [M, N], scales, and with `transpose` those of x.T (empty otherwise): blocks of 1 x 128 along
    the last dimension of the matrix concerned (tile_rows 1), or of 128 x 128 (tile_rows 128)."""
    q, s, qt, st = _quantize(x, tile_rows, True, transpose)
    if not transpose:
        qt, st = x.new_empty((0,), dtype=E4M3), x.new_empty((0,), dtype=_F32)
    return q, s, qt, st


def quantize_blocks(x: torch.Tensor, *, tile_rows: int = 1, transpose: bool = False):
    """(codes, scales) of a bf16 matrix, or ((codes, scales), (codes, scales) of x.T) with `transpose`, read once for both; without
    gradients.
    [E, M, N] weights of several experts (tile_rows 128, without `transpose`) give [E, M, N] codes and a scale per 128 x 128 of
    every expert."""
    if x.ndim == 3:
        _require(tile_rows == BLOCK and not transpose, "three dimensions are quantized with tile_rows 128 and without the transpose")
        E, M, N = x.shape
        if M % BLOCK == 0 and x.is_contiguous():
            q, s = quantize_blocks(x.view(E * M, N), tile_rows=BLOCK)
            if q.is_contiguous():
                return q.view(E, M, N), s.view(E, M // BLOCK, -1)
        parts = [quantize_blocks(m, tile_rows=BLOCK) for m in x]
        return torch.stack([q.view(torch.uint8) for q, _ in parts]).view(E4M3), torch.stack([s for _, s in parts])
    if _traced():
        q, s, qt, st = block_quantize(x, tile_rows, transpose)
    else:
        q, s, qt, st = _quantize(x, tile_rows, True, transpose)
    return ((q, s), (qt, st)) if transpose else (q, s)


# ------------------------------------------------------------------------------------------------------------
# product
# ------------------------------------------------------------------------------------------------------------
def _codes(name: str, q: torch.Tensor) -> tuple[torch.Tensor, int, int, int, int]:
    """q, or a copy that the kernels can address, its shape, row stride and address."""
    shape = q.shape
    _require(len(shape) == 2 and q.is_cuda, name + " must be a two-dimensional CUDA tensor")
    _require(q.dtype is E4M3, name + " must be float8_e4m3fn", TypeError)
    (rows, cols), (ld, step), address = shape, q.stride(), q.data_ptr()
    if step != 1 or ld % 16 or ld < cols or address % 16:
        out = _new_codes(q, rows, cols)
        out.copy_(q)
        q, ld, address = out, out.stride(0), out.data_ptr()
    return q, rows, cols, ld, address


def _matmul(a, a_scales, b, b_scales):
    a, M, K, a_ld, a_address = _codes("a", a)
    b, N, b_depth, b_ld, b_address = _codes("b", b)
    _require(b_depth == K and K > 0 and N > 0, "a and b must have shapes (M, K) and (N, K), N and K positive")
    blocks = -(-K // BLOCK)
    _require(a_scales.shape == (M, blocks), "a_scales must have shape (M, ceil(K / 128))")
    tile_rows = BLOCK if b_scales.shape == (-(-N // BLOCK), blocks) else 1
    _require(tile_rows == BLOCK or b_scales.shape == (N, blocks),
             "b_scales must have shape (ceil(N / 128), ceil(K / 128)) or (N, ceil(K / 128))")
    _require(a_scales.dtype is _F32 and b_scales.dtype is _F32, "scales must be float32", TypeError)
    dev = a.device
    _require(dev == b.device == a_scales.device == b_scales.device, "a, b and their scales must be on one device")
    out = a.new_empty((M, N), dtype=_BF16)
    if M:
        size = _entry("mok_block_matmul_scratch_bytes")(M, N, K)
        scratch = a.new_empty((size // 4,), dtype=_F32) if size else None
        launch("block_matmul", _entry("mok_block_matmul"), dev, a_address, a_ld, a_scales.data_ptr(), *a_scales.stride(), b_address, b_ld,
               b_scales.data_ptr(), *b_scales.stride(), tile_rows, M, N, K, out.data_ptr(), N, _address(scratch),
               status_word(dev).data_ptr())
    return out


@torch.library.custom_op("mok::block_matmul", mutates_args=())
def _block_matmul_op(a: torch.Tensor, a_scales: torch.Tensor, b: torch.Tensor, b_scales: torch.Tensor) -> torch.Tensor:
    """D bf16 [M, N] = (a_scales * a) (b_scales * b)^T.

    Inputs:  a e4m3 [M, K], a_scales f32 [M, ceil(K / 128)]; b e4m3 [N, K], b_scales f32 [ceil(N / 128), ceil(K / 128)] or
             [N, ceil(K / 128)]
    """
    return _matmul(a, a_scales, b, b_scales)


def block_matmul(a: tuple[torch.Tensor, torch.Tensor], b: tuple[torch.Tensor, torch.Tensor]) -> torch.Tensor:
    """bf16 [M, N] product of a [M, K] and the transpose of b [N, K], both (codes, scales): a with scales per 1 x 128, b per 128 x
    128 or per 1 x 128.  fp32 sums, one rounding.  Not differentiable, a backward through it raises (see `fp8_linear`)."""
    if _traced():
        return _block_matmul_op(*a, *b)
    return _without_derivative("block_matmul", lambda: _matmul(*a, *b), *a, *b)


class _Fp8Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, quantized_weight):
        need_w, need_x = ctx.needs_input_grad[1], ctx.needs_input_grad[0]
        quantize, multiply = _implementations()
        if quantized_weight is None:
            w, w_scales, w_t, w_t_scales = quantize(weight, BLOCK, need_x)
        else:
            (w, w_scales), (w_t, w_t_scales) = quantized_weight
        xq, x_scales, x_t, x_t_scales = quantize(x, 1, need_w)
        ctx.save_for_backward(*((w_t, w_t_scales) if need_x else (None, None)), *((x_t, x_t_scales) if need_w else (None, None)))
        return multiply(xq, x_scales, w, w_scales)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_y):
        w_t, w_t_scales, x_t, x_t_scales = ctx.saved_tensors
        need_x, need_w = ctx.needs_input_grad[:2]
        quantize, multiply = _implementations()
        q, scales, q_t, scales_t = quantize(d_y, 1, need_w)
        d_w = multiply(q_t, scales_t, x_t, x_t_scales) if need_w else None
        d_x = multiply(q, scales, w_t, w_t_scales) if need_x else None
        return d_x, d_w, None


def _implementations():
    """Quantizer (x, tile_rows, transpose) and product: the ops where the call is traced, else what they run."""
    if _traced():
        return block_quantize, _block_matmul_op
    return lambda x, tile_rows, transpose: _quantize(x, tile_rows, True, transpose), _matmul


def quantize_weight(weight: torch.Tensor, *, transpose: bool = True):
    """What `fp8_linear` reads of a weight [N, K]: 8-bit copies of it and of its transpose (None without), scales per 128 x 128."""
    q = quantize_blocks(weight, tile_rows=BLOCK, transpose=transpose)
    return q if transpose else (q, (None, None))


def fp8_linear(x: torch.Tensor, weight: torch.Tensor, *, quantized_weight=None) -> torch.Tensor:
    """y [T, N] = x [T, K] weight[N, K]^T in 8 bits, differentiable (K and N multiples of 8, x and weight bf16): x, and the incoming
    gradient in the backward, are quantized per 1 x 128 along the dimension that is summed, the weight per 128 x 128.
    The gradient of x uses the 8-bit weight, that of the weight the 8-bit x and gradient, as if quantization were the identity.
    With `quantized_weight` (from `quantize_weight`) the weight is not quantized again: once per optimizer step, or once for
    inference.  Its transposed half is needed where x requires a gradient."""
    _require(weight.ndim == 2 and x.ndim == 2 and x.shape[1] == weight.shape[1], "x and weight must have shapes (T, K) and (N, K)")
    _require(weight.shape[0] > 0 and weight.shape[0] % 8 == 0, "weight's first dimension must be a positive multiple of 8")
    _require(weight.dtype is _BF16, "weight must be bfloat16", TypeError)
    if quantized_weight is not None:
        (w, _), (w_t, _) = quantized_weight
        _require(w.shape == weight.shape, "quantized_weight must be that of weight: codes (N, K)")
        if w_t is None:
            _require(not (torch.is_grad_enabled() and x.requires_grad),
                     "x requires a gradient, for which quantized_weight must hold the transpose (quantize_weight(weight))")
        else:
            _require(w_t.shape == weight.shape[::-1], "quantized_weight must be that of weight: codes of its transpose (K, N)")
    if x.shape[0] == 0:
        return x @ weight.t()
    if _differentiated(x, weight):
        return _Fp8Linear.apply(x, weight, quantized_weight)
    quantize, multiply = _implementations()   # no gradient will be asked for: nothing is made for one
    w, w_scales = quantize(weight, BLOCK, False)[:2] if quantized_weight is None else quantized_weight[0]
    xq, x_scales = quantize(x, 1, False)[:2]
    return multiply(xq, x_scales, w, w_scales)
