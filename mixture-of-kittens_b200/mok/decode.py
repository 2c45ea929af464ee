"""The MoE layer and its router for a few tokens (1 to 256): what a serving step calls, where `mok.functional.forward` asks for 512
tokens or more.  No counterpart in the reference.

No workspace, schedule or process group: a call is a function of its tensors, on the current stream, and can be captured in a
graph.  A token's result does not depend on the other tokens of its batch.
"""
from __future__ import annotations

import torch

from ._native import entry as _entry
from ._native import launch, status_word
from .block_ops import BLOCK, E4M3, _address, _like, _rows, _traced, _without_derivative
from .ops import _require

MAX_TOKENS, MAX_TOPK, MAX_ROUTES, MAX_EXPERTS = 256, 32, 4096, 1024
_BF16, _F32 = torch.bfloat16, torch.float32


# A step of one token takes 40 us on the GPU: the checks below build their messages only where they fail.
def _check_tokens(x: torch.Tensor, multiple: int) -> None:
    _require(x.ndim == 2, "x must have shape (num_tokens, hidden_size)")
    T, H = x.shape
    _require(T <= MAX_TOKENS, "num_tokens must be at most 256 (mok.functional.forward takes 512 and more)")
    if H <= 0 or H % multiple:
        raise ValueError(f"hidden_size must be a positive multiple of {multiple}")
    _require(x.is_cuda, "x must be a CUDA tensor")
    _require(x.dtype is _BF16, "x must be bfloat16", TypeError)


# ------------------------------------------------------------------------------------------------------------
# router
# ------------------------------------------------------------------------------------------------------------
def _route(x, w_router, bias, topk):
    _check_tokens(x, 8)
    T, H = x.shape
    _require(w_router.ndim == 2 and w_router.shape[1] == H, "w_router must have shape (num_experts, hidden_size)")
    E = w_router.shape[0]
    _require(0 < E <= MAX_EXPERTS, "num_experts must be in [1, 1024]")
    _require(type(topk) is int and 0 < topk <= min(E, MAX_TOPK), "topk must be an integer in [1, min(num_experts, 32)]")
    _require(w_router.device == x.device, "w_router must be on the device of x")
    _require((w_router.dtype is _F32 or w_router.dtype is _BF16) and w_router.is_contiguous(), "w_router must be contiguous float32 or bfloat16",
             TypeError)
    if bias is not None:
        _require(bias.shape == (E,) and bias.device == x.device, "bias must have shape (num_experts,) on the device of x")
        _require(bias.dtype is _F32 and bias.is_contiguous(), "bias must be contiguous float32", TypeError)
    routes = x.new_empty((T, topk), dtype=torch.int32)
    weights = x.new_empty((T, topk), dtype=_F32)
    if T:
        x = _rows(x)
        if w_router.data_ptr() % 16:
            w_router = w_router.clone()
        logits = x.new_empty((T, E), dtype=_F32)
        launch("router_decode", _entry("mok_router_decode"), x.device, x.data_ptr(), x.stride(0), w_router.data_ptr(), w_router.dtype is _F32,
               _address(bias), T, H, E, topk, logits.data_ptr(), routes.data_ptr(), weights.data_ptr())
    return routes, weights


@torch.library.custom_op("mok::router_decode", mutates_args=())
def router_decode(x: torch.Tensor, w_router: torch.Tensor, bias: torch.Tensor | None, topk: int) -> tuple[torch.Tensor, torch.Tensor]:
    """router_fwd for 0 to 256 tokens, in fp32 throughout: top-k of x @ w_router.T (+ bias), softmax over the selected logits.

    Inputs:  x bf16 [T, H] (H % 8 == 0); w_router f32 | bf16 [E, H]; bias f32 [E] | None; topk int
    Outputs: top_experts int32 [T, topk] (descending, ties to the lower index); router_weights f32 [T, topk]
    """
    return _route(x, w_router, bias, topk)


def route_decode(x: torch.Tensor, w_router: torch.Tensor, bias: torch.Tensor | None = None, *, topk: int) -> tuple[torch.Tensor, torch.Tensor]:
    """`mok.route` for a few tokens: (top_experts int32 [T, topk], router_weights fp32 [T, topk]), chosen as torch.topk does.  Not
    differentiable: a backward through it raises."""
    if _traced():
        return router_decode(x, w_router, bias, topk)
    return _without_derivative("route_decode", lambda: _route(x, w_router, bias, topk), x, w_router, bias)


# ------------------------------------------------------------------------------------------------------------
# layer
# ------------------------------------------------------------------------------------------------------------
def _weight(name: str, w: torch.Tensor, shape, device, dtype) -> int:
    """The weight's address."""
    address = w.data_ptr()
    if w.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}")
    if w.device != device:
        raise ValueError(f"{name} must be on the device of x")
    if w.dtype is not dtype or address % 16 or not w.is_contiguous():
        raise TypeError(f"{name} must be contiguous {dtype}, 16-byte aligned")
    return address


def _decode(x, top_experts, router_weights, shared, routed, scales, first_expert, swiglu_limit):
    _check_tokens(x, 64)
    T, H = x.shape
    dev = x.device
    _require(top_experts.ndim == 2 and top_experts.shape[0] == T, "top_experts must have shape (num_tokens, topk)")
    K = top_experts.shape[1]
    _require(0 < K <= MAX_TOPK, "topk must be in [1, 32]")
    _require(T * K <= MAX_ROUTES, "num_tokens * topk must be at most 4096")
    _require(top_experts.dtype is torch.int32 or top_experts.dtype is torch.int64, "top_experts must be int32 or int64", TypeError)
    _require(router_weights.shape == (T, K), "router_weights must have shape (num_tokens, topk)")
    _require(router_weights.dtype is _F32, "router_weights must be float32", TypeError)
    _require(top_experts.device == dev and router_weights.device == dev, "top_experts and router_weights must be on the device of x")
    _require(type(first_expert) is int and first_expert >= 0, "first_expert must be a non-negative integer")
    _require(swiglu_limit is None or (type(swiglu_limit) in (int, float) and swiglu_limit >= 0), "swiglu_limit must be None or a non-negative number")
    gate, up, down = routed
    _require(gate.ndim == 3 and 0 < gate.shape[0] <= MAX_EXPERTS, "w_routed_gate must have shape (num_experts, intermediate_size, hidden_size)")
    E, I = gate.shape[:2]
    _require(I > 0 and I % 64 == 0, "intermediate_size must be a positive multiple of 64")
    w8 = scales[0] is not None
    _require((scales[1] is not None) == w8 == (scales[2] is not None), "the routed weights must be all bfloat16 or all (codes, scales)", TypeError)
    dtype = E4M3 if w8 else _BF16
    up_shape, down_shape = (E, I, H), (E, H, I)
    weights = (_weight("w_routed_gate", gate, up_shape, dev, dtype), _weight("w_routed_up", up, up_shape, dev, dtype),
               _weight("w_routed_down", down, down_shape, dev, dtype))
    if w8:
        h, i = -(-H // BLOCK), -(-I // BLOCK)
        weights += (_weight("scales of w_routed_gate", scales[0], (E, i, h), dev, _F32), _weight("scales of w_routed_up", scales[1], (E, i, h), dev, _F32),
                    _weight("scales of w_routed_down", scales[2], (E, h, i), dev, _F32))
    else:
        weights += (None, None, None)
    sg, su, sd = shared
    _require((sg is None) == (su is None) == (sd is None), "the three shared weights must be given together")
    shared_i, shared_weights = 0, (None, None, None)
    if sg is not None:
        _require(sg.ndim == 2, "w_shared_gate must have shape (shared_intermediate_size, hidden_size)")
        shared_i = sg.shape[0]
        _require(shared_i > 0 and shared_i % 64 == 0, "shared_intermediate_size must be a positive multiple of 64")
        shared_weights = (_weight("w_shared_gate", sg, (shared_i, H), dev, _BF16), _weight("w_shared_up", su, (shared_i, H), dev, _BF16),
                          _weight("w_shared_down", sd, (H, shared_i), dev, _BF16))
    out = _like(x)
    if T == 0:
        return out
    x = _rows(x)
    if top_experts.dtype is torch.int64:   # a number beyond 32 bits is no expert's; it must not become one
        top_experts = top_experts.clamp(-1, 2 ** 31 - 1).to(torch.int32)
    top_experts, router_weights = top_experts.contiguous(), router_weights.contiguous()
    scratch = x.new_empty((_entry("mok_moe_decode_scratch_bytes")(T, K, H, I, shared_i, w8) // 2,))
    launch("moe_decode", _entry("mok_moe_decode"), dev, x.data_ptr(), x.stride(0), top_experts.data_ptr(), router_weights.data_ptr(), T, K, H,
           *shared_weights, shared_i, *weights, I, E, first_expert, swiglu_limit is not None,
           0.0 if swiglu_limit is None else float(swiglu_limit), out.data_ptr(), scratch.data_ptr(), status_word(dev).data_ptr())
    return out


@torch.library.custom_op("mok::moe_decode", mutates_args=())
def _moe_decode_op(x: torch.Tensor, top_experts: torch.Tensor, router_weights: torch.Tensor, w_shared_gate: torch.Tensor | None,
                   w_shared_up: torch.Tensor | None, w_shared_down: torch.Tensor | None, w_routed_gate: torch.Tensor,
                   w_routed_gate_sc: torch.Tensor | None, w_routed_up: torch.Tensor, w_routed_up_sc: torch.Tensor | None,
                   w_routed_down: torch.Tensor, w_routed_down_sc: torch.Tensor | None, first_expert: int, swiglu_limit: float | None
                   ) -> torch.Tensor:
    """The layer for 0 to 256 tokens; see `moe_decode`."""
    return _decode(x, top_experts, router_weights, (w_shared_gate, w_shared_up, w_shared_down), (w_routed_gate, w_routed_up, w_routed_down),
                   (w_routed_gate_sc, w_routed_up_sc, w_routed_down_sc), first_expert, swiglu_limit)


def _pair(w):
    return w if isinstance(w, tuple) else (w, None)


def moe_decode(x: torch.Tensor, top_experts: torch.Tensor, router_weights: torch.Tensor,
               w_shared_gate: torch.Tensor | None, w_shared_up: torch.Tensor | None, w_shared_down: torch.Tensor | None,
               w_routed_gate, w_routed_up, w_routed_down, *, first_expert: int = 0, swiglu_limit: float | None = None) -> torch.Tensor:
    """MoE layer for a few tokens: out bf16 [T, H] = shared(x) + sum over k of router_weights[t, k] * expert(top_experts[t, k])(x),
    with expert(x) = W_down (silu(W_gate x) * (W_up x)).

    x bf16 [T, H], T <= 256; top_experts int32 or int64 [T, K]; router_weights fp32 [T, K]; shared weights bf16 [I', H], [I', H],
    [H, I'] or None; routed weights bf16 [E, I, H], [E, I, H], [E, H, I], or each (codes, scales) from `mok.quantize_blocks(w,
    tile_rows=128)` (e4m3, any fp32 scale per 128 x 128), which halves the bytes that a step reads.  H, I and I' are multiples of 64.

    The routed weights are those of experts first_expert .. first_expert + E - 1.  Routes to other experts (other ranks', or any
    number that is no expert's, such as -1) contribute nothing: expert-parallel ranks sum their outputs.  An expert that a token
    names twice counts with the sum of both weights.  With `swiglu_limit` gate is clamped from above and up from both sides.
    hidden is rounded to bf16 between the products, as in the layer; sums are fp32.  The output is NaN while the device status word reports a
    problem, like that of `mok.functional.forward`.  Not differentiable: a backward through it raises."""
    (g, gs), (u, us), (d, ds) = _pair(w_routed_gate), _pair(w_routed_up), _pair(w_routed_down)
    shared = (w_shared_gate, w_shared_up, w_shared_down)
    if _traced():
        return _moe_decode_op(x, top_experts, router_weights, *shared, g, gs, u, us, d, ds, first_expert, swiglu_limit)
    return _without_derivative(
        "moe_decode", lambda: _decode(x, top_experts, router_weights, shared, (g, u, d), (gs, us, ds), first_expert, swiglu_limit),
        x, router_weights, *shared, g, gs, u, us, d, ds)
