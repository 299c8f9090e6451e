"""``torch.library`` registration of cross attention and rotary positions on top of the C-ABI shim.

    cross_attention_forward(query, key, value, key_padding_mask?, attention_mask?, float scale)
        -> (out, lse, packed mask)
    cross_attention_backward(query, key, value, packed, int mask_heads, out, grad_output, lse, float scale)
        -> (grad_query, grad_key, grad_value)
    rotary_turn(x, positions, float[] frequencies, int[] axes, bool interleaved, bool inverse) -> Tensor

They have no counterpart in the reference.  These are what tracing sees and what serves the calls
that ``csrc/torch_host.cpp`` leaves alone; outputs and workspaces come from torch's allocator.
"""

from __future__ import annotations

import ctypes
from typing import Any

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from ._loader import AttentionCall, load_library
from .ops import DTYPE_CODES, NAMESPACE, _raise

__all__ = ["ATTENTION_OPS", "POSITION_CODES", "ROTARY_OP"]

ATTENTION_OPS = ("cross_attention_forward", "cross_attention_backward")
ROTARY_OP = "rotary_turn"

#: codes of the positions' types (``enum msda_b200_dtype``)
POSITION_CODES = {torch.float32: 0, torch.float64: 3, torch.int32: 4, torch.int64: 5}


def _ptr(t: Tensor | None) -> ctypes.c_void_p:
    return ctypes.c_void_p(t.data_ptr() if t is not None else 0)


def _int64s(values) -> ctypes.Array:
    return (ctypes.c_int64 * len(values))(*values)


def _strides(t: Tensor) -> list[int]:
    # an axis of one element may have any stride; it is never taken
    return [0 if n <= 1 else s for n, s in zip(t.shape[:3], t.stride()[:3])]


def _readable(t: Tensor, share: int = 1) -> Tensor:
    """``t`` as the kernels read it: dense last axis, everything else in whole 16-byte vectors, every token (and, where
    ``share`` heads of it meet one key head, every head) at a place of its own."""
    vec = 16 // t.element_size()
    strides = _strides(t)
    if (t.stride(3) == 1 or t.shape[3] <= 1) and t.data_ptr() % 16 == 0 and all(
            s >= 0 and s % vec == 0 for s in strides) and not (
            (strides[1] == 0 and t.shape[1] > 1) or (strides[2] == 0 and share > 1)):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _call(query: Tensor, key: Tensor, value: Tensor, packed: Tensor, mask_heads: int, scale: float) -> AttentionCall:
    B, Q, G, D = query.shape
    _, S, K, _ = key.shape
    return AttentionCall(B, Q, S, G, K, D, _int64s(_strides(query)), _int64s(_strides(key)), _int64s(_strides(value)),
                         packed.data_ptr() if packed.numel() else None, mask_heads, DTYPE_CODES[query.dtype], scale)


def _stream(t: Tensor) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _workspace(shim, call: AttentionCall, backward: bool, like: Tensor) -> Tensor | None:
    nbytes = shim.attention_workspace_bytes(ctypes.byref(call), int(backward))
    return torch.empty(nbytes, dtype=torch.uint8, device=like.device) if nbytes else None


def _check(query: Tensor, key: Tensor, value: Tensor) -> None:
    for name, t in (("query", query), ("key", key), ("value", value)):
        if not t.is_cuda:
            raise RuntimeError("deformops_b200 kernels run on CUDA tensors only (there is no CPU path)")
        if t.device != query.device or t.dtype != query.dtype:
            raise RuntimeError(f"{name} is {t.dtype} on {t.device}, query {query.dtype} on {query.device}")
    if query.dtype not in DTYPE_CODES or query.dtype == torch.float64:
        raise RuntimeError(f"unsupported dtype {query.dtype}; use float32, float16 or bfloat16")


def _mask_heads(mask: Tensor | None) -> int:
    return 0 if mask is None else mask.shape[1] if mask.dim() == 4 else 1


def _pack(shim, query: Tensor, key: Tensor, padding: Tensor | None, mask: Tensor | None) -> Tensor:
    heads = _mask_heads(mask)
    B, Q, S, K = query.shape[0], query.shape[1], key.shape[1], key.shape[2]
    if padding is None and mask is None:
        return torch.empty(0, dtype=torch.uint8, device=query.device)
    packed = torch.empty(shim.attention_mask_bytes(B, Q, S, K, heads), dtype=torch.uint8, device=query.device)
    strides = None
    if mask is not None:
        strides = list(mask.stride())
        strides = [0, 0, *strides] if mask.dim() == 2 else [strides[0], 0, *strides[1:]] if mask.dim() == 3 else strides
    st = shim.attention_pack_mask(
        _ptr(padding), _int64s(padding.stride()) if padding is not None else None, _ptr(mask),
        _int64s(strides) if strides is not None else None, heads, B, Q, S, K, _ptr(packed), query.device.index,
        _stream(query))
    if st != 0:
        _raise(shim, st, "msda_b200_attention_pack_mask")
    return packed


def _forward_cuda(query, key, value, key_padding_mask, attention_mask, scale):
    _check(query, key, value)
    B, Q, G, D = query.shape
    out = torch.empty((B, Q, G * D), dtype=query.dtype, device=query.device)
    lse = torch.empty((B, key.shape[2], Q, G // key.shape[2]), dtype=torch.float32, device=query.device)
    shim = load_library()
    packed = _pack(shim, query, key, key_padding_mask, attention_mask)
    query, key, value = _readable(query, query.shape[2] // key.shape[2]), _readable(key), _readable(value)
    call = _call(query, key, value, packed, _mask_heads(attention_mask), scale)
    workspace = _workspace(shim, call, False, query)
    st = shim.attention_forward(ctypes.byref(call), _ptr(query), _ptr(key), _ptr(value), _ptr(out), _ptr(lse),
                                _ptr(workspace), workspace.numel() if workspace is not None else 0,
                                query.device.index, _stream(query))
    if st != 0:
        _raise(shim, st, "msda_b200_attention_forward")
    return out, lse, packed


def _backward_cuda(query, key, value, packed, mask_heads, out, grad_output, lse, scale):
    _check(query, key, value)
    if grad_output.dtype != query.dtype or not grad_output.is_contiguous():
        raise RuntimeError("grad_output must be contiguous and have the query's dtype")
    grads = [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (query, key, value)]
    shim = load_library()
    query, key, value = _readable(query, query.shape[2] // key.shape[2]), _readable(key), _readable(value)
    out, grad_output = (t if t.data_ptr() % 16 == 0 else t.clone() for t in (out.contiguous(), grad_output))
    call = _call(query, key, value, packed, mask_heads, scale)
    workspace = _workspace(shim, call, True, query)
    st = shim.attention_backward(ctypes.byref(call), _ptr(query), _ptr(key), _ptr(value), _ptr(out),
                                 _ptr(grad_output), _ptr(lse), *map(_ptr, grads), _ptr(workspace),
                                 workspace.numel() if workspace is not None else 0, query.device.index,
                                 _stream(query))
    if st != 0:
        _raise(shim, st, "msda_b200_attention_backward")
    return tuple(grads)


def _forward_meta(query, key, value, key_padding_mask, attention_mask, scale):
    B, Q, G, D = query.shape
    S, K = key.shape[1], key.shape[2]
    # the packed mask's size as msda_b200_attention_mask_bytes has it
    words, lists = (S + 127) // 128 * 4, (2 + (S + 63) // 64 + (S + 127) // 128 + 3) // 4 * 4
    heads = _mask_heads(attention_mask)
    nbytes = 0
    if key_padding_mask is not None or attention_mask is not None:
        key_heads = K if heads > 1 else 1
        nbytes = 4 * B * (key_heads * lists + words * (key_heads + heads * Q))
    return (query.new_empty((B, Q, G * D)), query.new_empty((B, K, Q, G // K), dtype=torch.float32),
            query.new_empty((nbytes,), dtype=torch.uint8))


def _backward_meta(query, key, value, packed, mask_heads, out, grad_output, lse, scale):
    return query.new_empty(query.shape), key.new_empty(key.shape), value.new_empty(value.shape)


def _setup_context(ctx: Any, inputs: tuple[Any, ...], output: tuple[Tensor, ...]) -> None:
    query, key, value, _, mask, ctx.scale = inputs
    ctx.mask_heads = _mask_heads(mask)
    ctx.save_for_backward(query, key, value, *output)


@once_differentiable
def _autograd_backward(ctx: Any, grad_output: Tensor, *_: Any):
    query, key, value, out, lse, packed = ctx.saved_tensors
    with torch.autocast("cuda", enabled=False):
        grads = torch.ops.deformops_b200.cross_attention_backward(
            query, key, value, packed, ctx.mask_heads, out, grad_output.contiguous().type_as(query), lse, ctx.scale)
    return (*grads, None, None, None)


def _rotary_cuda(x, positions, frequencies, axes, interleaved, inverse):
    if not x.is_cuda:
        raise RuntimeError("deformops_b200 kernels run on CUDA tensors only (there is no CPU path)")
    if x.dtype not in DTYPE_CODES or x.dtype == torch.float64:
        raise RuntimeError(f"unsupported dtype {x.dtype}; use float32, float16 or bfloat16")
    if positions.device != x.device:
        raise RuntimeError(f"positions are on {positions.device}, x on {x.device}")
    B, N, G, D = x.shape
    out = torch.empty((B, N, G, D), dtype=x.dtype, device=x.device)
    if x.numel() == 0:
        return out
    if x.stride(3) != 1 and D > 1:
        x = x.contiguous()
    shim = load_library()
    pairs = len(frequencies)
    places = positions if positions.dim() == 3 else positions.unsqueeze(0).expand(B, *positions.shape)
    st = shim.rotary(_ptr(x), _int64s(x.stride()[:3]), _ptr(places), _int64s(places.stride()),
                     POSITION_CODES[positions.dtype], _ptr(out), B, N, G, D, places.shape[2], pairs,
                     (ctypes.c_double * pairs)(*frequencies), (ctypes.c_int * pairs)(*axes), int(interleaved),
                     int(inverse), DTYPE_CODES[x.dtype], x.device.index, _stream(x))
    if st != 0:
        _raise(shim, st, "msda_b200_rotary")
    return out


def _rotary_meta(x, positions, frequencies, axes, interleaved, inverse):
    return x.new_empty(x.shape)


def _rotary_setup(ctx: Any, inputs: tuple[Any, ...], output: Tensor) -> None:
    _, positions, ctx.frequencies, ctx.axes, ctx.interleaved, ctx.inverse = inputs
    ctx.save_for_backward(positions)


def _rotary_backward(ctx: Any, grad_output: Tensor):
    (positions,) = ctx.saved_tensors
    grad = torch.ops.deformops_b200.rotary_turn(grad_output, positions, ctx.frequencies, ctx.axes, ctx.interleaved,
                                                not ctx.inverse)
    return grad, None, None, None, None, None


def _define() -> None:
    namespace = getattr(torch.ops, NAMESPACE)
    if hasattr(namespace, ROTARY_OP):  # survives importlib.reload
        return
    fwd, bwd = (f"{NAMESPACE}::{name}" for name in ATTENTION_OPS)
    torch.library.define(fwd, "(Tensor query, Tensor key, Tensor value, Tensor? key_padding_mask, "
                              "Tensor? attention_mask, float scale) -> (Tensor, Tensor, Tensor)")
    torch.library.define(bwd, "(Tensor query, Tensor key, Tensor value, Tensor packed, int mask_heads, Tensor out, "
                              "Tensor grad_output, Tensor lse, float scale) -> (Tensor, Tensor, Tensor)")
    torch.library.impl(fwd, "CUDA")(_forward_cuda)
    torch.library.impl(bwd, "CUDA")(_backward_cuda)
    torch.library.register_fake(fwd)(_forward_meta)
    torch.library.register_fake(bwd)(_backward_meta)
    torch.library.register_autograd(fwd, _autograd_backward, setup_context=_setup_context)
    turn = f"{NAMESPACE}::{ROTARY_OP}"
    torch.library.define(turn, "(Tensor x, Tensor positions, float[] frequencies, int[] axes, bool interleaved, "
                               "bool inverse) -> Tensor")
    torch.library.impl(turn, "CUDA")(_rotary_cuda)
    torch.library.register_fake(turn)(_rotary_meta)
    torch.library.register_autograd(turn, _rotary_backward, setup_context=_rotary_setup)


_define()
