"""Cross attention of queries to all states of an encoder: the dense counterpart of :data:`msda`.

``softmax(scale * query key^T) value`` per head, in one pass that never holds the scores.  The
reference has no such operator; names, checks and errors follow :mod:`deformops_b200.registry.msda`.
"""

from __future__ import annotations

import math

import torch
from torch import Tensor

from .. import attention_ops as _ops  # noqa: F401  (defines the operators)
from .._loader import load_library
from ..core.errors import NoBackendError
from ..core.runtime import sm_version_for
from ..core.sanitize import check_cross_attention_call
from .msda import Backend, _native_path, msda

__all__ = ["cross_attention"]

_VECTOR = {torch.float32: 4, torch.float16: 8, torch.bfloat16: 8}
_MAX_HEAD_DIM = 128


def _unsupported(query: Tensor) -> str | None:
    if query.device.type != "cuda":
        return f"tensors are on {query.device}; the kernels need a CUDA device (no CPU path)"
    major, minor = sm_version_for(query.device)
    if major != 10:
        return f"device has compute capability {major}.{minor}; the kernels are built for sm_100a only"
    if query.dtype not in _VECTOR:
        return f"dtype {query.dtype} is not float32, float16 or bfloat16"
    D = query.shape[3]
    if D == 0 or D % _VECTOR[query.dtype] != 0 or D > _MAX_HEAD_DIM:
        return (f"head dimension {D} is not a multiple of {_VECTOR[query.dtype]} (16-byte channel vectors) up to "
                f"{_MAX_HEAD_DIM}")
    return None


def cross_attention(query: Tensor, key: Tensor, value: Tensor, *, key_padding_mask: Tensor | None = None,
                    attention_mask: Tensor | None = None, scale: float | None = None,
                    backend: Backend | None = None) -> Tensor:
    """``query (B,Q,G,D)``, ``key`` and ``value (B,S,K,D)`` -> ``(B,Q,G*D)``.

    Query head ``g`` meets key head ``g // (G / K)``; ``K`` divides ``G``.  ``scale`` defaults to
    ``D ** -0.5`` and must be positive.  Both masks are bool and true where a state may *not* be seen:
    ``key_padding_mask (B,S)`` for all queries, ``attention_mask`` ``(Q,S)``, ``(B,Q,S)`` or
    ``(B,1|G,Q,S)`` for each.  A query that may see nothing gets zeros, and so do its gradients;
    states that no query may see may hold anything, NaN as well (states that some query
    may see must be finite).  Scores, times ``scale``, are float32: of 10^6 they leave weights a few per cent
    off in the backward pass, and above 10^7 results and gradients need not be finite.  Strides are free; what the kernels cannot read in 16-byte vectors is
    copied, and so are tokens expanded from one.

    Gradients flow to query, key and value, once.  The same call gives the same bits every time.
    Raises ``ValueError`` for operands that disagree in rank, size, dtype or device and
    :class:`NoBackendError` for what the kernels do not take (the message says why).
    """
    if backend is None or backend is Backend.CUDA:
        native = _native_path(query)
        if native is not None and (scale is None or type(scale) is float):
            out = native.cross_attention(query, key, value, key_padding_mask, attention_mask, scale)
            if out is not None:
                return out
    msda._only_cuda(backend)
    check_cross_attention_call(query, key, value, key_padding_mask, attention_mask)
    reason = _unsupported(query)
    if reason is not None:
        raise NoBackendError(f"cross_attention cannot run this call: {reason}")
    scale = query.shape[3] ** -0.5 if scale is None else float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    load_library()
    with torch.autocast("cuda", enabled=False):
        return torch.ops.deformops_b200.cross_attention_forward(query, key, value, key_padding_mask, attention_mask,
                                                                scale)[0]
