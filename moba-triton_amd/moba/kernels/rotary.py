"""Norm of queries and keys per head with the position rotation, in one pass.

What stands between a layer's projections and `moba_attention`: for each head
of each token

    n = x / sqrt(mean(x^2) + eps) * weight       (n = x without a weight)

and the first `2 * cos.shape[1]` features of n turned by the token's position.
No counterpart in the reference, whose inputs come normed and rotated.
"""

import ctypes

import torch
from torch.autograd.forward_ad import unpack_dual
from torch.autograd.function import once_differentiable

from moba import _lib
from moba.device import check_gathered_head_dim

MAX_HEAD_DIM = 1024


def check_weights(q, q_weight, k_weight) -> int:
    """Dtype code of the norm weights, after checking them.

    Raises:
        ValueError: If a weight is not [D], or not float32 / of q's dtype, or
            the two differ in dtype.
    """
    found = None
    for w in (q_weight, k_weight):
        if w is None:
            continue
        if w.ndim != 1 or w.shape[0] != q.shape[-1]:
            raise ValueError(f"norm weight shape {tuple(w.shape)} must be ({q.shape[-1]},)")
        if w.dtype is not torch.float32 and w.dtype is not q.dtype:
            raise ValueError(f"norm weight dtype {w.dtype} must be float32 or {q.dtype}")
        if found is not None and w.dtype is not found:
            raise ValueError(f"norm weight dtypes differ: {found}, {w.dtype}")
        found = w.dtype
    return _lib.DTYPE_CODE[found or torch.float32]


def check_tables(cos, sin, head_dim: int) -> int:
    """Rotated features of the tables cos, sin [positions, rotary / 2] (0
    without tables), after checking them.

    Raises:
        ValueError: If only one is given, they disagree, are not float32, or
            rotate more than head_dim or no multiple of 16 features.
    """
    if cos is None and sin is None:
        return 0
    if cos is None or sin is None:
        raise ValueError("cos and sin go together")
    if cos.ndim != 2 or cos.shape != sin.shape or cos.shape[0] == 0:
        raise ValueError(f"cos / sin must be [positions, rotary / 2], got {tuple(cos.shape)}, "
                         f"{tuple(sin.shape)}")
    if cos.dtype is not torch.float32 or sin.dtype is not torch.float32:
        raise ValueError(f"cos / sin must be float32, got {cos.dtype}, {sin.dtype}")
    rotary = 2 * cos.shape[1]
    if rotary % 16 or rotary > head_dim or rotary == 0:
        raise ValueError(f"{rotary} rotated features: must be a multiple of 16, at most "
                         f"head_dim {head_dim}")
    return rotary


def _check(q, k, cos, sin, positions, q_weight, k_weight):
    """(dtype code of the weights, rotated features)."""
    qs, ks = q.shape, k.shape
    if len(qs) != 4 or len(ks) != 4 or qs[:2] != ks[:2] or qs[3] != ks[3]:
        raise ValueError(f"shape mismatch: {tuple(qs)}, {tuple(ks)}")
    if 0 in qs[2:] or 0 in ks[2:]:
        raise ValueError(f"head counts and head_dim must be positive: {tuple(qs)}, {tuple(ks)}")
    if q.dtype is not k.dtype:
        raise ValueError(f"dtype mismatch: {q.dtype}, {k.dtype}")
    if q.dtype not in _lib.DTYPE_CODE:
        raise ValueError(f"unsupported dtype {q.dtype}")
    d = qs[3]
    ok, reason = check_gathered_head_dim(d, q.element_size())
    if not ok:
        raise ValueError(reason)
    if d > MAX_HEAD_DIM:
        raise ValueError(f"head_dim {d} above {MAX_HEAD_DIM} is not supported")
    code = check_weights(q, q_weight, k_weight)
    rotary = check_tables(cos, sin, d)
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")
        if positions.shape not in (qs[:2], qs[1:2]):
            raise ValueError(f"positions shape {tuple(positions.shape)} must be "
                             f"{tuple(qs[:2])} or ({qs[1]},)")
    elif rotary and cos.shape[0] < qs[1]:
        raise ValueError(f"cos / sin cover {cos.shape[0]} positions, the rows have {qs[1]}")
    return code, rotary


_Strides = ctypes.c_int64 * 6


def _shape_args(q, k, cos, code, eps, interleaved):
    strides = _Strides(*_lib.row_strides(q), *_lib.row_strides(k))
    rotary, length = (0, 0) if cos is None else (2 * cos.shape[1], cos.shape[0])
    b, s, h, d = q.shape
    return (b, s, h, k.shape[2], d, strides, rotary, length, interleaved, eps,
            _lib.DTYPE_CODE[q.dtype], code)


def _forward(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, code):
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    k_out = torch.empty(k.shape, dtype=q.dtype, device=q.device)
    if q_out.numel():
        a = _lib.addr
        _lib.call_on(q.device, "moba_norm_rotate", q.data_ptr(), k.data_ptr(), q_out.data_ptr(),
                     k_out.data_ptr(), a(cos), a(sin), a(positions), a(q_weight), a(k_weight),
                     *_shape_args(q, k, cos, code, eps, interleaved))
    return q_out, k_out


class NormRotateFunction(torch.autograd.Function):
    """Differentiable in q, k and the weights; the inputs are what is kept for
    the backward."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, code):
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.eps, ctx.interleaved, ctx.code = eps, interleaved, code
        return _forward(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, code)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        q, k, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
        gq, gk = _lib.aligned_contiguous(gq), _lib.aligned_contiguous(gk)
        dev = q.device
        dq, dk = (torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (q, k))
        if not dq.numel():
            zero = [None if w is None else torch.zeros_like(w) for w in (q_weight, k_weight)]
            return dq, dk, *zero, None, None, None, None, None, None
        dwq, dwk = (None if w is None else torch.empty(w.shape, dtype=w.dtype, device=dev)
                    for w in (q_weight, k_weight))
        size = 0 if dwq is None and dwk is None else \
            _lib.load().moba_norm_rotate_bwd_workspace_size(q.shape[-1])
        ws = torch.empty(size, device=dev, dtype=torch.uint8)
        _lib.call_on(dev, "moba_norm_rotate_bwd", *map(_lib.addr, (
            gq, gk, q, k, dq, dk, dwq, dwk, cos, sin, positions, q_weight, k_weight)),
            *_shape_args(q, k, cos, ctx.code, ctx.eps, ctx.interleaved), ws.data_ptr(), size)
        return dq, dk, dwq, dwk, None, None, None, None, None, None


def norm_rotate(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor | None,
                sin: torch.Tensor | None, positions: torch.Tensor | None = None,
                q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                eps: float = 1e-6, interleaved: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """Queries and keys normed per head and rotated by position, with gradient
    support for q, k and the weights. Computed in float32, rounded once. In a
    captured graph take the gradients with `torch.autograd.grad`, of leaves that
    no live eager graph shares. Forward-mode derivatives are refused.

    Args:
        q: [B, S, H_q, D]; k: [B, S, H_kv, D]. Any strides (views of one fused
            projection): rows that cannot be read in 16-byte pieces are copied.
        cos, sin: float32 [positions, rotary / 2], rotary a multiple of 16 of
            at most D; None: no rotation.
        positions: int32 / int64 [B, S] or [S]; None: 0, 1, .. in each row. A
            position outside the tables gives NaN in the rotated features.
        q_weight, k_weight: [D], float32 or of q's dtype; None: that tensor is
            not normed.
        interleaved: Rotate neighbours (2i, 2i + 1) instead of halves
            (i, i + rotary / 2).

    Returns:
        (q, k), contiguous, in their dtype.

    Raises:
        ValueError: On mismatched shapes, dtypes, tables or weights.
        RuntimeError: On dual tensors (forward-mode).
    """
    code, rotary = _check(q, k, cos, sin, positions, q_weight, k_weight)
    _lib.require_gpu(q, k, q_weight, k_weight, cos, sin, positions)
    q, k = _lib.aligned_rows(q), _lib.aligned_rows(k)
    if rotary:
        cos, sin = _lib.aligned_contiguous(cos), _lib.aligned_contiguous(sin)
    if q_weight is not None:
        q_weight = q_weight.contiguous()
    if k_weight is not None:
        k_weight = k_weight.contiguous()
    if positions is not None and (positions.dtype is not torch.int32 or positions.ndim != 2 or
                                  not positions.is_contiguous()):
        if positions.dtype is torch.int64:  # far positions stay outside the tables
            positions = positions.clamp(-1, 2 ** 31 - 1)
        positions = positions.to(torch.int32).expand(q.shape[:2]).contiguous()
    args = (q, k, q_weight, k_weight, cos, sin, positions, float(eps), bool(interleaved), code)
    grad = torch.is_grad_enabled()
    for t in (q, k, q_weight, k_weight):
        # Tangents of forward-mode go there too, to be refused.
        if t is not None and (grad and t.requires_grad or unpack_dual(t).tangent is not None):
            return NormRotateFunction.apply(*args)
    return _forward(*args)
