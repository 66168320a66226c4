"""`apply_rope(xq, xk, freqs_cis)` (reference: triton_kernels/kernels/positional_embedding.py:55-82), and
`apply_rope_axes`, the same rotation straight from position ids."""
from __future__ import annotations

from ctypes import c_int64

import torch
from torch.autograd.function import once_differentiable

from triton_kernels_b200 import _lib


def apply_rope(xq: torch.Tensor, xk: torch.Tensor, freqs_cis: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Applies the per-position 2x2 transforms in `freqs_cis` ([1,1,L,D/2,2,2], fp32) to every
    (even, odd) pair of q and k ([B,H,L,D]).  The table may be any 2x2 matrices, not only
    rotations.  A table with a batch or head dimension other than 1 is rejected (the reference
    kernel silently ignores those dims)."""
    _lib.require_cuda(xq, xk, freqs_cis)
    assert xq.shape == xk.shape and xq.dtype == xk.dtype
    b, h, s, d = xq.shape
    if freqs_cis.numel() != s * (d // 2) * 4:
        raise ValueError(f"freqs_cis must hold one [L, D/2, 2, 2] table, got shape {tuple(freqs_cis.shape)}")
    xq, xk = xq.contiguous(), xk.contiguous()
    f = freqs_cis.to(torch.float32).contiguous()
    xq_out = torch.empty_like(xq)
    xk_out = torch.empty_like(xk)
    _lib.check(
        _lib.load().fluxb_rope(
            _lib.ptr(xq), _lib.ptr(xk), _lib.ptr(f), _lib.ptr(xq_out), _lib.ptr(xk_out), b * h, s, d,
            _lib.dtype_code(xq), _lib.stream_handle(),
        )
    )
    return xq_out, xk_out


_ID_TYPES = {torch.float32: _lib.ID_F32, torch.int32: _lib.ID_I32, torch.int64: _lib.ID_I64}


def _rope_axes(xq, xk, ids, axes_dim, theta: float, backward: bool):
    """Rotates xq and xk (either may be None); the results have the inputs' memory layout."""
    some = xq if xq is not None else xk
    B, _, L, D = some.shape
    args, outs = [], []
    for x in (xq, xk):
        if x is None:
            args += [None, None, None, None, 0]
            outs.append(None)
            continue
        if x.stride(3) != 1:
            x = x.contiguous()
        out = torch.empty_like(x)
        if out.stride(3) != 1:
            out = torch.empty(x.shape, device=x.device, dtype=x.dtype)
        args += [x.data_ptr(), out.data_ptr(), (c_int64 * 3)(*x.stride()[:3]), (c_int64 * 3)(*out.stride()[:3]), x.shape[1]]
        outs.append((out, x))
    id_strides = (c_int64 * 3)(ids.stride(0) if ids.shape[0] > 1 else 0, ids.stride(1), ids.stride(2))
    with _lib.on_device_of(some):
        _lib.check(
            _lib.load().fluxb_rope_axes(
                *args, ids.data_ptr(), _ID_TYPES[ids.dtype], id_strides, B, L, D, (c_int64 * len(axes_dim))(*axes_dim),
                len(axes_dim), theta, int(backward), _lib.dtype_code(some), _lib.stream_handle(),
            )
        )
    return tuple(o[0] if o is not None else None for o in outs)


class _RopeAxes(torch.autograd.Function):
    @staticmethod
    def forward(ctx, xq, xk, ids, axes_dim, theta):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(ids)
        ctx.plan = axes_dim, theta
        return _rope_axes(xq, xk, ids, axes_dim, theta, False)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        dq, dk = (d if need else None for d, need in zip((dq, dk), ctx.needs_input_grad))
        if dq is None and dk is None:
            return None, None, None, None, None
        return *_rope_axes(dq, dk, ctx.saved_tensors[0], *ctx.plan, True), None, None, None


def apply_rope_axes(xq: torch.Tensor, xk: torch.Tensor, ids: torch.Tensor, axes_dim, theta: float = 10000.0
                    ) -> tuple[torch.Tensor, torch.Tensor]:
    """Rotary positions with several axes (time, height, width) from the tokens' position ids:
    `apply_rope(xq, xk, EmbedND(...)(ids))` without the table, and with positions per batch item.

    xq [B, H, L, D] and xk [B, G, L, D], fp32 or bf16, any strides with unit stride on D (other
    layouts are copied); the results have the inputs' layout.  ids: [B, L, n_axes] or
    [1, L, n_axes], float32 (fractions allowed), int32 or int64.  axes_dim: the even number of
    columns of each axis, in order; their sum may be less than D, and the columns behind them are
    copied.  Pair j of an axis of d columns turns by ids * theta^(-2j/d), taken in fp64.
    Differentiable once in xq and xk."""
    _lib.require_cuda(xq, xk, ids)
    _lib.require_same_device(xq, xk, ids)
    axes_dim = tuple(int(d) for d in axes_dim)
    assert xq.dim() == xk.dim() == 4 and xq.dtype == xk.dtype
    B, _, L, D = xq.shape
    assert xk.shape[0] == B and xk.shape[2:] == xq.shape[2:], "xq and xk differ in more than the head count"
    assert ids.dim() == 3 and ids.shape[0] in (1, B) and ids.shape[1:] == (L, len(axes_dim)), (
        f"ids must be [{B} or 1, {L}, {len(axes_dim)}], got {tuple(ids.shape)}")
    if ids.dtype not in _ID_TYPES:
        raise NotImplementedError(f"position ids are float32, int32 or int64, got {ids.dtype}")
    _lib.dtype_code(xq)
    if torch.is_grad_enabled() and (xq.requires_grad or xk.requires_grad):
        return _RopeAxes.apply(xq, xk, ids, axes_dim, float(theta))
    return _rope_axes(xq, xk, ids, axes_dim, float(theta), False)
