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


_NOTHING = (None, 0, 0, 0, None, 0, 0, 0, 0)
_axes_arrays = {}  # axes_dim -> the same as a C array


def _rope_axes(xq, xk, ids, axes_dim, theta: float, backward: bool):
    """Rotates xq and xk (either may be None); the results have the inputs' memory layout."""
    args, outs, keep = (), [], []
    for x in (xq, xk):
        if x is None:
            args += _NOTHING
            outs.append(None)
            continue
        if x.stride(3) != 1:
            x = x.contiguous()
            keep.append(x)
        out = torch.empty_like(x)
        if out.stride(3) != 1:  # an input that overlaps itself
            out = torch.empty(x.shape, device=x.device, dtype=x.dtype)
        args += (x.data_ptr(), *x.stride()[:3], out.data_ptr(), *out.stride()[:3], x.shape[1])
        outs.append(out)
    some = outs[0] if xq is not None else outs[1]
    axes = _axes_arrays.get(axes_dim)
    if axes is None:
        axes = _axes_arrays[axes_dim] = (c_int64 * len(axes_dim))(*axes_dim)
    i0, i1, i2 = ids.stride()
    B, _, L, D = some.shape
    _lib.launch(
        _lib.load().fluxb_rope_axes, some.get_device(), *args, ids.data_ptr(), _ID_TYPES[ids.dtype],
        i0 if ids.shape[0] > 1 else 0, i1, i2, B, L, D, axes, len(axes_dim), theta, backward, _lib.DTYPE_CODES[some.dtype],
    )
    return tuple(outs)


class _RopeAxes(torch.autograd.Function):
    @staticmethod
    def forward(ctx, xq, xk, ids, axes_dim, theta):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(ids)
        ctx.plan = axes_dim, theta
        return _rope_axes(xq, xk, ids, axes_dim, theta, False)

    @staticmethod
    def _backward(ctx, dq, dk):
        need_q, need_k = ctx.needs_input_grad[:2]
        dq, dk = dq if need_q else None, dk if need_k else None
        if dq is not None or dk is not None:
            dq, dk = _rope_axes(dq, dk, ctx.saved_tensors[0], *ctx.plan, True)
        return dq, dk, None, None, None

    _backward_once = once_differentiable(_backward.__func__)

    @staticmethod
    def backward(ctx, dq, dk):
        # the wrapper that refuses second gradients is asked for only where somebody may take them
        return (_RopeAxes._backward_once if torch.is_grad_enabled() else _RopeAxes._backward)(ctx, dq, dk)


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
    axes_dim = tuple(axes_dim)
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
