"""`layer_norm_modulation` and `rms_norm` (reference: triton_kernels/kernels/normalization.py), and
`layer_norm`, which the reference does not have."""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from triton_kernels_b200 import _lib


def _vec(t: torch.Tensor) -> int:
    return 8 if t.dtype == torch.bfloat16 else 4


def layer_norm_modulation_into(x2d, scale2d, shift2d, y2d, rows_per_batch: int, eps: float) -> None:
    """x2d/y2d: [rows, C] views (row stride free); scale2d/shift2d: [B, C] views with a common
    batch stride (chunks of the packed modulation tensor are fine)."""
    rows, C = x2d.shape
    assert scale2d.stride(0) == shift2d.stride(0) or scale2d.shape[0] == 1
    _lib.check(
        _lib.load().fluxb_layer_norm_modulation(
            _lib.ptr(x2d), _lib.ptr(scale2d), _lib.ptr(shift2d), _lib.ptr(y2d), rows, C, rows_per_batch,
            x2d.stride(0), y2d.stride(0), scale2d.stride(0) if scale2d.shape[0] > 1 else 0, eps,
            _lib.dtype_code(x2d), _lib.stream_handle(),
        )
    )


def _dense16(t: torch.Tensor) -> torch.Tensor:
    """t contiguous and 16-byte aligned; a copy where it is not."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x as [rows, C] with unit column stride and 16-byte aligned rows (of whole 16-byte pieces); a
    view where the rows are evenly spaced."""
    C = x.shape[-1]
    if x.dim() == 2 and x.stride(1) == 1 and x.stride(0) >= C and x.stride(0) % _vec(x) == 0 and x.data_ptr() % 16 == 0:
        return x
    return _dense16(x).view(-1, C)


def _norm_backward(dy, x2, factor2, mean, rstd, unit: float, groups: int, want_dx: bool, want_sums: bool, grads_dtype):
    """(dx [rows, C] or None, dfactor, doffset [groups, C] or None) through fluxb_layer_norm_bwd.
    factor2: [groups, C] view with unit column stride, or None (ones)."""
    rows, C = x2.shape
    dy2 = _rows(dy)
    lib = _lib.load()
    dx = torch.empty((rows, C), device=x2.device, dtype=x2.dtype) if want_dx else None
    df = do = scratch = None
    per_group = rows // groups if groups else 0
    if want_sums:
        make = torch.zeros if rows == 0 else torch.empty
        df, do = make((2, groups, C), device=x2.device, dtype=grads_dtype).unbind(0)
        scratch = torch.empty(lib.fluxb_layer_norm_bwd_scratch(rows, C, per_group), device=x2.device, dtype=torch.float32)
    with _lib.on_device_of(x2):
        _lib.check(
            lib.fluxb_layer_norm_bwd(
                _lib.ptr(dy2), _lib.ptr(x2), _lib.ptr(factor2), _lib.ptr(mean), _lib.ptr(rstd), _lib.ptr(dx), _lib.ptr(df),
                _lib.ptr(do), _lib.ptr(scratch), rows, C, per_group, dy2.stride(0), x2.stride(0), C,
                factor2.stride(0) if factor2 is not None and groups > 1 else 0, unit,
                int(grads_dtype == torch.float32), _lib.dtype_code(x2), _lib.stream_handle(),
            )
        )
    return dx, df, do


def _layer_norm_forward(x, weight, bias, eps, stats: bool):
    """(x as rows, y, mean, rstd) of `layer_norm`; mean and rstd are None without `stats`."""
    C = x.shape[-1]
    x2 = _rows(x)
    rows = x2.shape[0]
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    mean = rstd = None
    if stats:
        mean, rstd = torch.empty((2, rows), device=x.device, dtype=torch.float32).unbind(0)
    with _lib.on_device_of(x):
        _lib.check(
            _lib.load().fluxb_layer_norm(
                _lib.ptr(x2), _lib.ptr(weight), _lib.ptr(bias), _lib.ptr(y), _lib.ptr(mean), _lib.ptr(rstd), rows, C, rows,
                x2.stride(0), C, 0, 0.0, eps, _lib.dtype_code(x), _lib.stream_handle(),
            )
        )
    return x2, y, mean, rstd


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x2, y, mean, rstd = _layer_norm_forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x2, weight, mean, rstd)
        ctx.shape = x.shape
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x2, weight, mean, rstd = ctx.saved_tensors
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        dx, dw, db = _norm_backward(dy, x2, weight[None], mean, rstd, 0.0, 1, need_x,
                                    need_w or need_b, x2.dtype)
        return dx.view(ctx.shape) if need_x else None, dw[0] if need_w else None, db[0] if need_b else None, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """LayerNorm over the last dim with a learned scale and offset ([C] each, or None), for fp32 or
    bf16 tensors of any width; weight and bias have x's dtype.  Statistics are fp32, taken as the
    mean and then the centred variance.  Differentiable once in x, weight and bias; the scale's and
    the offset's gradients are summed in fp32 in a fixed order.  (No counterpart in the reference,
    whose only LayerNorm is the modulated one.)"""
    _lib.require_cuda(x, weight, bias)
    _lib.require_same_device(x, weight, bias)
    for p in (weight, bias):
        if p is not None:
            assert p.shape == x.shape[-1:], "weight and bias are vectors of x's last dim"
            assert p.dtype == x.dtype, "Incompatible dtypes"
    _lib.dtype_code(x)
    C = x.shape[-1:]
    weight = torch.ones(C, device=x.device, dtype=x.dtype) if weight is None else _dense16(weight)
    bias = torch.zeros(C, device=x.device, dtype=x.dtype) if bias is None else _dense16(bias)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _LayerNorm.apply(x, weight, bias, eps)
    return _layer_norm_forward(x, weight, bias, eps, False)[1]


def _ln_mod_forward(x, weight, bias, eps, stats: bool):
    """(x as rows, scale as [B, C], y, mean, rstd) of `layer_norm_modulation`; mean and rstd are
    None without `stats`."""
    B, C = x.shape[0], x.shape[-1]
    x = x.contiguous()
    v = _vec(x)
    w2 = weight.reshape(B, C).to(x.dtype)
    b2 = bias.reshape(B, C).to(x.dtype)

    def ok(t):
        return t.stride(1) == 1 and t.stride(0) % v == 0 and t.data_ptr() % 16 == 0

    if not (ok(w2) and ok(b2) and (B == 1 or w2.stride(0) == b2.stride(0))):
        w2, b2 = w2.contiguous(), b2.contiguous()
    y = torch.empty_like(x)
    x2 = x.reshape(-1, C)
    rows = x2.shape[0]
    per_batch = rows // B if B else 0
    mean = rstd = None
    if stats:
        mean, rstd = torch.empty((2, rows), device=x.device, dtype=torch.float32).unbind(0)
    with _lib.on_device_of(x):
        if C % v or x.data_ptr() % 16:  # rows that no 16-byte piece fits: the kernels for any width
            _lib.check(
                _lib.load().fluxb_layer_norm(
                    _lib.ptr(x2), _lib.ptr(w2), _lib.ptr(b2), _lib.ptr(y), _lib.ptr(mean), _lib.ptr(rstd), rows, C, per_batch,
                    C, C, w2.stride(0) if B > 1 else 0, 1.0, eps, _lib.dtype_code(x), _lib.stream_handle(),
                )
            )
        elif stats:
            _lib.check(
                _lib.load().fluxb_layer_norm_modulation_stats(
                    _lib.ptr(x2), _lib.ptr(w2), _lib.ptr(b2), _lib.ptr(y), _lib.ptr(mean), _lib.ptr(rstd), rows, C, per_batch,
                    C, C, w2.stride(0) if B > 1 else 0, eps, _lib.dtype_code(x), _lib.stream_handle(),
                )
            )
        else:
            layer_norm_modulation_into(x2, w2, b2, y.reshape(-1, C), per_batch, eps)
    return x2, w2, y, mean, rstd


class _LayerNormModulation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x2, w2, y, mean, rstd = _ln_mod_forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x2, w2, mean, rstd)
        ctx.shapes = x.shape, weight.shape, bias.shape
        ctx.dtypes = weight.dtype, bias.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x2, w2, mean, rstd = ctx.saved_tensors
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        # a scale kept in another type than the rows gets its gradient from the fp32 sums
        sums = x2.dtype if ctx.dtypes == (x2.dtype, x2.dtype) else torch.float32
        dx, dw, db = _norm_backward(dy, x2, w2, mean, rstd, 1.0, w2.shape[0], need_x, need_w or need_b, sums)
        return (dx.view(ctx.shapes[0]) if need_x else None,
                dw.reshape(ctx.shapes[1]).to(ctx.dtypes[0]) if need_w else None,
                db.reshape(ctx.shapes[2]).to(ctx.dtypes[1]) if need_b else None, None)


def layer_norm_modulation(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    """LayerNorm(x) without affine, then `* (1 + weight) + bias` with weight/bias of shape
    [B, 1, C] broadcast over the sequence (reference :47-77; its default eps 1e-5 is kept).
    Statistics are fp32 whatever the storage dtype (rows of 2-24 KB: sum and sum of squares in
    one pass, fp32 rows shifted by their first element; other widths: mean, then centred variance).
    Differentiable once in x, weight and bias (the reference's is forward only)."""
    assert x.shape[0] == weight.shape[0] == bias.shape[0]
    assert x.shape[-1] == weight.shape[-1] == bias.shape[-1]
    _lib.require_cuda(x, weight, bias)
    _lib.require_same_device(x, weight, bias)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or bias.requires_grad):
        return _LayerNormModulation.apply(x, weight, bias, eps)
    return _ln_mod_forward(x, weight, bias, eps, False)[2]


class _rms_norm(torch.autograd.Function):
    """Forward and backward of RMSNorm over the last dim (reference :142-190)."""

    @staticmethod
    def forward(ctx, x: torch.Tensor, scale: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
        assert x.shape[-1] == scale.shape[-1]
        _lib.require_cuda(x, scale)
        N = x.shape[-1]
        v = _vec(x)
        # Up to 3 leading dims are addressed through strides (head-split views need no copy).
        lead = x.shape[:-1]
        strided_ok = (
            x.dim() <= 4 and x.stride(-1) == 1 and all(s % v == 0 for s in x.stride()[:-1]) and x.data_ptr() % 16 == 0
        )
        if not strided_ok:
            x = x.contiguous()
        dims = [1] * (3 - len(lead)) + list(lead)
        strides = [0] * (3 - len(lead)) + list(x.stride()[:-1])
        # decided on the caller's tensors: the cast copy of `scale` below never requires grad
        need_grad = any(ctx.needs_input_grad[:2])
        ctx.scale_dtype = scale.dtype
        scale = scale.to(x.dtype).contiguous()
        y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
        M = y.numel() // N
        rstd = torch.empty((M,), dtype=torch.float32, device=x.device) if need_grad else None
        _lib.check(
            _lib.load().fluxb_rms_norm(
                _lib.ptr(x), _lib.ptr(scale), _lib.ptr(y), _lib.ptr(rstd), dims[0], dims[1], dims[2], N,
                strides[0], strides[1], strides[2], eps, _lib.dtype_code(x), _lib.stream_handle(),
            )
        )
        if need_grad:
            ctx.save_for_backward(x, scale, rstd)
        return y

    @staticmethod
    def backward(ctx, dy: torch.Tensor):
        x, w, rstd = ctx.saved_tensors
        N = x.shape[-1]
        xc = x.contiguous().reshape(-1, N)
        dyc = dy.contiguous().reshape(-1, N).to(x.dtype)
        M = xc.shape[0]
        lib = _lib.load()
        dx = torch.empty_like(xc)
        parts = lib.fluxb_rms_norm_bwd_partial_rows(M)
        dw_partial = torch.empty((parts, N), dtype=torch.float32, device=x.device)
        _lib.check(
            lib.fluxb_rms_norm_bwd(
                _lib.ptr(dyc), _lib.ptr(xc), _lib.ptr(w), _lib.ptr(rstd), _lib.ptr(dx), _lib.ptr(dw_partial),
                M, N, _lib.dtype_code(xc), _lib.stream_handle(),
            )
        )
        dw = dw_partial.sum(dim=0).to(ctx.scale_dtype)
        return dx.reshape(x.shape), dw, None


rms_norm = _rms_norm.apply
