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
    """x as evenly spaced rows of its last dim, 16-byte aligned (rows of whole 16-byte pieces): x
    itself where it is contiguous or a 2-D view with a row stride, else a copy."""
    if x.is_contiguous():
        return x if x.data_ptr() % 16 == 0 else x.clone()
    if (x.dim() == 2 and x.stride(1) == 1 and x.stride(0) >= x.shape[1] and x.stride(0) % _vec(x) == 0
            and x.data_ptr() % 16 == 0):
        return x
    return x.contiguous()


def _row_stride(x: torch.Tensor) -> int:
    return x.stride(0) if x.dim() == 2 else x.shape[-1]


def _norm_backward(dy, x, factor, factor_stride: int, stats, unit: float, groups: int, want_dx: bool, df, do, grads_f32: bool):
    """dx (or None), with the groups' gradients of factor and offset left in df and do (or None),
    through fluxb_layer_norm_bwd.  x: as `_rows` gives it; stats: fp32, the rows' means, then their
    reciprocal deviations."""
    lib = _lib.load()
    C = x.shape[-1]
    rows = x.numel() // C
    dy = _rows(dy)
    dx = torch.empty(x.shape, device=x.device, dtype=x.dtype) if want_dx else None
    per_group = rows // groups if groups else 0
    scratch = None
    if df is not None or do is not None:
        scratch = stats.new_empty(lib.fluxb_layer_norm_bwd_scratch(rows, C, per_group))
    mean = stats.data_ptr()
    _lib.launch(
        lib.fluxb_layer_norm_bwd, x.get_device(), dy.data_ptr(), x.data_ptr(), factor.data_ptr(), mean, mean + 4 * rows,
        _lib.ptr(dx), _lib.ptr(df), _lib.ptr(do), _lib.ptr(scratch), rows, C, per_group, _row_stride(dy), _row_stride(x), C,
        factor_stride, unit, int(grads_f32), _lib.DTYPE_CODES[x.dtype],
    )
    return dx


def _layer_norm_forward(x, weight, bias, eps, stats):
    """y of `layer_norm` for x as `_rows` gives it; fills `stats` (see `_norm_backward`) if given."""
    C = x.shape[-1]
    rows = x.numel() // C
    y = torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, device=x.device, dtype=x.dtype)
    mean = rstd = None
    if stats is not None:
        mean = stats.data_ptr()
        rstd = mean + 4 * rows
    _lib.launch(
        _lib.load().fluxb_layer_norm, x.get_device(), x.data_ptr(), weight.data_ptr(), bias.data_ptr(), y.data_ptr(), mean, rstd,
        rows, C, rows, _row_stride(x), C, 0, 0.0, eps, _lib.DTYPE_CODES[x.dtype],
    )
    return y


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x = _rows(x)
        stats = x.new_empty(2 * (x.numel() // x.shape[-1]), dtype=torch.float32)
        y = _layer_norm_forward(x, weight, bias, eps, stats)
        ctx.save_for_backward(x, weight, stats)
        return y

    @staticmethod
    def _backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        make = torch.empty_like if x.numel() else torch.zeros_like
        dw = make(weight) if need_w else None
        db = make(weight) if need_b else None
        return _norm_backward(dy, x, weight, 0, stats, 0.0, 1, need_x, dw, db, False), dw, db, None

    _backward_once = once_differentiable(_backward.__func__)

    @staticmethod
    def backward(ctx, dy):
        # the wrapper that refuses second gradients is asked for only where somebody may take them
        return (_LayerNorm._backward_once if torch.is_grad_enabled() else _LayerNorm._backward)(ctx, dy)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """LayerNorm over the last dim with a learned scale and offset ([C] each, or None), for fp32 or
    bf16 tensors of any width; weight and bias have x's dtype.  Statistics are fp32 (rows of 2-24 KB:
    sum and sum of squares in one pass, shifted by the row's first element; others: mean, then
    centred variance).  Differentiable once in x, weight and bias; the scale's and the offset's
    gradients are summed in fp32 in a fixed order.  (No counterpart in the reference, whose only
    LayerNorm is the modulated one.)"""
    _lib.require_cuda(x, weight, bias)
    _lib.require_same_device(x, weight, bias)
    _lib.dtype_code(x)
    C = x.shape[-1:]
    if weight is None:
        weight = torch.ones(C, device=x.device, dtype=x.dtype)
    if bias is None:
        bias = torch.zeros(C, device=x.device, dtype=x.dtype)
    assert weight.shape == C and bias.shape == C, "weight and bias are vectors of x's last dim"
    assert weight.dtype == bias.dtype == x.dtype, "Incompatible dtypes"
    weight, bias = _dense16(weight), _dense16(bias)
    if (x.requires_grad or weight.requires_grad or bias.requires_grad) and torch.is_grad_enabled():
        return _LayerNorm.apply(x, weight, bias, eps)
    return _layer_norm_forward(_rows(x), weight, bias, eps, None)


def _ln_mod_forward(x, weight, bias, eps, stats):
    """(scale as [B, C], y) of `layer_norm_modulation` for a contiguous x; fills `stats` if given."""
    B, C = x.shape[0], x.shape[-1]
    v = _vec(x)
    w2 = weight.reshape(B, C).to(x.dtype)
    b2 = bias.reshape(B, C).to(x.dtype)

    def ok(t):
        return t.stride(1) == 1 and t.stride(0) % v == 0 and t.data_ptr() % 16 == 0

    if not (ok(w2) and ok(b2) and (B == 1 or w2.stride(0) == b2.stride(0))):
        w2, b2 = w2.contiguous(), b2.contiguous()
    y = torch.empty_like(x)
    rows = x.numel() // C
    per_batch = rows // B if B else 0
    stride = w2.stride(0) if B > 1 else 0
    lib = _lib.load()
    mean = rstd = None
    if stats is not None:
        mean = stats.data_ptr()
        rstd = mean + 4 * rows
    args = x.data_ptr(), w2.data_ptr(), b2.data_ptr(), y.data_ptr()
    code = _lib.dtype_code(x)
    if C % v or x.data_ptr() % 16:  # rows that no 16-byte piece fits: the kernels for any width
        _lib.launch(lib.fluxb_layer_norm, x.get_device(), *args, mean, rstd, rows, C, per_batch, C, C, stride, 1.0, eps, code)
    elif stats is not None:
        _lib.launch(lib.fluxb_layer_norm_modulation_stats, x.get_device(), *args, mean, rstd, rows, C, per_batch, C, C, stride,
                    eps, code)
    else:
        _lib.launch(lib.fluxb_layer_norm_modulation, x.get_device(), *args, rows, C, per_batch, C, C, stride, eps, code)
    return w2, y


class _LayerNormModulation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x = x.contiguous()
        stats = x.new_empty(2 * (x.numel() // x.shape[-1]), dtype=torch.float32)
        w2, y = _ln_mod_forward(x, weight, bias, eps, stats)
        ctx.save_for_backward(x, w2, stats)
        ctx.vectors = weight.shape, weight.dtype, bias.shape, bias.dtype
        return y

    @staticmethod
    def _backward(ctx, dy):
        x, w2, stats = ctx.saved_tensors
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        w_shape, w_dtype, b_shape, b_dtype = ctx.vectors
        # a scale or shift kept in another type than the rows gets its gradient from the fp32 sums
        own = w_dtype == b_dtype == x.dtype
        make = x.new_empty if x.numel() else x.new_zeros
        dw = make(w_shape, dtype=x.dtype if own else torch.float32) if need_w else None
        db = make(b_shape, dtype=x.dtype if own else torch.float32) if need_b else None
        B = w2.shape[0]
        dx = _norm_backward(dy, x, w2, w2.stride(0) if B > 1 else 0, stats, 1.0, B, need_x, dw, db,
                            not own or x.dtype == torch.float32)
        if not own:
            dw, db = dw.to(w_dtype) if need_w else None, db.to(b_dtype) if need_b else None
        return dx, dw, db, None

    _backward_once = once_differentiable(_backward.__func__)

    @staticmethod
    def backward(ctx, dy):
        return (_LayerNormModulation._backward_once if torch.is_grad_enabled() else _LayerNormModulation._backward)(ctx, dy)


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
    if (x.requires_grad or weight.requires_grad or bias.requires_grad) and torch.is_grad_enabled():
        return _LayerNormModulation.apply(x, weight, bias, eps)
    return _ln_mod_forward(x.contiguous(), weight, bias, eps, None)[1]


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
