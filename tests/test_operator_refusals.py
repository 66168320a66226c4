"""What the LayerNorm, rotary-position and adapter entry points refuse, on the host, before anything is launched.
Pointers here are numbers that no call may follow."""
from ctypes import c_int64

import pytest
import torch

P = 1 << 20  # an aligned address, never followed


def ln(lib, rows=4, cols=64, per=4, x=P, y=P, mean=None, rstd=None, x_ld=64, y_ld=64, dtype=1):
    return lib.fluxb_layer_norm(x, P, P, y, mean, rstd, rows, cols, per, x_ld, y_ld, 0, 0.0, 1e-5, dtype, None)


def ln_bwd(lib, rows=4, cols=64, per=4, dy=P, scratch=P, dx_ld=64, dtype=1):
    return lib.fluxb_layer_norm_bwd(dy, P, P, P, P, P, P, P, scratch, rows, cols, per, 64, 64, dx_ld, 0, 0.0, 0, dtype, None)


def test_layer_norm(lib):
    from triton_kernels_b200 import _lib

    assert ln(lib, rows=0, per=0, x=None, y=None) == 0 and ln_bwd(lib, rows=0, per=0, dy=None) == 0
    assert ln(lib, dtype=7) == ln_bwd(lib, dtype=7) == _lib.ERR_UNSUPPORTED
    for bad in (dict(cols=0), dict(rows=-1), dict(per=3), dict(per=0), dict(x=None), dict(y=None), dict(mean=P), dict(y_ld=63), dict(x=P + 1)):
        assert ln(lib, **bad) == _lib.ERR_BAD_ARG, bad
    for bad in (dict(cols=0), dict(rows=-1), dict(per=3), dict(dy=None), dict(scratch=None), dict(dx_ld=8), dict(dy=P + 1)):
        assert ln_bwd(lib, **bad) == _lib.ERR_BAD_ARG, bad
    assert ln(lib, rows=1 << 40, per=1 << 40) == ln(lib, cols=1 << 30, y_ld=1 << 30, x_ld=1 << 30) == _lib.ERR_UNSUPPORTED
    assert lib.fluxb_layer_norm_bwd_scratch(0, 64, 0) == 0 and lib.fluxb_layer_norm_bwd_scratch(64, 128, 32) % 256 == 0
    assert lib.fluxb_layer_norm_modulation_stats(P, P, P, P, None, None, 4, 64, 4, 64, 64, 0, 1e-6, 1, None) == _lib.ERR_BAD_ARG


def rope(lib, axes=(16, 48), B=1, L=4, D=64, H=2, q=P, ids=P, id_type=0, theta=1e4, dtype=1, n=None):
    s = (512, 256, 64)
    return lib.fluxb_rope_axes(q, *s, P, *s, H, P, *s, P, *s, H, ids, id_type, 8, 2, 1, B, L, D, (c_int64 * len(axes))(*axes),
                               len(axes) if n is None else n, theta, 0, dtype, None)


def test_rope_axes(lib):
    from triton_kernels_b200 import _lib

    assert rope(lib, L=0, q=None, ids=None) == rope(lib, B=0) == 0
    for bad in (dict(axes=(15, 49)), dict(axes=(0, 64)), dict(axes=(-2, 64)), dict(axes=(64, 2)), dict(theta=0.0), dict(theta=float("nan")),
                dict(theta=-1.0), dict(q=None), dict(ids=None), dict(D=0, axes=(2,)), dict(B=-1)):
        assert rope(lib, **bad) == _lib.ERR_BAD_ARG, bad
    for bad in (dict(dtype=2), dict(id_type=3), dict(axes=(2,) * 9), dict(n=0), dict(axes=(258,), D=512), dict(B=1 << 20, L=1 << 20)):
        assert rope(lib, **bad) == _lib.ERR_UNSUPPORTED, bad


def lora(lib, B=2, L=3, N=64, K=64, R=8, n=2, ldx=None, ldw=None, ldy=None, ldb=None, x=P, adapter=P, scratch=P, epi=0, a=P):
    return lib.fluxb_linear_lora(x, P, P, P, a, P, None, adapter, 1, scratch, B, L, N, K, R, n, ldx or K, ldw or K, ldy or N, ldb or R, epi, None)


def test_linear_lora(lib):
    from triton_kernels_b200 import _lib

    assert lora(lib, B=0) == lora(lib, L=0) == lora(lib, N=0) == 0
    for bad in (dict(K=0), dict(R=0), dict(n=0), dict(B=-1), dict(K=60), dict(N=60), dict(ldx=60), dict(ldw=56), dict(ldy=56), dict(ldb=4), dict(R=4), dict(x=None),
                dict(adapter=None), dict(scratch=None), dict(x=P + 2), dict(a=P + 8)):
        assert lora(lib, **bad) == _lib.ERR_BAD_ARG, bad
    for bad in (dict(epi=2), dict(R=264), dict(B=1 << 20, L=1 << 20)):
        assert lora(lib, **bad) == _lib.ERR_UNSUPPORTED, bad


def test_wrappers_refuse_cpu_tensors_and_wrong_shapes():
    import triton_kernels_b200 as tk

    x = torch.randn(2, 8, 64)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        tk.layer_norm(x)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        tk.LayerNorm(64)(x)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        tk.apply_rope_axes(x[None], x[None], torch.zeros(1, 8, 1), (64,))
    b = x.bfloat16()
    args = (b, torch.zeros(64, 64).bfloat16(), None, torch.zeros(1, 8, 64).bfloat16(), torch.zeros(1, 64, 8).bfloat16(), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        tk.linear_lora(*args)
    with pytest.raises(AssertionError):
        tk.linear_lora(*args, None, "SILU")
    with pytest.raises(AssertionError):
        tk.linear_lora(*args[:5], torch.zeros(3, dtype=torch.int64))
