"""Tensors of more than 2^31 elements: what lies behind that offset, against the same call on a copy of that part alone.

The part alone may run on another kernel, so two results of one value are two roundings to bf16 of fp32 numbers that differ
in the order of their sums: at most one step (2^-7 of the value) and the difference before rounding apart.  That one is
below 2^-10 here: sums of 64 to 2944 terms of the size of one, each off by 2^-24 of the terms' sum, and for the adapters the
low-rank rows' 2^-17.  The rotation has no sums: the same bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.fixture(scope="module")
def tk(lib):
    import triton_kernels_b200 as tk

    assert torch.cuda.is_available()
    yield tk
    torch.cuda.empty_cache()


@pytest.fixture(autouse=True)
def seed():
    torch.manual_seed(91)


def normal(*shape):
    return torch.empty(*shape, device="cuda", dtype=BF).normal_()


def close(a, b):
    return bool(((a.double() - b.double()).abs() <= 2.0**-7 * b.double().abs() + 2.0**-10).all())


@pytest.mark.parametrize("C", [2944, 2701])
def test_layer_norm(tk, C):
    rows, part = 2**31 // C + 6000, 5000
    x, dy, w, b = normal(rows, C), normal(rows, C), normal(C), normal(C)
    assert x.numel() > 2**31
    x.requires_grad_(True)
    y = tk.layer_norm(x, w, b)
    (dx,) = torch.autograd.grad(y, x, dy)
    xp = x.detach()[-part:].clone().requires_grad_(True)
    yp = tk.layer_norm(xp, w, b)
    (dxp,) = torch.autograd.grad(yp, xp, dy[-part:].clone())
    assert close(y[-part:], yp) and close(dx[-part:], dxp)


def test_layer_norm_modulation(tk):
    L, C = 2**30 // 2944 + 3000, 2944
    x, s, h = normal(2, L, C), normal(2, 1, C), normal(2, 1, C)
    y = tk.layer_norm_modulation(x, s, h)
    assert close(y[1:, -5000:], tk.layer_norm_modulation(x[1:, -5000:].clone(), s[1:], h[1:]))


@pytest.mark.parametrize("token_major", [False, True])
def test_rotation(tk, token_major):
    L, H = 710000, 24
    q = normal(1, L, H, 128).transpose(1, 2) if token_major else normal(1, H, L, 128)
    k = normal(1, 1, L, 128)
    ids = torch.randint(0, 1000, (1, L, 3), device="cuda")
    oq, _ = tk.apply_rope_axes(q, k, ids, (16, 56, 56))
    part, _ = tk.apply_rope_axes(q[:, :, -300:].clone(), k[:, :, -300:].clone(), ids[:, -300:], (16, 56, 56))
    assert torch.equal(oq[:, :, -300:], part)


@pytest.mark.parametrize("B,L,K,N", [(4, 67000, 64, 8192), (267000, 1, 64, 8192), (267000, 1, 8192, 64)])
def test_adapters_of_many_rows(tk, B, L, K, N):
    x, w, a, b = normal(B, L, K), normal(N, K) / 64, normal(3, 16, K) / 64, normal(3, N, 16) / 4
    index = torch.arange(B, device="cuda") % 3
    y = tk.linear_lora(x, w, None, a, b, index)
    take = 1 if L > 1 else 64
    assert close(y[-take:, -100:], tk.linear_lora(x[-take:, -100:].clone(), w, None, a, b, index[-take:]))


@pytest.mark.parametrize("B,L", [(4, 1), (12, 3), (2, 40)])
def test_adapters_far_out(tk, B, L):
    n, N, R, K = 520, 16384, 256, 64
    x, w, a, b = normal(B, L, K), normal(N, K) / 8, normal(n, R, K) / 8, normal(n, N, R) / 16
    assert (n - 1) * N * R > 2**31
    index = torch.full((B,), n - 1, device="cuda")
    near = tk.linear_lora(x, w, None, a[-1:].clone(), b[-1:].clone(), torch.zeros_like(index))
    assert close(tk.linear_lora(x, w, None, a, b, index), near)
