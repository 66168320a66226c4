"""`_lib.kernel_calls` counts every C-ABI call, whichever way it is bound."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_calls_are_counted(lib):
    import triton_kernels_b200 as tk
    from triton_kernels_b200 import _lib

    x, m, w = torch.randn(2, 8, 64, device="cuda"), torch.zeros(2, 1, 64, device="cuda"), torch.ones(64, device="cuda")
    b = x.bfloat16()
    ids, adapter = torch.zeros(2, 8, 1, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    a, lb, wb = (torch.zeros(*s, device="cuda").bfloat16() for s in ((1, 8, 64), (1, 64, 8), (64, 64)))

    def count(call):
        before = _lib.kernel_calls
        call()
        return _lib.kernel_calls - before

    xg = x.clone().requires_grad_()
    assert count(lambda: tk.layer_norm_modulation(x, m, m)) == 1
    assert count(lambda: tk.layer_norm(x, w, w)) == 1
    assert count(lambda: torch.autograd.grad(tk.layer_norm(xg, w, w).sum(), xg)) == 2
    assert count(lambda: tk.apply_rope_axes(x[None], x[None], ids[:1], (64,))) == 1
    assert count(lambda: tk.linear_lora(b, wb, None, a, lb, adapter)) == 1
    assert count(lambda: tk.linear(b, wb, None)) == 1
    with pytest.raises(ValueError):
        tk.linear_lora(b, wb[:60], None, a, lb[:, :60], adapter)
    assert count(lambda: None) == 0
