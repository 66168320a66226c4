"""The operators that bind through torch's C++ API have no forward-mode derivative: a dual tensor is refused, on the host and
before anything else is looked at, instead of losing its tangent without a word."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import triton_kernels_b200 as tk

X = torch.randn(2, 8, 64)
V = torch.ones(64)
M = torch.zeros(2, 1, 64)
IDS = torch.zeros(1, 8, 1)
B16 = X.bfloat16()
LORA = (B16, torch.zeros(64, 64).bfloat16(), torch.zeros(64).bfloat16(), torch.zeros(1, 8, 64).bfloat16(), torch.zeros(1, 64, 8).bfloat16(),
        torch.zeros(2, dtype=torch.int64), torch.ones(1))
CALLS = [(tk.layer_norm, (X, V, V), (0, 1, 2)), (tk.layer_norm_modulation, (X, M, M), (0, 1, 2)),
         (lambda q, k, ids: tk.apply_rope_axes(q, k, ids, (64,)), (X[None], X[None], IDS), (0, 1, 2)), (tk.linear_lora, LORA, (0, 1, 2, 3, 4, 6))]


@pytest.mark.parametrize("i", range(len(CALLS)))
def test_dual_tensors_are_refused(i):
    call, args, places = CALLS[i]
    for place in places:
        for needs_grad in (False, True):
            with fwd.dual_level():
                primal = args[place].clone().requires_grad_(needs_grad)
                dual = [fwd.make_dual(primal, torch.ones_like(primal)) if j == place else a for j, a in enumerate(args)]
                for mode in (torch.enable_grad, torch.no_grad):
                    with mode(), pytest.raises(NotImplementedError, match="forward-mode"):
                        call(*dual)
                with fwd._set_fwd_grad_enabled(False), pytest.raises(RuntimeError, match="CUDA tensors only"):
                    call(*(a.detach() for a in dual))  # as any tensor on the host


def test_the_modules_refuse_them():
    m = tk.LayerNorm(64)
    with fwd.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        m(fwd.make_dual(X, X))
