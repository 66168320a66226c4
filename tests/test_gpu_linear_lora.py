"""A shared projection plus a low-rank adapter per request, against the definition in 64 bits on the same inputs.

Tolerance of one output before rounding: a sum of K products is off by K u sum|x w| at most (u = 2^-24, any order),
the low-rank product by (K + R) u of its own sum of absolute products; the low-rank rows t are held in two bf16 parts,
2^-17 of |t| at most.  With GELU the slope is at most 1.13, its fp32 evaluation (one exponential with an argument
error of |x| u times the exponent, one division) stays within 32 u of |v| + 1.  The result is rounded to bf16: 2^-8."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
BF = torch.bfloat16


@pytest.fixture(scope="module")
def tk(lib):
    import triton_kernels_b200 as tk

    assert torch.cuda.is_available()
    return tk


def problem(seed, B, L, K, N, R, n, bias=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale)  # noqa: E731
    return dict(
        x=r(B, L, K).to(BF).cuda(), w=r(N, K, scale=K**-0.5).to(BF).cuda(), b=r(N, scale=0.2).to(BF).cuda() if bias else None,
        lora_a=r(n, R, K, scale=K**-0.5).to(BF).cuda(), lora_b=r(n, N, R, scale=R**-0.5).to(BF).cuda(),
        adapter=torch.randint(-1, n, (B,), generator=g).cuda(), lora_scale=(0.5 + torch.rand(n, generator=g)).cuda())


def definition(p, activation=""):
    """(y, what it can be off by) in 64 bits."""
    x, w = p["x"].double(), p["w"].double()
    K, R = w.shape[1], p["lora_a"].shape[1]
    pick = p["adapter"].long()
    pick = torch.where((pick >= 0) & (pick < p["lora_a"].shape[0]), pick, -1)
    lead = x.shape
    x = x.reshape(lead[0], -1, K)
    sc = torch.where(pick >= 0, p["lora_scale"].double()[pick.clamp(min=0)] if p["lora_scale"] is not None else 1.0, 0.0)[:, None, None]
    A, Bm = p["lora_a"].double()[pick.clamp(min=0)], p["lora_b"].double()[pick.clamp(min=0)]
    t = x @ A.transpose(1, 2) * sc
    y = x @ w.T + t @ Bm.transpose(1, 2)
    tol = (K + 1) * U * (x.abs() @ w.abs().T)
    t_abs = x.abs() @ A.abs().transpose(1, 2) * sc
    tol = tol + ((K + 3) * U * t_abs + (2.0**-17 + R * U) * t.abs()) @ Bm.abs().transpose(1, 2)
    if p["b"] is not None:
        y = y + p["b"].double()
    tol = tol + 2 * U * y.abs()
    if activation:
        v = y
        y = 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v**3)))
        tol = 1.13 * tol + 32 * U * (v.abs() + 1)
    return y.reshape(*lead[:-1], -1), tol.reshape(*lead[:-1], -1)


def call(tk, p, activation=""):
    return tk.linear_lora(p["x"], p["w"], p["b"], p["lora_a"], p["lora_b"], p["adapter"], p["lora_scale"], activation)


def check(got, p, activation=""):
    want, tol = definition(p, activation)
    limit = tol + torch.finfo(BF).eps / 2 * (want.abs() + tol)
    err = (got.double() - want).abs()
    assert got.dtype == BF and got.shape == want.shape
    assert bool((err <= limit).all()), f"{int((err > limit).sum())} of {err.numel()} off, worst {float((err / limit).max()):.3g} x the limit"


SHAPES = [  # B, L, K, N, R, adapters
    (1, 1, 64, 64, 16, 1), (1, 1, 8, 8, 1, 2), (8, 1, 256, 512, 16, 8), (3, 1, 3072, 3072, 16, 2), (5, 1, 1536, 1024, 64, 4),
    (8, 1, 12296, 264, 8, 3), (2, 4, 512, 768, 32, 3), (9, 1, 256, 512, 16, 4), (64, 1, 512, 1024, 16, 5), (48, 5, 256, 512, 64, 16),
    (33, 3, 136, 200, 24, 4), (2, 128, 256, 512, 16, 2), (3, 129, 320, 264, 8, 3), (4, 255, 128, 256, 128, 4), (2, 300, 512, 768, 48, 3),
    (1, 1000, 256, 512, 100, 2), (7, 77, 192, 1032, 4, 6), (2, 513, 64, 2048, 33, 2), (130, 2, 64, 64, 16, 130), (1, 600, 1024, 1024, 256, 1),
    (20, 13, 2048, 512, 16, 20), (2, 16, 72, 88, 16, 2),
]


@pytest.mark.parametrize("B,L,K,N,R,n", SHAPES)
def test_against_definition(tk, B, L, K, N, R, n):
    p = problem(B * 7 + L, B, L, K, N, R, n)
    check(call(tk, p), p)
    p["lora_scale"] = None
    check(call(tk, p, "GELU"), p, "GELU")


def test_every_request_the_same_none_or_its_own(tk):
    for B, L in ((6, 1), (6, 50), (3, 300)):
        p = problem(B + L, B, L, 256, 512, 16, 6, bias=False)
        for idx in ([2] * B, [-1] * B, list(range(B)), list(range(B))[::-1], [0, -1] * (B // 2) + [0] * (B % 2)):
            for dtype in (torch.int32, torch.int64):
                p["adapter"] = torch.tensor(idx, dtype=dtype, device="cuda")
                check(call(tk, p), p)


def test_requests_without_an_adapter_equal_the_shared_projection(tk):
    """To the rounding: the kernels may add up in another order than `linear`'s."""
    p = problem(3, 4, 96, 512, 512, 16, 2)
    p["adapter"].fill_(-1)
    check(tk.linear(p["x"], p["w"], p["b"]), p)
    check(call(tk, p), p)


def test_indices_outside_the_adapters_are_recorded_and_count_as_none(tk):
    from triton_kernels_b200 import _lib

    _lib.device_status()
    for B, L in ((4, 1), (4, 40)):
        p = problem(11, B, L, 128, 256, 16, 2)
        p["adapter"] = torch.tensor([0, 2, -2, 2**40], device="cuda")
        got = call(tk, p)
        assert _lib.device_status() == (_lib.ERR_BAD_ARG, 81)
        check(got, p)
        assert _lib.device_status() == (0, 0)


def test_values_that_are_not_finite_stay_with_their_request(tk):
    """An adapter or a row that holds NaN reaches no request but those that use it."""
    for B, L in ((4, 1), (12, 1), (4, 37), (3, 200)):
        p = problem(12, B, L, 256, 512, 16, 3)
        p["adapter"] = (torch.arange(B, device="cuda") % 2)
        want = call(tk, p)
        p["lora_a"][2] = float("nan")  # nobody uses it
        p["lora_b"][2] = float("inf")
        assert torch.equal(call(tk, p), want)
        p["lora_b"][1] = float("nan")
        got = call(tk, p)
        assert torch.equal(got[0::2], want[0::2]) and bool(got[1::2].isnan().all())
        p["lora_b"][1] = 0
        want = call(tk, p)
        p["x"][0, 0] = float("inf")
        got = call(tk, p)
        assert torch.equal(got[1:], want[1:]) and torch.equal(got[0, 1:], want[0, 1:])


def test_layouts(tk):
    p = problem(13, 3, 40, 256, 264, 16, 3)
    want = call(tk, p)
    q = dict(p)
    wide = torch.zeros(3, 40, 300, device="cuda", dtype=BF)
    wide[..., 4:260] = p["x"]
    q["x"] = wide[..., 4:260]
    assert torch.equal(call(tk, q), want)
    q = dict(p)
    q["w"] = torch.cat((p["w"], p["w"]), 1)[:, :256]
    assert torch.equal(call(tk, q), want)
    q["w"] = p["w"].t().contiguous().t()
    assert torch.equal(call(tk, q), want)
    q = dict(p)
    q["lora_a"], q["lora_b"] = p["lora_a"].transpose(1, 2).contiguous().transpose(1, 2), p["lora_b"].transpose(1, 2).contiguous().transpose(1, 2)
    q["adapter"] = torch.stack((p["adapter"], p["adapter"]), 1)[:, 0]
    assert torch.equal(call(tk, q), want)
    store = torch.empty(p["lora_b"].numel() + 1, device="cuda", dtype=BF)
    store[1:] = p["lora_b"].flatten()
    q["lora_b"] = store[1:].view_as(p["lora_b"])
    assert torch.equal(call(tk, q), want)
    q = dict(p)
    q["x"] = p["x"].view(3, 2, 20, 256)
    assert torch.equal(call(tk, q), want.view(3, 2, 20, 264))
    p2 = problem(14, 5, 1, 256, 264, 16, 3)
    q = dict(p2)
    q["x"] = p2["x"][:, 0]
    assert torch.equal(call(tk, q), call(tk, p2)[:, 0])


def test_no_rows(tk):
    p = problem(15, 2, 4, 64, 64, 8, 1)
    p["x"] = p["x"][:, :0]
    assert call(tk, p).shape == (2, 0, 64)
    p["x"], p["adapter"] = p["x"][:0], p["adapter"][:0]
    assert call(tk, p).shape == (0, 0, 64)


def test_same_bits_on_every_call_stream_and_replay(tk):
    for shape in ((8, 1, 512, 1024, 16, 4), (30, 3, 512, 512, 32, 4), (3, 300, 512, 768, 64, 3)):
        p = problem(16, *shape)
        want = call(tk, p)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = call(tk, p)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = call(tk, p)
            graphs.append((g, out))
        p2 = problem(17, *shape)
        for name in ("x", "adapter", "lora_a"):
            p[name].copy_(p2[name])
        want = call(tk, p)
        for g, _ in graphs:
            g.replay()
        assert all(torch.equal(o, want) for _, o in graphs)


def test_two_calls_at_once(tk):
    a, b = problem(18, 2, 300, 512, 768, 16, 2), problem(19, 8, 1, 512, 768, 16, 2)
    wa, wb = call(tk, a), call(tk, b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(20):
        with torch.cuda.stream(s1):
            outs.append((call(tk, a), wa))
        with torch.cuda.stream(s2):
            outs.append((call(tk, b), wb))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in outs)


def test_first_call_of_a_process_inside_a_capture(lib):
    """Nothing that a first call sets up needs to run outside a capture."""
    code = """
import torch, triton_kernels_b200 as tk
torch.manual_seed(0)
r = lambda *s: torch.randn(*s, device="cuda").bfloat16()
sets = [(r(B, L, 256), r(512, 256), r(512), r(2, 16, 256), r(2, 512, 16), torch.arange(B, device="cuda") % 2) for B, L in ((2, 1), (3, 100), (2, 3000))]
x, w = r(64, 1024).requires_grad_(), r(1024).requires_grad_()
dy = r(64, 1024)
torch.cuda.synchronize()
def work():
    y = tk.layer_norm(x, w, w)
    return [tk.linear_lora(*s) for s in sets] + [y.detach(), *torch.autograd.grad(y, (x, w), dy)]
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = work()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, work()))
print("same")
"""
    import subprocess
    import sys
    from pathlib import Path

    root = Path(__file__).resolve().parent.parent
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


def test_module(tk):
    torch.manual_seed(0)
    m = tk.LinearLoRA(256, 512, num_adapters=3, rank=8).to(BF).cuda()
    x = torch.randn(4, 20, 256, device="cuda").to(BF)
    idx = torch.tensor([0, 2, -1, 1], device="cuda")
    assert torch.equal(m(x), tk.linear(x, m.weight, m.bias))
    m.lora_b.normal_()
    p = dict(x=x, w=m.weight.detach(), b=m.bias.detach(), lora_a=m.lora_a, lora_b=m.lora_b, adapter=idx, lora_scale=m.lora_scale.float())
    check(m(x, idx), p)


def test_refusals_on_the_device(tk):
    p = problem(20, 2, 4, 64, 64, 8, 2)
    with pytest.raises(NotImplementedError, match="forward only"):
        tk.linear_lora(p["x"].requires_grad_(), p["w"], p["b"], p["lora_a"], p["lora_b"], p["adapter"])
    x = p["x"].detach()
    with pytest.raises(TypeError):
        tk.linear_lora(x.float(), p["w"], p["b"], p["lora_a"], p["lora_b"], p["adapter"])
    with pytest.raises(TypeError):
        tk.linear_lora(x, p["w"], p["b"], p["lora_a"], p["lora_b"], p["adapter"].float())
    with pytest.raises(AssertionError):
        tk.linear_lora(x, p["w"], p["b"], p["lora_a"], p["lora_b"][:, :32], p["adapter"])
    with pytest.raises(AssertionError):
        tk.linear_lora(x, p["w"], p["b"], p["lora_a"], p["lora_b"], p["adapter"][:1])
    with pytest.raises(RuntimeError):
        tk.linear_lora(x, p["w"], p["b"], p["lora_a"], p["lora_b"], p["adapter"].cpu())
    with pytest.raises(AssertionError):
        e = lambda *s: torch.empty(*s, device="cuda", dtype=BF)  # noqa: E731
        tk.linear_lora(e(2, 0), e(8, 0), None, e(1, 8, 0), e(1, 8, 8), p["adapter"])
    with pytest.raises(NotImplementedError, match="rank"):
        call(tk, problem(23, 2, 4, 64, 64, 264, 1))
    odd = problem(21, 2, 4, 64, 60, 8, 2)
    with pytest.raises(ValueError, match="multiples of 8"):
        call(tk, odd)


def test_norm_adapter_rotation_attention_as_they_are_used_together(tk):
    """A batch of two requests with adapters and picture sizes of their own through the attention half of a block:
    modulated norm, q|k|v projection with adapters, rotation by each request's positions, attention, output projection.
    Every step rounds to bf16 once; six roundings of 2^-8 on values that later steps average: relative L2 below 6 * 2^-8."""
    B, L, H, D, axes = 2, 96, 4, 64, (8, 28, 28)
    C = H * D
    g = torch.Generator().manual_seed(22)
    r = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).to(BF).cuda()  # noqa: E731
    x, sc, sh = r(B, L, C), r(B, 1, C, scale=0.2), r(B, 1, C, scale=0.2)
    qkv = dict(w=r(3 * C, C, scale=C**-0.5), b=r(3 * C, scale=0.1), lora_a=r(2, 16, C, scale=C**-0.5), lora_b=r(2, 3 * C, 16, scale=0.2),
               adapter=torch.tensor([1, 0], device="cuda"), lora_scale=torch.tensor([1.0, 0.5], device="cuda"))
    out = dict(w=r(C, C, scale=C**-0.5), b=None, lora_a=r(2, 8, C, scale=C**-0.5), lora_b=r(2, C, 8, scale=0.2), adapter=qkv["adapter"],
               lora_scale=None)
    at = torch.arange(L, device="cuda")
    ids = torch.stack([torch.stack((0 * at, at // w, at % w), -1) for w in (8, 12)]).float()

    h = tk.layer_norm_modulation(x, sc, sh, 1e-6)
    q, k, v = call(tk, dict(qkv, x=h)).view(B, L, 3, H, D).permute(2, 0, 3, 1, 4)
    q, k = tk.apply_rope_axes(q, k, ids, axes)
    o = tk.scaled_dot_product_attention(q, k, v).transpose(1, 2).reshape(B, L, C)
    y = call(tk, dict(out, x=o))

    xd = x.double()
    hd = (xd - xd.mean(-1, keepdim=True)) * (xd.var(-1, keepdim=True, unbiased=False) + 1e-6).rsqrt() * (1 + sc.double()) + sh.double()
    qd, kd, vd = definition(dict(qkv, x=hd))[0].view(B, L, 3, H, D).permute(2, 0, 3, 1, 4)
    a = torch.cat([ids[..., i : i + 1].double() * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
                   for i, d in enumerate(axes)], -1)[:, None]
    rot = lambda t: torch.stack((t[..., 0::2] * a.cos() - t[..., 1::2] * a.sin(), t[..., 0::2] * a.sin() + t[..., 1::2] * a.cos()), -1).flatten(-2)  # noqa: E731
    od = ((rot(qd) @ rot(kd).transpose(2, 3) * D**-0.5).softmax(-1) @ vd).transpose(1, 2).reshape(B, L, C)
    yd = definition(dict(out, x=od))[0]
    assert float((y.double() - yd).norm() / yd.norm()) < 6 * 2.0**-8


@pytest.mark.parametrize("L", [1, 20, 200])
def test_an_infinite_input_stays_infinite(tk, L):
    """Rank 5: the ranks that fill up the tensor cores' sixteen must not turn infinity into NaN."""
    p = problem(41, 3, L, 64, 48, 5, 2)
    for key in ("w", "lora_a", "lora_b"):
        p[key] = p[key].abs() + 2.0**-10  # all positive: no infinity meets one of the other sign
    p["adapter"] = torch.tensor([1, -1, 0]).cuda()
    clean = call(tk, p)
    p["x"][0, 0, 3] = float("inf")
    y = call(tk, p)
    assert bool((y[0, 0] == float("inf")).all())
    y[0, 0] = clean[0, 0]
    assert torch.equal(y, clean)


MANY = [  # B, L, K, N, R, adapters: tiles whose rows use many adapters, several parts of ranks, several tiles a block
    (130, 1, 64, 136, 72, 130), (128, 1, 128, 64, 256, 128), (61, 2, 264, 328, 130, 61), (600, 2, 64, 4096, 16, 600),
    (300, 9, 64, 2048, 8, 7), (40, 60, 192, 1544, 64, 40), (3, 700, 512, 2048, 40, 3), (1, 2100, 256, 3096, 16, 1),
    (150, 130, 128, 24, 16, 5), (11, 129, 320, 1160, 200, 11), (3, 333, 1536, 3064, 64, 3), (9, 128, 4096, 2048, 8, 4),
]


@pytest.mark.parametrize("B,L,K,N,R,n", MANY)
def test_many_adapters_and_many_tiles(tk, B, L, K, N, R, n):
    p = problem(51 + B, B, L, K, N, R, n)
    p["adapter"] = (torch.arange(B) % (n + 1) - 1).cuda()
    check(call(tk, p), p)
    p["adapter"] = torch.arange(B).clamp(max=n - 1).cuda()
    check(call(tk, p), p)
