"""The statistics of both LayerNorm forms on rows that cancel: a column far from the others, rows of almost one value, rows
far from zero, and rows of ordinary values, in calls of so many rows that the forward stages them in shared memory, and at
widths of each of its forms.  Against the definition in 64 bits, outputs and gradients.

The tolerances are those of centred statistics (`stat_tol` of test_gpu_layer_norm): the mean is off by s u mean|x|, the
variance by s u of itself and the square of the mean's error, s = C / 32 + 16.  The result's own step x rstd - mean rstd
rounds mean rstd once (u |mean| rstd), which the 16 of s holds: a sum that 32 lanes share has a chain of C / 32 + 5 sums and
one division."""
import pytest
import torch
from test_gpu_layer_norm import U, check, definition, grad_tols, make, stat_tol

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]
# 2 KB to 24 KB are staged; up to 6 KB with the vectors beside them; 1536 fp32 and 3072 bf16 unrolled; others in registers
WIDTHS = {torch.float32: [96, 384, 520, 1000, 1536, 2048, 6144, 6200], torch.bfloat16: [96, 512, 1024, 1480, 3072, 4096, 12288, 12296]}
KINDS = ["ordinary", "first", "inner", "one", "thirty", "far"]


@pytest.fixture(scope="module")
def tk(lib):
    import triton_kernels_b200 as tk

    assert torch.cuda.is_available()
    return tk


def rows(kind, n, C, dtype):
    g = torch.Generator().manual_seed(C)
    x = torch.randn(n, C, generator=g)
    if kind == "ordinary":
        x = 1.5 * x + 0.4
    elif kind in ("first", "inner"):  # one column of 20 to 10000
        x[:, 0 if kind == "first" else C // 3] = 10.0 ** (1.3 + 2.7 * torch.rand(n, generator=g)) * torch.randn(n, generator=g).sign()
    elif kind in ("one", "thirty"):  # all columns the same value but for one, or for thirty
        x = torch.tensor([100.5, 10.0, 300.0, -40.0])[torch.arange(n) % 4][:, None].repeat(1, C)
        for i in range(n):
            x[i, torch.randperm(C, generator=g)[: 1 if kind == "one" else 30]] *= 1.01 if kind == "one" else 1.006
    else:
        x = x + torch.tensor([256.0, -1000.0])[torch.arange(n) % 2][:, None]
    return x.to(dtype).cuda()


CASES = [(kind, width, dtype) for dtype in TYPES for width in WIDTHS[dtype] for kind in KINDS]


@pytest.mark.parametrize("kind,width,dtype", CASES)
def test_learned_scale(tk, kind, width, dtype):
    x = rows(kind, 301, width, dtype).requires_grad_()
    w, b = make(2, (width,), dtype, 0.2, 1.0).requires_grad_(), make(3, (width,), dtype, 0.3).requires_grad_()
    dy = make(4, (301, width), dtype)
    y = tk.layer_norm(x, w, b)
    grads = torch.autograd.grad(y, (x, w, b), dy)
    xd, wd, bd = x.detach(), w.detach(), b.detach()
    assert torch.equal(y, tk.layer_norm(xd, wd, bd))
    want, h, rstd, *wants = definition(xd, wd, bd, 1e-5, dy, 0)
    dh = stat_tol(xd, h, rstd)
    check(y.detach(), want, dh * wd.double().abs() + 3 * U * ((h * wd.double()).abs() + bd.double().abs()), dtype)
    for got, ref, tol in zip(grads, wants, grad_tols(xd, wd, h, rstd, dy, dh, 0)):
        check(got, ref, tol, dtype)


@pytest.mark.parametrize("L", [160, 151])  # blocks of 16 rows within one request, and across two
@pytest.mark.parametrize("kind,width,dtype", CASES)
def test_modulated(tk, kind, width, dtype, L):
    x = rows(kind, 2 * L, width, dtype).view(2, L, width).requires_grad_()
    sc, sh = make(6, (2, 1, width), dtype, 0.3).requires_grad_(), make(7, (2, 1, width), dtype, 0.3).requires_grad_()
    dy = make(8, x.shape, dtype)
    y = tk.layer_norm_modulation(x, sc, sh, 1e-6)
    grads = torch.autograd.grad(y, (x, sc, sh), dy)
    xd, f, o = x.detach(), 1 + sc.detach().double(), sh.detach()
    assert torch.equal(y, tk.layer_norm_modulation(xd, sc.detach(), o, 1e-6))
    want, h, rstd, *wants = definition(xd, f, o, 1e-6, dy, 1)
    dh = stat_tol(xd, h, rstd)
    check(y.detach(), want, dh * f.abs() + 4 * U * ((h * f).abs() + o.double().abs()), dtype)
    for got, ref, tol in zip(grads, wants, grad_tols(xd, f, h, rstd, dy, dh, 1)):
        check(got, ref, tol, dtype)


def test_an_infinite_value_leaves_no_number_in_its_row(tk):
    """(x - mean) rstd has a mean that is infinite: NaN in every column, however many rows the call has."""
    for dtype, width in ((torch.float32, 1536), (torch.float32, 2048), (torch.bfloat16, 3072), (torch.bfloat16, 8192)):
        x = make(9, (400, width), dtype)
        w, z = torch.ones(width, device="cuda", dtype=dtype), torch.zeros(1, 1, width, device="cuda", dtype=dtype)
        for call in (lambda t: tk.layer_norm(t, w, w), lambda t: tk.layer_norm_modulation(t[None], z, z)[0]):
            want = call(x)
            bad = x.clone()
            bad[3, 7], bad[8, 0], bad[399, -1] = float("inf"), float("-inf"), float("nan")
            got = call(bad)
            assert bool(got[[3, 8, 399]].isnan().all())
            got[[3, 8, 399]] = want[[3, 8, 399]]
            assert torch.equal(got, want)


@pytest.mark.parametrize("dtype,width", [(torch.float32, 1536), (torch.float32, 2048), (torch.float32, 1000), (torch.bfloat16, 3072)])
def test_gradients_of_more_rows_than_the_rings_hold(tk, dtype, width):
    """The backward's rings wrap several times; outputs and gradients."""
    n = 6007
    x = rows("first", n, width, dtype).requires_grad_()
    w, b = make(10, (width,), dtype, 0.1, 1.0).requires_grad_(), make(11, (width,), dtype).requires_grad_()
    dy = make(12, (n, width), dtype)
    y = tk.layer_norm(x, w, b)
    grads = torch.autograd.grad(y, (x, w, b), dy)
    xd, wd, bd = x.detach(), w.detach(), b.detach()
    want, h, rstd, *wants = definition(xd, wd, bd, 1e-5, dy, 0)
    dh = stat_tol(xd, h, rstd)
    check(y.detach(), want, dh * wd.double().abs() + 3 * U * ((h * wd.double()).abs() + bd.double().abs()), dtype)
    for got, ref, tol in zip(grads, wants, grad_tols(xd, wd, h, rstd, dy, dh, 0)):
        check(got, ref, tol, dtype)
