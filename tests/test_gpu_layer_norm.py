"""LayerNorm with a learned scale and offset, and the gradients of both LayerNorm forms, against the definition in
64 bits on the same inputs.

Tolerances are sums of what each step can be off by.  u = 2^-24 is half a step of fp32, `half(dtype)` half a step of
the stored type.  A sum of n fp32 terms whose longest chain of additions is s long is off by at most
s u sum|terms| (s <= C / 32 + 16 for the sums over a row, which 32 lanes share at least; s <= rows for the sums over
rows).  `stat_tol` carries the statistics' error into h = (x - mean) rstd."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
TYPES = [torch.float32, torch.bfloat16]


def half(dtype):
    return torch.finfo(dtype).eps / 2


@pytest.fixture(scope="module")
def tk(lib):
    import triton_kernels_b200 as tk

    assert torch.cuda.is_available()
    return tk


def make(seed, shape, dtype, scale=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + mean).to(dtype).cuda()


def definition(x, f, o, eps, dy=None, rows_dim=None):
    """(y, h, rstd[, dx, df, do]) in 64 bits; f is the whole factor (1 + scale for the modulated form)."""
    x, f, o = x.double(), f.double(), o.double()
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    h = (x - mean) * rstd
    if dy is None:
        return h * f + o, h, rstd
    dy = dy.double()
    g = dy * f
    dx = rstd * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    return h * f + o, h, rstd, dx, (dy * h).sum(rows_dim, keepdim=True), dy.sum(rows_dim, keepdim=True)


def stat_tol(x, h, rstd, one_pass=False):
    """What h can be off by: the mean's error, the variance's (half of it, relative), and h's own roundings."""
    s = x.shape[-1] / 32 + 16
    x = x.double()
    d_mean = s * U * x.abs().mean(-1, keepdim=True)
    # centred: sum of squares s u; the mean's error enters squared.  One pass: s u of E[x^2] instead of the variance.
    d_var = s * U * (x.square().mean(-1, keepdim=True) * rstd.square() if one_pass else 1.0) + (d_mean * rstd).square()
    return d_mean * rstd + h.abs() * (0.5 * d_var + 4 * U)


def check(got, want, tol, dtype):
    want = want.reshape(got.shape)
    err = (got.double() - want).abs()
    limit = tol.reshape(want.shape) if tol.numel() == want.numel() else tol.expand_as(want)
    limit = limit + half(dtype) * (want.abs() + limit)
    bad = err > limit
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, worst {float((err / limit).max()):.3g} x the limit"


def grad_tols(x, f, h, rstd, dy, dh, rows_dim):
    """What dx, df and do can be off by before they are rounded."""
    s = x.shape[-1] / 32 + 16
    n = 1
    for d in (rows_dim if isinstance(rows_dim, tuple) else (rows_dim,)):
        n *= x.shape[d]
    dy = dy.double()
    g = (dy * f.double()).abs()
    mg, mgh = g.mean(-1, keepdim=True), (g * h.abs()).mean(-1, keepdim=True)
    d_s2 = (s + 4) * U * mgh + (g * dh).mean(-1, keepdim=True)
    dx = rstd * ((s + 4) * U * mg + 4 * U * (g + mg + h.abs() * mgh) + h.abs() * d_s2 + dh * mgh)
    # rstd's own error, relative, is within dh at |h| = 1 or more; a row's largest |h| is
    d_r = dh.amax(-1, keepdim=True) / h.abs().amax(-1, keepdim=True).clamp(min=1e-30)
    dx = dx + d_r * rstd * (g + mg + h.abs() * mgh)
    df = ((n + 4) * U * (dy * h).abs() + dy.abs() * dh).sum(rows_dim, keepdim=True)
    do = (n * U * dy.abs()).sum(rows_dim, keepdim=True)
    return dx, df, do


WIDTHS = [1, 2, 7, 8, 40, 63, 128, 384, 515, 768, 1000, 1001, 1024, 2046, 2048, 3003, 3072, 4096, 6001, 8192, 8200, 12288, 20000]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_layer_norm_and_its_gradients(tk, width, dtype):
    for rows in (1, 2, 67):
        x = make(1, (rows, width), dtype, 1.5, 0.4).requires_grad_()
        w, b = make(2, (width,), dtype, 0.2, 1.0).requires_grad_(), make(3, (width,), dtype, 0.3).requires_grad_()
        dy = make(4, (rows, width), dtype)
        y = tk.layer_norm(x, w, b, 1e-5)
        grads = torch.autograd.grad(y, (x, w, b), dy)
        assert torch.equal(y, tk.layer_norm(x.detach(), w.detach(), b.detach(), 1e-5))
        xd, wd, bd = x.detach(), w.detach(), b.detach()
        want, h, rstd, *wants = definition(xd, wd, bd, 1e-5, dy, 0)
        dh = stat_tol(xd, h, rstd)
        check(y.detach(), want, dh * wd.double().abs() + 3 * U * ((h * wd.double()).abs() + bd.double().abs()), dtype)
        for got, ref, tol in zip(grads, wants, grad_tols(xd, wd, h, rstd, dy, dh, 0)):
            assert got.dtype == dtype
            check(got, ref, tol, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,L,C", [(1, 1, 128), (2, 9, 72), (3, 37, 3072), (2, 300, 1024), (5, 64, 1000), (1, 700, 256), (2, 11, 1001), (200, 3, 64)])
def test_modulated_gradients(tk, B, L, C, dtype):
    x = make(5, (B, L, C), dtype, 1.5, 0.3).requires_grad_()
    sc, sh = make(6, (B, 1, C), dtype, 0.3).requires_grad_(), make(7, (B, 1, C), dtype, 0.3).requires_grad_()
    dy = make(8, (B, L, C), dtype)
    y = tk.layer_norm_modulation(x, sc, sh, 1e-6)
    grads = torch.autograd.grad(y, (x, sc, sh), dy)
    xd, f, o = x.detach(), 1 + sc.detach().double(), sh.detach()
    assert torch.equal(y, tk.layer_norm_modulation(xd, sc.detach(), o, 1e-6)), "gradients do not change the forward"
    want, h, rstd, *wants = definition(xd, f, o, 1e-6, dy, 1)
    dh = stat_tol(xd, h, rstd, one_pass=True)
    check(y.detach(), want, dh * f.abs() + 4 * U * ((h * f).abs() + o.double().abs()), dtype)
    for got, ref, tol, shape in zip(grads, wants, grad_tols(xd, f, h, rstd, dy, dh, 1), (x.shape, sc.shape, sh.shape)):
        assert got.shape == shape and got.dtype == dtype
        check(got, ref, tol, dtype)


def test_many_rows_and_long_sums(tk):
    """More rows than the machine holds at once; the column sums run over all of them."""
    for shape, dtype in (((9001, 320), torch.float32), ((2, 5000, 1536), torch.bfloat16)):
        C = shape[-1]
        x = make(9, shape, dtype).requires_grad_()
        w, b = make(10, (C,), dtype, 0.1, 1.0).requires_grad_(), make(11, (C,), dtype).requires_grad_()
        dy = make(12, shape, dtype)
        y = tk.layer_norm(x, w, b)
        grads = torch.autograd.grad(y, (x, w, b), dy)
        dims = tuple(range(len(shape) - 1))
        _, h, rstd, *wants = definition(x.detach(), w.detach(), b.detach(), 1e-5, dy, dims)
        dh = stat_tol(x.detach(), h, rstd)
        for got, ref, tol in zip(grads, wants, grad_tols(x.detach(), w.detach(), h, rstd, dy, dh, dims)):
            check(got, ref, tol, dtype)
        again = torch.autograd.grad(tk.layer_norm(x, w, b), (x, w, b), dy)
        assert all(torch.equal(p, q) for p, q in zip(grads, again)), "the sums' order does not change from call to call"


@pytest.mark.parametrize("dtype", TYPES)
def test_parts_that_are_absent_or_not_wanted(tk, dtype):
    rows, C = 33, 264
    x, w, b, dy = make(13, (rows, C), dtype), make(14, (C,), dtype, 0.1, 1.0), make(15, (C,), dtype), make(16, (rows, C), dtype)
    one, zero = torch.ones_like(w), torch.zeros_like(w)
    assert torch.equal(tk.layer_norm(x), tk.layer_norm(x, one, zero))
    assert torch.equal(tk.layer_norm(x, w), tk.layer_norm(x, w, zero))
    assert torch.equal(tk.layer_norm(x, None, b), tk.layer_norm(x, one, b))
    full = [t.clone().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(tk.layer_norm(*full), full, dy)
    for i in range(3):
        only = [t.clone() for t in (x, w, b)]
        only[i].requires_grad_()
        assert torch.equal(torch.autograd.grad(tk.layer_norm(*only), only[i], dy)[0], want[i])
    xg = x.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(tk.layer_norm(xg), xg, dy)[0],
                       torch.autograd.grad(tk.layer_norm(xg, one, zero), xg, dy)[0])


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_offsets_and_layouts(tk, dtype):
    """Row strides, a column slice, a start that is not 16-byte aligned, permuted dims, an expanded gradient."""
    C = 512
    base = make(17, (40, C + 24), dtype)
    w, b = make(18, (C + 1,), dtype, 0.1, 1.0), make(19, (C + 1,), dtype)
    for x in (base[:, :C], base[:, 8 : 8 + C], base[:, 1 : 1 + C], base[::2, :C], make(20, (C, 40), dtype).t(),
              make(21, (4, 10, C), dtype).transpose(0, 1)):
        for ww, bb in ((w[:C], b[:C]), (w[1:], b[1:])):
            xg = x.detach().requires_grad_()
            y = tk.layer_norm(xg, ww, bb)
            assert y.shape == x.shape and torch.equal(y, tk.layer_norm(x.clone().contiguous(), ww.clone(), bb.clone()))
            dy = torch.ones((), device="cuda", dtype=dtype).expand(y.shape)
            dx = torch.autograd.grad(y, xg, dy)[0]
            xc = x.detach().clone().contiguous().requires_grad_()
            ref = torch.autograd.grad(tk.layer_norm(xc, ww.clone(), bb.clone()), xc, dy.contiguous())[0]
            assert torch.equal(dx, ref)


def test_rows_that_are_not_finite_stay_by_themselves(tk):
    x = make(22, (12, 1024), torch.float32)
    bad = x.clone()
    bad[3, 7], bad[8, 0] = float("nan"), float("inf")
    keep = [i for i in range(12) if i not in (3, 8)]
    w = torch.ones(1024, device="cuda")
    assert torch.equal(tk.layer_norm(bad, w, w)[keep], tk.layer_norm(x, w, w)[keep])
    assert bool(tk.layer_norm(bad, w, w)[[3, 8]].isnan().any(-1).all())
    bg = bad.requires_grad_()
    dx = torch.autograd.grad(tk.layer_norm(bg, w, w), bg, torch.ones_like(bad))[0]
    assert bool(dx[keep].isfinite().all())


def test_rows_far_from_zero_and_constant_rows(tk):
    """The statistics are centred: rows whose mean is thousands of deviations from zero, and rows of one value."""
    for dtype, mean in ((torch.float32, 4000.0), (torch.bfloat16, 256.0)):
        x = make(23, (16, 2048), dtype, 1.0, mean)
        x[5] = x[5, 0]
        w, b = make(24, (2048,), dtype, 0.1, 1.0), make(25, (2048,), dtype)
        want, h, rstd = definition(x, w, b, 1e-5)
        # a row of one value has h = 0; its mean may be off by s u |mean|, times rstd = 1 / sqrt(eps)
        check(tk.layer_norm(x, w, b), want, stat_tol(x, h, rstd) * w.double().abs() + 3 * U * ((h * w.double()).abs() + b.double().abs()), dtype)


@pytest.mark.parametrize("mod", [False, True])
def test_gradients_against_differences(tk, mod):
    """<grad, v> against (loss(x + e v) - loss(x - e v)) / 2e with the forward kernel itself, fp32.  The central
    difference is off by e^2 / 6 of a third derivative (order 10 rstd^3 sum|dy| here) and by the roundings of the two
    losses, 8 u sum|dy y| / e at most."""
    e = 2.0**-7
    B, L, C = 2, 3, 48
    x = make(26, (B, L, C), torch.float32)
    f, o = (make(27, (B, 1, C) if mod else (C,), torch.float32, 0.3, 0.0 if mod else 1.0), make(28, (B, 1, C) if mod else (C,), torch.float32))
    dy = make(29, (B, L, C), torch.float32)
    fn = tk.layer_norm_modulation if mod else tk.layer_norm
    args = [t.requires_grad_() for t in (x, f, o)]
    grads = torch.autograd.grad(fn(*args), args, dy)
    with torch.no_grad():
        for i in range(3):
            v = make(30 + i, args[i].shape, torch.float32)
            plus, minus = ([t + s * e * v if j == i else t for j, t in enumerate(args)] for s in (1, -1))
            diff = ((fn(*plus).double() - fn(*minus).double()) * dy.double()).sum() / (2 * e)
            y = fn(*args)
            tol = 8 * U * (dy * y).abs().double().sum() / e + e * e / 6 * 10 * dy.abs().double().sum()
            assert abs(float(diff - (grads[i].double() * v.double()).sum())) < float(tol)


def test_no_rows(tk):
    w = torch.ones(64, device="cuda", requires_grad=True)
    x = torch.empty(0, 64, device="cuda", requires_grad=True)
    y = tk.layer_norm(x, w, None)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert y.shape == dx.shape == (0, 64) and bool((dw == 0).all())
    x3 = torch.empty(2, 0, 64, device="cuda", requires_grad=True)
    sc = torch.zeros(2, 1, 64, device="cuda", requires_grad=True)
    y = tk.layer_norm_modulation(x3, sc, sc.detach())
    dx, ds = torch.autograd.grad(y, (x3, sc), torch.empty_like(y))
    assert y.shape == dx.shape == (2, 0, 64) and ds.shape == (2, 1, 64) and bool((ds == 0).all())


def test_empty_last_dim_is_refused(tk):
    for call in (lambda: tk.layer_norm(torch.empty(3, 0, device="cuda")),
                 lambda: tk.layer_norm_modulation(*(torch.empty(2, n, 0, device="cuda") for n in (4, 1, 1)))):
        with pytest.raises(AssertionError):
            call()


def test_scale_of_another_type_gets_a_gradient_of_its_own(tk):
    """bf16 rows with an fp32 scale and shift, in shapes that broadcast: gradients in fp32, unrounded."""
    x, dy = make(33, (2, 50, 256), torch.bfloat16), make(34, (2, 50, 256), torch.bfloat16)
    sc, sh = make(35, (2, 1, 256), torch.float32, 0.2).requires_grad_(), make(36, (2, 1, 256), torch.float32).requires_grad_()
    ds, db = torch.autograd.grad(tk.layer_norm_modulation(x, sc, sh), (sc, sh), dy)
    assert ds.dtype == db.dtype == torch.float32 and ds.shape == sc.shape
    _, h, rstd, _, df, do = definition(x, 1 + sc.detach().bfloat16().double(), sh.detach(), 1e-5, dy, 1)
    _, tf, to = grad_tols(x, 1 + sc.detach(), h, rstd, dy, stat_tol(x, h, rstd, True), 1)
    check(ds, df, tf, torch.float32)
    check(db, do, to, torch.float32)


@pytest.mark.parametrize("mod", [False, True])
def test_other_stream_and_graph_replay(tk, mod):
    B, L, C = 2, 130, 3072
    fn = tk.layer_norm_modulation if mod else tk.layer_norm
    vec = (B, 1, C) if mod else (C,)
    x, dy = make(37, (B, L, C), torch.bfloat16).requires_grad_(), make(38, (B, L, C), torch.bfloat16)
    f, o = make(39, vec, torch.bfloat16, 0.2).requires_grad_(), make(40, vec, torch.bfloat16).requires_grad_()

    def step():
        y = fn(x, f, o)
        return (y.detach(), *torch.autograd.grad(y, (x, f, o), dy))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    with torch.no_grad():
        x.copy_(make(41, x.shape, torch.bfloat16))
        dy.copy_(make(42, dy.shape, torch.bfloat16))
    for g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    want = step()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_module_has_the_keys_of_the_torch_module(tk):
    m, ref = tk.LayerNorm(96).cuda(), torch.nn.LayerNorm(96).cuda()
    assert list(m.state_dict()) == list(ref.state_dict())
    x = make(43, (5, 96), torch.float32)
    m(x).sum().backward()
    assert m.weight.grad.shape == (96,) and m.bias.grad.shape == (96,)
    with pytest.raises(AssertionError):
        tk.LayerNorm((4, 24)).cuda()(x.view(5, 4, 24))


def test_gradients_are_not_differentiable_again(tk):
    x = make(44, (3, 64), torch.float32).requires_grad_()
    dx = torch.autograd.grad(tk.layer_norm(x).square().sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()


def test_a_single_row_of_any_stride(tk):
    """The row stride of a single row says nothing (a view may have any)."""
    base = make(71, (96,), torch.float32)
    x = base.as_strided((1, 96), (1, 1))
    assert x.is_contiguous()
    w = make(72, (96,), torch.float32)
    want = tk.layer_norm(base[None].clone(), w, w)
    assert torch.equal(tk.layer_norm(x, w, w), want)
    leaf = x.detach().requires_grad_(True)
    ref = base[None].clone().requires_grad_(True)
    (got,) = torch.autograd.grad(tk.layer_norm(leaf, w, w).square().sum(), leaf)
    (exp,) = torch.autograd.grad(tk.layer_norm(ref, w, w).square().sum(), ref)
    assert torch.equal(got, exp)
