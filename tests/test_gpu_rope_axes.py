"""Rotary positions from ids against the rotation in 64 bits on the same inputs.

Tolerances: an angle that is off by d radians moves an output by at most d |pair|.  The kernel's reduced turn is
rounded to fp32 (2^-25 turns at most, 2 pi 2^-25 radians) and sine and cosine are off by two fp32 steps at most
(2^-22 near 1, relative to values of up to 1); two products and a sum add 3 u.  Together below 16 u |pair|,
u = 2^-24, and half a step of the stored type on the result."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
TYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def tk(lib):
    import triton_kernels_b200 as tk

    assert torch.cuda.is_available()
    return tk


def make(seed, shape, dtype):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def rotation(x, ids, axes, theta, sign=1):
    x = x.double()
    rot = sum(axes)
    freq = [ids[..., i : i + 1].double() * theta ** (-torch.arange(0, d, 2, dtype=torch.float64, device=x.device) / d)
            for i, d in enumerate(axes)]
    a = sign * torch.cat(freq, -1)[:, None]
    c, s = a.cos(), a.sin()
    e, o = x[..., 0:rot:2], x[..., 1:rot:2]
    out = torch.stack((e * c - o * s, e * s + o * c), -1).flatten(-2)
    return torch.cat((out, x[..., rot:]), -1)


def check(got, x, ids, axes, theta, sign=1):
    want = rotation(x, ids, axes, theta, sign)
    rot = sum(axes)
    xd = x.double()
    pair = (xd[..., 0:rot:2].square() + xd[..., 1:rot:2].square()).sqrt().repeat_interleave(2, -1)
    limit = 16 * U * pair
    limit = limit + torch.finfo(got.dtype).eps / 2 * (want[..., :rot].abs() + limit)
    err = (got.double() - want)[..., :rot].abs()
    assert got.shape == x.shape and got.dtype == x.dtype
    assert bool((err <= limit).all()), f"worst {float((err / limit).max()):.3g} x the limit"
    assert torch.equal(got[..., rot:], x[..., rot:]), "columns behind the axes are copied"


def positions(seed, B, L, n, top=5000):
    return torch.randint(0, top, (B, L, n), generator=torch.Generator().manual_seed(seed)).cuda()


SHAPES = [  # B, H, G, L, D, axes
    (1, 1, 1, 1, 8, (8,)), (2, 3, 1, 7, 128, (16, 56, 56)), (1, 24, 24, 130, 128, (16, 56, 56)), (3, 4, 2, 65, 64, (8, 28, 28)),
    (8, 24, 24, 1, 128, (16, 56, 56)), (2, 2, 2, 33, 96, (32, 64)), (1, 5, 5, 19, 72, (24, 24, 24)), (2, 3, 3, 9, 128, (64, 32)),
    (1, 2, 1, 40, 256, (256,)), (1, 2, 2, 5, 10, (4, 6)), (1, 1, 1, 3, 7, (2, 4)), (1, 2, 2, 12, 40, (2, 2, 2, 2, 2, 2, 2, 2)),
    (5, 1, 1, 300, 64, (64,)), (1, 40, 8, 17, 128, (128,)),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,H,G,L,D,axes", SHAPES)
def test_rotation_and_gradients(tk, B, H, G, L, D, axes, dtype):
    q, k = make(1, (B, H, L, D), dtype).requires_grad_(), make(2, (B, G, L, D), dtype).requires_grad_()
    dq, dk = make(3, q.shape, dtype), make(4, k.shape, dtype)
    for ids in (positions(5, B, L, len(axes)).float(), positions(6, 1, L, len(axes)).int(), positions(7, B, L, len(axes))):
        oq, ok = tk.apply_rope_axes(q, k, ids, axes, 10000.0)
        gq, gk = torch.autograd.grad((oq, ok), (q, k), (dq, dk))
        check(oq.detach(), q.detach(), ids, axes, 10000.0)
        check(ok.detach(), k.detach(), ids, axes, 10000.0)
        check(gq, dq, ids, axes, 10000.0, -1)
        check(gk, dk, ids, axes, 10000.0, -1)


def test_far_and_fractional_and_negative_positions(tk):
    q, k = make(8, (1, 2, 6, 64), torch.float32), make(9, (1, 2, 6, 64), torch.float32)
    far = torch.tensor([0, 1, -7, 2**24, 2**31 + 12345, -(2**40) + 1], device="cuda").view(1, 6, 1)
    # 2^40 turns of fp64 leave 2^-12 of a unit in the last place of an angle of one radian per position:
    # compare where the product still is exact to 2^-26 turns, i.e. positions below 2^27
    for ids in (far[:, :4].contiguous(), far[:, :4].float() * 0.5 + 0.25):
        oq, _ = tk.apply_rope_axes(q[:, :, :4], k[:, :, :4], ids, (64,), 10000.0)
        check(oq, q[:, :, :4], ids, (64,), 10000.0)
    oq, ok = tk.apply_rope_axes(q, k, far, (64,), 500000.0)
    assert bool(oq.isfinite().all()) and torch.allclose(oq.norm(dim=-1), q.norm(dim=-1), rtol=1e-5)


def test_layouts_are_kept(tk):
    B, H, G, L, D, axes = 2, 6, 3, 37, 128, (16, 56, 56)
    ids = positions(10, B, L, 3).float()
    for dtype in TYPES:
        qkv = make(11, (B, L, (H + 2 * G) * D), dtype)
        q = qkv[..., : H * D].unflatten(-1, (H, D)).permute(0, 2, 1, 3)
        k = qkv[..., H * D : (H + G) * D].unflatten(-1, (G, D)).permute(0, 2, 1, 3)
        want = tk.apply_rope_axes(q.contiguous(), k.contiguous(), ids, axes)
        got = tk.apply_rope_axes(q, k, ids, axes)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        t = make(12, (B, L, H, D), dtype).permute(0, 2, 1, 3)
        o, _ = tk.apply_rope_axes(t, t, ids, axes)
        assert o.stride() == t.stride() and torch.equal(o, tk.apply_rope_axes(t.contiguous(), t.contiguous(), ids, axes)[0])
        # a start that is not 16-byte aligned, rows at odd strides, the head dim not innermost, shared ids by stride 0
        wide = make(13, (B, H, L, D + 3), dtype)
        for v in (wide[..., 1 : 1 + D], wide[..., :D], make(14, (B, H, D, L), dtype).transpose(2, 3)):
            for i in (ids, ids[:1].expand(B, L, 3), ids.flip(-1)[..., [2, 1, 0]], ids.transpose(0, 1).contiguous().transpose(0, 1)):
                a = tk.apply_rope_axes(v, v, i, axes)
                b = tk.apply_rope_axes(v.contiguous(), v.contiguous(), i.contiguous(), axes)
                assert all(torch.equal(p, r) for p, r in zip(a, b))


def test_agrees_with_the_table_form_and_the_embedder(tk):
    from triton_kernels_b200.flux import EmbedND, flux_position_ids

    ids = flux_position_ids(32, 8, 12, device="cuda")
    pe = EmbedND(128, 10000, [16, 56, 56])
    q, k = make(15, (1, 4, 128, 128), torch.float32), make(16, (1, 4, 128, 128), torch.float32)
    table = tk.apply_rope(q, k, pe(ids))
    rotated = pe.rotate(q, k, ids)
    # both within the module's bound of the exact rotation
    pair = (q.unflatten(-1, (-1, 2)).norm(dim=-1).max(), k.unflatten(-1, (-1, 2)).norm(dim=-1).max())
    for a, b, p in zip(table, rotated, pair):
        assert float((a - b).abs().max()) <= 2 * 16 * U * float(p) * 1.01


def test_one_of_the_two_gradients(tk):
    axes, ids = (16, 56, 56), positions(17, 2, 9, 3)
    q, k = make(18, (2, 3, 9, 128), torch.bfloat16).requires_grad_(), make(19, (2, 3, 9, 128), torch.bfloat16)
    dq = make(20, q.shape, torch.bfloat16)
    oq, ok = tk.apply_rope_axes(q, k, ids, axes)
    assert oq.requires_grad
    check(torch.autograd.grad(oq, q, dq)[0], dq, ids, axes, 10000.0, -1)
    k.requires_grad_()
    oq, ok = tk.apply_rope_axes(q.detach(), k, ids, axes)
    check(torch.autograd.grad(ok, k, dq.expand_as(k))[0], dq, ids, axes, 10000.0, -1)
    # the same tensor as q and as k: the gradients add up
    q2 = make(21, (2, 3, 9, 128), torch.float32).requires_grad_()
    d1, d2 = make(22, q2.shape, torch.float32), make(23, q2.shape, torch.float32)
    g = torch.autograd.grad(tk.apply_rope_axes(q2, q2, ids, axes), q2, (d1, d2))[0]
    want = rotation(d1, ids, axes, 10000.0, -1) + rotation(d2, ids, axes, 10000.0, -1)
    assert float((g.double() - want).abs().max()) <= 40 * U * float((d1.abs().max() + d2.abs().max()) * 2)


def test_gradient_against_differences(tk):
    """The rotation is linear in q: a difference of any length is exact up to the roundings of the two values."""
    axes, ids = (8, 28, 28), positions(24, 1, 11, 3)
    q = make(25, (1, 2, 11, 64), torch.float32).requires_grad_()
    d, v = make(26, q.shape, torch.float32), make(27, q.shape, torch.float32)
    g = torch.autograd.grad(tk.apply_rope_axes(q, q.detach(), ids, axes)[0], q, d)[0]
    with torch.no_grad():
        diff = ((tk.apply_rope_axes(q + v, q, ids, axes)[0].double() - tk.apply_rope_axes(q - v, q, ids, axes)[0].double()) * d).sum() / 2
        tol = 20 * U * float((d.abs() * (q.abs() + v.abs()) * 3).double().sum())
        assert abs(float(diff - (g.double() * v).sum())) <= tol


def test_positions_that_are_not_finite_stay_by_themselves(tk):
    ids = positions(28, 1, 9, 3).float()
    bad = ids.clone()
    bad[0, 4, 1] = float("nan")
    q = make(29, (1, 2, 9, 128), torch.bfloat16)
    a, b = tk.apply_rope_axes(q, q, ids, (16, 56, 56))[0], tk.apply_rope_axes(q, q, bad, (16, 56, 56))[0]
    same = (a == b)
    assert bool(same[:, :, [0, 1, 2, 3, 5, 6, 7, 8]].all()) and bool(same[:, :, 4, :16].all()) and bool(b[:, :, 4, 16:72].isnan().all())


def test_no_tokens(tk):
    q = torch.empty(2, 3, 0, 64, device="cuda", requires_grad=True)
    o, _ = tk.apply_rope_axes(q, q.detach(), torch.empty(2, 0, 1, device="cuda"), (64,))
    assert o.shape == q.shape and torch.autograd.grad(o, q, torch.empty_like(o))[0].shape == q.shape


def test_other_stream_and_graph_replay(tk):
    axes = (16, 56, 56)
    q, k = make(30, (2, 24, 50, 128), torch.bfloat16).requires_grad_(), make(31, (2, 24, 50, 128), torch.bfloat16).requires_grad_()
    d, ids = make(32, q.shape, torch.bfloat16), positions(33, 2, 50, 3).float()

    def step():
        o = tk.apply_rope_axes(q, k, ids, axes)
        return (o[0].detach(), o[1].detach(), *torch.autograd.grad(o, (q, k), (d, d)))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    ids.copy_(positions(34, 2, 50, 3).float())
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_refusals_on_the_device(tk):
    q, ids = make(35, (1, 2, 4, 64), torch.float32), positions(36, 1, 4, 2)
    with pytest.raises(ValueError, match="even"):
        tk.apply_rope_axes(q, q, ids, (33, 31))
    with pytest.raises(ValueError, match="more than head_dim"):
        tk.apply_rope_axes(q, q, ids, (64, 2))
    with pytest.raises(ValueError, match="theta"):
        tk.apply_rope_axes(q, q, ids, (32, 32), math.inf)
    with pytest.raises(NotImplementedError):
        tk.apply_rope_axes(q, q, ids.half(), (32, 32))
    with pytest.raises(NotImplementedError):
        tk.apply_rope_axes(q.half(), q.half(), ids, (32, 32))
    with pytest.raises(AssertionError):
        tk.apply_rope_axes(q, q, ids[:, :3], (32, 32))
    with pytest.raises(AssertionError):
        tk.apply_rope_axes(q, q[:, :, :3], ids, (32, 32))
    with pytest.raises(NotImplementedError, match="no gradient"):
        tk.apply_rope_axes(q, q, ids.float().requires_grad_(True), (32, 32))


def test_a_theta_below_one_turns_faster(tk):
    """theta 2^-10, positions up to 2^24: 7.3e9 radians.  The angle itself is a product of three fp64 roundings on either
    side (frequency, turn, product), 6 x 2^-53 of it, next to the kernel's 16 u."""
    axes, theta = (16,), 2.0**-10
    ids = (2**24 - 1 - torch.randint(0, 2**20, (1, 70, 1), generator=torch.Generator().manual_seed(5))).cuda()
    q = make(6, (1, 2, 70, 16), torch.float32)
    got, _ = tk.apply_rope_axes(q, q, ids, axes, theta)
    want = rotation(q, ids, axes, theta)
    pair = q.double().unflatten(-1, (8, 2)).norm(dim=-1).repeat_interleave(2, -1)
    angle = float(ids.max()) * theta ** (-14 / 16)
    limit = (16 * U + 6 * 2.0**-53 * angle) * pair
    limit = limit + U * (want.abs() + limit)
    assert bool(((got.double() - want).abs() <= limit).all())


LONG = [  # B, H, G, L, D, axes: so many tokens that each piece of a row has one thread for all heads
    (3, 1, 2, 2000, 128, (16, 56, 56)), (2, 5, 1, 2501, 128, (10, 14, 22)), (6000, 1, 1, 1, 128, (64, 64)),
    (1, 4, 0, 5003, 256, (128, 126)), (7, 2, 3, 1400, 64, (64,)),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,H,G,L,D,axes", LONG)
def test_many_tokens(tk, B, H, G, L, D, axes, dtype):
    q, k = make(81, (B, H, L, D), dtype), make(82, (B, G, L, D), dtype)
    for ids in (positions(83, B, L, len(axes)), positions(84, 1, L, len(axes), 2**24).int(),
                positions(85, B, L, len(axes)).float() + 0.25, positions(86, B, L, len(axes)) + 2**33):
        oq, ok = tk.apply_rope_axes(q, k, ids, axes)
        slack = 2**33 * 6 * 2.0**-53 if ids.dtype == torch.int64 and int(ids.max()) > 2**32 else 0.0
        for got, x in ((oq, q), (ok, k)):
            if slack == 0.0:
                check(got, x, ids, axes, 10000.0)
            elif x.numel():  # fp64 angles of 2^33: three roundings on either side, next to the 16 u
                want = rotation(x, ids, axes, 10000.0)
                limit = (16 * U + slack) * x.double().abs().amax() * 2**0.5
                limit = limit + torch.finfo(dtype).eps / 2 * (want.abs() + limit)
                assert bool(((got.double() - want).abs() <= limit).all())
