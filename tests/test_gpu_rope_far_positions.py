"""How exact the rotation's angles are, against angles in extended precision (64 bits of significand): the turn left over after
whole turns is right to 2^-24 of a turn for up to 2^27 turns, and beyond that to 2^-52 of the number of turns.

The bound of an output is then 2 pi times that, in radians, times the pair's length, and 4 u for sine and cosine and 3 u for the
products and their sum (u = 2^-24), and half a step of the stored type."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
D = 64


@pytest.fixture(scope="module")
def tk(lib):
    import triton_kernels_b200 as tk

    assert torch.cuda.is_available()
    return tk


def turns(ids, theta):
    """[L, D / 2] whole and fractional turns in extended precision."""
    assert np.finfo(np.longdouble).nmant >= 63
    two_pi = 2 * np.longdouble("3.14159265358979323846264338327950288")
    freq = np.power(np.longdouble(theta), -np.arange(0, D, 2, dtype=np.longdouble) / D) / two_pi
    return ids.numpy().astype(np.longdouble)[:, None] * freq


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("theta", [10000.0, 500000.0, 2.0**-6])
@pytest.mark.parametrize("top", [2**12, 2**20, 2**22, 2**24, 2**24 + 2**10, 2**27, 800_000_000, 2**33, 2**45])
def test_far_positions(tk, top, theta, sign):
    g = torch.Generator().manual_seed(top % 1000003)
    ids = sign * (top - 1 - torch.randint(0, min(top, 2**14), (257,), generator=g))
    x = torch.randn(1, 2, 257, D, generator=g).cuda()
    t = turns(ids, theta)
    left = torch.from_numpy((2 * (t - np.rint(t))).astype(np.float64)).cuda() * math.pi
    c, s = left.cos(), left.sin()
    e, o = x[..., 0::2].double(), x[..., 1::2].double()
    want = torch.stack((e * c - o * s, e * s + o * c), -1).flatten(-2)
    many = torch.from_numpy(np.abs(t).astype(np.float64)).cuda()
    off = torch.where(many <= 2.0**27, 2.0**-24, 2.0**-24 + 2.0**-52 * many)
    limit = ((2 * math.pi * off + 7 * U) * (e.square() + o.square()).sqrt()).repeat_interleave(2, -1)
    kinds = [ids[None, :, None].cuda()]
    if top <= 2**31:
        kinds.append(kinds[0].int())
    if top <= 2**24:
        kinds.append(kinds[0].float())
    for i in kinds:
        for got in tk.apply_rope_axes(x, x, i, (D,), theta):
            err = (got.double() - want).abs()
            assert bool((err <= limit + U * (want.abs() + limit)).all()), float((err / limit).max())
