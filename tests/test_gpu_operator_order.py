"""Kernels that may start while the one in front of them ends: every call sees what the calls, copies and fills in front of
it on its stream wrote, and leaves alone what they still read.  Unsynchronised runs and graph replays have to give the bits
of a run that is synchronised after every call."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
AXES = (16, 24, 24)


@pytest.fixture(scope="module")
def tk(lib):
    import triton_kernels_b200 as tk

    assert torch.cuda.is_available()
    return tk


class Block:
    """A small layer: norm, adapters, rotation, and torch operations between them; its buffers come and go, so that later
    calls write where earlier ones read."""

    def __init__(self, tk, B, L):
        g = torch.Generator().manual_seed(B * 1000 + L)
        r = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).to(BF).cuda()  # noqa: E731
        self.tk, self.B, self.L, C = tk, B, L, 512
        self.x, self.host = r(B, L, C), (torch.randn(B, L, C, generator=g)).to(BF).pin_memory()
        self.w, self.b, self.norm = r(3 * C, C, scale=C**-0.5), r(3 * C, scale=0.1), (1 + r(C, scale=0.1), r(C, scale=0.1))
        self.back = r(C, C, scale=C**-0.5)
        self.a, self.lb, self.la2 = r(4, 16, C, scale=C**-0.5), r(4, 3 * C, 16, scale=0.25), r(4, C, 16, scale=0.25)
        self.ids = torch.randint(0, 500, (B, L, 3), generator=g).cuda()
        self.adapter = (torch.arange(B) % 5 - 1).cuda()
        self.buffer = torch.empty_like(self.x)

    def run(self, side, pause=lambda: None):
        tk, B, L = self.tk, self.B, self.L
        self.buffer.zero_()
        x = self.x
        for i in range(6):
            h = tk.layer_norm(x, *self.norm)
            pause()
            qkv = tk.linear_lora(h, self.w, self.b, self.a, self.lb, self.adapter)
            pause()
            q, k, v = qkv.view(B, L, 3, 8, 64).permute(2, 0, 3, 1, 4)
            q, k = tk.apply_rope_axes(q, k, self.ids, AXES)
            pause()
            y = (q + k + v).transpose(1, 2).reshape(B, L, -1)
            self.buffer.copy_(self.host, non_blocking=True)  # a copy right in front of a call that reads it
            z = tk.linear_lora(self.buffer, self.back, None, self.a, self.la2, self.adapter, activation="GELU")
            pause()
            now = torch.cuda.current_stream()
            side.wait_stream(now)
            with torch.cuda.stream(side):  # a call on another stream, joined in front of the next one
                s = tk.linear_lora(y, self.back, None, self.a, self.la2, self.adapter)
                s.record_stream(now)
            now.wait_stream(side)
            y.record_stream(side)
            pause()
            x = tk.linear_lora(s, self.back, None, self.a, self.la2, self.adapter) + z * 0.5 + x * 0.5
            self.buffer.fill_(float(i))  # while the call in front may still be reading
            pause()
        return x


@pytest.mark.parametrize("B,L", [(1, 1), (5, 1), (48, 5), (3, 100), (2, 700)])
def test_order(tk, B, L):
    block, side = Block(tk, B, L), torch.cuda.Stream()
    want = block.run(side, torch.cuda.synchronize)
    torch.cuda.synchronize()
    got = [block.run(side) for _ in range(8)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("B,L", [(5, 1), (48, 5), (3, 100)])
def test_order_in_a_graph(tk, B, L):
    block, side = Block(tk, B, L), torch.cuda.Stream()
    want = block.run(side, torch.cuda.synchronize)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block.run(torch.cuda.Stream())
    for _ in range(5):
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    for _ in range(10):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
