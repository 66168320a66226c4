"""Cases for timing three operators of the package on a GPU, each with its plain form beside it.

  norm   LayerNorm with a learned scale and offset (`layer_norm`) or with the per-request modulation of the adaLN
         blocks (`layer_norm_modulation`), forward alone or with the backward pass: gradients of the rows and of the
         scale and offset
  rope   rotary positions with several axes, taken from the position ids of every token (`apply_rope_axes`), forward
         alone or with the backward pass
  lora   a projection shared by all requests plus a low-rank adapter per request (`linear_lora`)

`own` chooses what `run` does: the plain form in elementary torch operations (32 bits; angles in 64), or the package's
kernels.  `exact` gives the same outputs in 64 bits.
"""
import math

import torch

own = False

EPS = 1e-5
THETA = 10000.0
BF16, F32 = "bf16", "f32"
DTYPES = {BF16: torch.bfloat16, F32: torch.float32}
AXES = {"128": (128,), "64+64": (64, 64), "16+56+56": (16, 56, 56), "16+24+24": (16, 24, 24), "8+28+28": (8, 28, 28)}


def listed():
    return [
        # one row: the norm of a single token (latency)
        dict(name="norm one token", op="norm", mod=False, batch=1, length=1, width=3072, dtype=BF16, train=False),
        # a training step's final norm over a ragged batch of short texts, in 32 bits, at a width that fills no tile
        dict(name="norm ragged fp32 train", op="norm", mod=False, batch=3, length=517, width=1000, dtype=F32, train=True),
        # fine-tuning a block: the image stream's modulated norm, two images of 4096 tokens
        dict(name="norm image stream train", op="norm", mod=True, batch=2, length=4096, width=3072, dtype=BF16, train=True),
        # four images of 16384 + 512 tokens: the largest sequences that the blocks are run with
        dict(name="norm long sequences train", op="norm", mod=True, batch=4, length=16896, width=3072, dtype=BF16, train=True),
        # one new token of eight requests, each at a position of its own (latency)
        dict(name="rope one token each", op="rope", batch=8, heads=24, kv_heads=24, length=1, axes="16+56+56", dtype=BF16, seq_major=False, train=False),
        # the joint text and image sequence of one picture
        dict(name="rope joint sequence", op="rope", batch=1, heads=24, kv_heads=24, length=4608, axes="16+56+56", dtype=BF16, seq_major=False, train=False),
        # pictures of different sizes in one batch, q and k as views of the token-major projection, with gradients
        dict(name="rope mixed sizes train", op="rope", batch=4, heads=24, kv_heads=24, length=1037, axes="16+56+56", dtype=BF16, seq_major=True, train=True),
        # a video's tokens (time, height, width) in 32 bits, fewer key heads than query heads
        dict(name="rope video fp32", op="rope", batch=1, heads=16, kv_heads=4, length=16896, axes="16+24+24", dtype=F32, seq_major=False, train=False),
        # the modulation projection of eight requests with an adapter each: one row per request
        dict(name="lora one row each", op="lora", batch=8, length=1, k=3072, n=18432, rank=16, adapters=8, dtype=BF16, gelu=False),
        # many small requests in one call, up-projection with its activation
        dict(name="lora many requests", op="lora", batch=48, length=5, k=1024, n=4096, rank=64, adapters=16, dtype=BF16, gelu=True),
        # the text stream of four requests, output projection
        dict(name="lora text stream", op="lora", batch=4, length=512, k=3072, n=3072, rank=32, adapters=6, dtype=BF16, gelu=False),
        # the q|k|v projection of two pictures' joint sequences with large adapters
        dict(name="lora joint qkv", op="lora", batch=2, length=4608, k=3072, n=9216, rank=128, adapters=4, dtype=BF16, gelu=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "rope", "lora", "lora"])
    if op == "norm":
        width = _log(rng, 64, 8192)
        if rng.random() < 0.85:
            width = max(8, width // 8 * 8)
        batch = rng.choice([1, 2, 3, 4, 7, 16])
        length = min(_log(rng, 1, 16384), max(1, 120_000_000 // (batch * width)))
        return dict(op=op, mod=rng.random() < 0.5, batch=batch, length=length, width=width, dtype=rng.choice([BF16, BF16, F32]), train=rng.random() < 0.7)
    if op == "rope":
        heads = rng.choice([1, 3, 8, 16, 24, 32])
        batch = rng.choice([1, 2, 5, 8, 16])
        length = min(_log(rng, 1, 16384), max(1, 90_000_000 // (batch * heads * 128)))
        return dict(op=op, batch=batch, heads=heads, kv_heads=rng.choice([h for h in (1, 2, 3, 4, 8, 16, 24, 32) if heads % h == 0]), length=length,
                    axes=rng.choice(sorted(AXES)), dtype=rng.choice([BF16, BF16, F32]), seq_major=rng.random() < 0.5, train=rng.random() < 0.5)
    batch = _log(rng, 1, 64)
    k, n = (8 * _log(rng, 8, 768) for _ in range(2))
    length = min(_log(rng, 1, 4608), max(1, 200_000_000_000 // (batch * k * n)))
    return dict(op=op, batch=batch, length=length, k=k, n=n, rank=rng.choice([4, 8, 16, 24, 32, 64, 128]), adapters=rng.choice([1, 4, 16]), dtype=BF16,
                gelu=rng.random() < 0.3)


def _normal(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, s = DTYPES[case["dtype"]], dict(case)
    B, L = case["batch"], case["length"]
    if case["op"] == "norm":
        C = case["width"]
        # rows with an offset of their own and a few wide channels, as residual streams have them
        x = _normal(g, B, L, C) * (1 + 4 * (torch.rand(C, generator=g, device="cuda") < 0.01)) + _normal(g, B, L, 1)
        s["x"] = x.to(dt)
        if case["mod"]:
            s["weight"], s["bias"] = (_normal(g, B, 1, C, scale=0.2).to(dt) for _ in range(2))
        else:
            s["weight"], s["bias"] = (1 + _normal(g, C, scale=0.1)).to(dt), _normal(g, C, scale=0.1).to(dt)
        if case["train"]:
            s["dy"] = _normal(g, B, L, C).to(dt)
            for name in ("x", "weight", "bias"):
                s[name].requires_grad_()
    elif case["op"] == "rope":
        axes, H, G = AXES[case["axes"]], case["heads"], case["kv_heads"]
        D = sum(axes)
        names = [("q", H), ("k", G)] + ([("dq", H), ("dk", G)] if case["train"] else [])
        for name, h in names:
            if case["seq_major"]:
                s[name] = _normal(g, B, L, h, D).to(dt).permute(0, 2, 1, 3)
            else:
                s[name] = _normal(g, B, h, L, D).to(dt)
        # every request has a frame, a first row and column and a row length of its own; the last axis runs fastest
        at = torch.arange(L, device="cuda") + torch.randint(0, 4096, (B, 1), generator=g, device="cuda")
        row = torch.randint(16, 129, (B, 1), generator=g, device="cuda")
        grid = torch.stack((at // (row * row), at // row % row, at % row), dim=-1)
        s["ids"] = (grid[..., 3 - len(axes):] if len(axes) > 1 else at[..., None]).float().contiguous()
        if case["train"]:
            for name in ("q", "k"):
                s[name].requires_grad_()
    else:
        K, N, R, A = case["k"], case["n"], case["rank"], case["adapters"]
        s["x"] = _normal(g, B, L, K).to(dt)
        s["w"] = _normal(g, N, K, scale=K**-0.5).to(dt)
        s["b"] = _normal(g, N, scale=0.1).to(dt)
        s["lora_a"] = _normal(g, A, R, K, scale=K**-0.5).to(dt)
        s["lora_b"] = _normal(g, A, N, R, scale=0.3 * R**-0.5).to(dt)
        s["lora_scale"] = 0.5 + torch.rand(A, generator=g, device="cuda")
        # -1: a request without an adapter
        s["adapter"] = torch.randint(0 if A == 1 else -1, A, (B,), generator=g, device="cuda")
    return s


def _norm_plain(s):
    dt = s["x"].dtype
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    factor = 1 + w if s["mod"] else w
    centred = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    hat = centred * rstd
    y = (hat * factor + b).to(dt)
    if not s["train"]:
        return y
    dy = s["dy"].float()
    rows = 1 if s["mod"] else (0, 1)
    g = dy * factor
    dx = rstd * (g - g.mean(-1, keepdim=True) - hat * (g * hat).mean(-1, keepdim=True))
    return y, dx.to(dt), (dy * hat).sum(rows).reshape(w.shape).to(dt), dy.sum(rows).reshape(w.shape).to(dt)


def _angles(s):
    """[B, 1, L, D/2] cosines and sines; the angles in 64 bits."""
    axes, dev = AXES[s["axes"]], s["ids"].device
    ids = s["ids"].double()
    angle = torch.cat([ids[..., i:i + 1] * THETA ** (-torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d) for i, d in enumerate(axes)], dim=-1)
    return torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]


def _rotate(x, c, s):
    even, odd = x[..., 0::2].float(), x[..., 1::2].float()
    return torch.stack((even * c - odd * s, even * s + odd * c), dim=-1).flatten(-2).to(x.dtype)


def _rope_plain(s):
    c, sn = _angles(s)
    out = _rotate(s["q"], c, sn), _rotate(s["k"], c, sn)
    return out + (_rotate(s["dq"], c, -sn), _rotate(s["dk"], c, -sn)) if s["train"] else out


def _gelu(v):
    return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))


def _lora_plain(s):
    x, pick = s["x"].float(), s["adapter"].clamp(min=0)
    scale = torch.where(s["adapter"] >= 0, s["lora_scale"][pick], 0.0)[:, None, None]
    low = x @ s["lora_a"][pick].float().transpose(1, 2) * scale
    y = x @ s["w"].float().T + s["b"].float() + low @ s["lora_b"][pick].float().transpose(1, 2)
    return (_gelu(y) if s["gelu"] else y).to(s["x"].dtype)


def run(state):
    if not own:
        with torch.no_grad():
            return {"norm": _norm_plain, "rope": _rope_plain, "lora": _lora_plain}[state["op"]](state)
    import triton_kernels_b200 as tk

    s = state
    if s["op"] == "norm":
        call = tk.layer_norm_modulation if s["mod"] else tk.layer_norm
        y = call(s["x"], s["weight"], s["bias"], EPS)
        if not s["train"]:
            return y
        return (y.detach(), *torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"]))
    if s["op"] == "rope":
        q, k = tk.apply_rope_axes(s["q"], s["k"], s["ids"], AXES[s["axes"]], THETA)
        if not s["train"]:
            return q, k
        return (q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"])))
    return tk.linear_lora(s["x"], s["w"], s["b"], s["lora_a"], s["lora_b"], s["adapter"], s["lora_scale"], "GELU" if s["gelu"] else "")


def work(case):
    size = 2 if case["dtype"] == BF16 else 4
    B, L = case["batch"], case["length"]
    if case["op"] == "norm":
        n, vec = B * L * case["width"], case["width"] * (B if case["mod"] else 1)
        times = 2 if case["train"] else 1  # x, y and, backwards, dy, dx; scale and offset and their gradients
        return {"bytes": size * times * (2 * n + 2 * vec), "flops": n * (25 if case["train"] else 9)}
    if case["op"] == "rope":
        axes = AXES[case["axes"]]
        n = B * L * (case["heads"] + case["kv_heads"]) * sum(axes)
        times = 2 if case["train"] else 1
        return {"bytes": size * times * 2 * n + 4 * B * L * len(axes), "flops": 3 * times * n}
    m, K, N, R = B * L, case["k"], case["n"], case["rank"]
    used = min(B, case["adapters"])
    return {"bytes": size * (m * K + m * N + N * K + N + used * R * (K + N)), "flops": 2 * m * (N * K + R * (K + N))}


def exact(case, seed):
    s = prepare(case, seed)
    wide = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if case["op"] == "norm":
        x, w, b = (wide[k].requires_grad_(case["train"]) for k in ("x", "weight", "bias"))
        var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
        y = (x - mean) / torch.sqrt(var + EPS)
        y = torch.addcmul(b, y, w + 1 if case["mod"] else w)
        if not case["train"]:
            return y
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), wide["dy"]))
    if case["op"] == "rope":
        axes = AXES[case["axes"]]
        steps = [(i, -2 * j / d * math.log(THETA)) for i, d in enumerate(axes) for j in range(d // 2)]
        which = torch.tensor([i for i, _ in steps], device="cuda")
        freq = torch.tensor([e for _, e in steps], device="cuda", dtype=torch.float64).exp()
        turn = torch.polar(torch.ones((), device="cuda", dtype=torch.float64), wide["ids"][..., which] * freq)[:, None]
        names = (("q", turn), ("k", turn)) + ((("dq", turn.conj()), ("dk", turn.conj())) if case["train"] else ())
        return tuple(torch.view_as_real(torch.view_as_complex(wide[k].contiguous().unflatten(-1, (-1, 2))) * t).flatten(-2) for k, t in names)
    out = []
    for x, a in zip(wide["x"], s["adapter"].tolist()):
        w = wide["w"] if a < 0 else torch.addmm(wide["w"], wide["lora_b"][a], wide["lora_a"][a], alpha=float(s["lora_scale"][a]))
        out.append(torch.addmm(wide["b"], x, w.T))
    y = torch.stack(out)
    if not case["gelu"]:
        return y
    # 0.5 (1 + tanh u) is the logistic function of 2u
    return y * torch.sigmoid(math.sqrt(8 / math.pi) * (y + 0.044715 * y**3))
