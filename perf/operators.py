"""Workloads of the sequence-mixing operators beside the long convolution: linear attention with a
decay for each head (prompts, training, single tokens), rotary positions, and the norms around a
block fused with its gate and residual scale.

`listed()` names the cases, `prepare` makes a case's inputs, `run` makes one call: in plain torch
operations of 32 bits (`own = False`), or through the framework's operators (`own = True`).
`exact` gives the same outputs from the definitions in 64 bits, and `work` the bytes and
operations that a call cannot do without. Channels (768, 1536) and lengths (up to 131072) are
those of this repository's configurations.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one stream answering: a single token, 768 channels as 12 heads of 64
        {"name": "attn_step_one", "op": "step", "B": 1, "H": 12, "Hk": 12, "Dk": 64, "Dv": 64, "io": "bf16",
         "slots": 0},
        # a serving batch of 96 streams in a state cache of 128 slots, 1536 channels
        {"name": "attn_step_batch", "op": "step", "B": 96, "H": 12, "Hk": 12, "Dk": 128, "Dv": 128, "io": "bf16",
         "slots": 128},
        # prompts of different lengths in one batch, one of them empty, that continue earlier ones
        {"name": "attn_prompt_ragged", "op": "attn", "B": 5, "T": 1237, "H": 12, "Hk": 12, "Dk": 64, "Dv": 64,
         "io": "bf16", "ragged": True, "state": True, "train": False},
        # one prompt of the longest length of the repository, 1536 channels
        {"name": "attn_prompt_long", "op": "attn", "B": 1, "T": 131072, "H": 12, "Hk": 12, "Dk": 128, "Dv": 128,
         "io": "bf16", "ragged": False, "state": False, "train": False},
        # a training step of the batch and width of the convolution's benchmark
        {"name": "attn_train", "op": "attn", "B": 8, "T": 2048, "H": 12, "Hk": 12, "Dk": 64, "Dv": 64, "io": "bf16",
         "ragged": False, "state": False, "train": True},
        # full precision, key and value heads shared by three query heads, odd length, carried state
        {"name": "attn_train_shared", "op": "attn", "B": 3, "T": 1531, "H": 12, "Hk": 4, "Dk": 96, "Dv": 64,
         "io": "fp32", "ragged": True, "state": True, "train": True},
        # positions of one token in each of 8 streams far into long contexts
        {"name": "rotary_step", "op": "rotary", "B": 8, "T": 1, "H": 12, "Hk": 12, "D": 64, "R": 64, "io": "bf16",
         "interleaved": False, "scaling": "parts", "table": 131072, "train": False},
        # a training step, half of the head rotated, interleaved pairs, shared key heads
        {"name": "rotary_train", "op": "rotary", "B": 8, "T": 2048, "H": 12, "Hk": 4, "D": 128, "R": 64, "io": "bf16",
         "interleaved": True, "scaling": "none", "table": 2048, "train": True},
        # a long prompt in full precision, positions stretched
        {"name": "rotary_long", "op": "rotary", "B": 1, "T": 65536, "H": 12, "Hk": 12, "D": 64, "R": 64, "io": "fp32",
         "interleaved": False, "scaling": "linear", "table": 131072, "train": False},
        # one token in each of 8 streams
        {"name": "norm_step", "op": "norm", "B": 8, "T": 1, "C": 768, "io": "bf16", "gate": "token", "act": "silu",
         "post": True, "scale": True, "train": False},
        # full precision, odd sizes, one gate for a whole sequence, with its gradient
        {"name": "norm_odd", "op": "norm", "B": 4, "T": 1021, "C": 1531, "io": "fp32", "gate": "sequence",
         "act": "none", "post": True, "scale": False, "train": True},
        # a training step of the long-filter configuration's batch, width and length
        {"name": "norm_train", "op": "norm", "B": 4, "T": 16384, "C": 1536, "io": "bf16", "gate": "token",
         "act": "silu", "post": True, "scale": True, "train": True},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the same ranges; a tensor has at most 16 Mi elements (training) or 48 Mi."""
    op = rng.choice(["step", "attn", "attn", "rotary", "norm"])
    io = rng.choice(["bf16", "bf16", "fp32"])
    train = rng.random() < 0.5
    limit = (16 << 20) if train else (48 << 20)
    H = rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
    Hk = rng.choice([n for n in (1, 2, 4, H) if H % n == 0])
    if op == "step":
        B = _log_int(rng, 1, 160)
        return {"op": op, "B": B, "H": H, "Hk": Hk, "Dk": rng.choice([32, 64, 96, 128]),
                "Dv": rng.choice([32, 64, 96, 128]), "io": io, "slots": rng.choice([0, B + rng.randint(1, 40)])}
    if op == "attn":
        B = rng.randint(1, 8)
        Dk, Dv = rng.choice([32, 64, 72, 96, 128]), rng.choice([32, 64, 96, 128])
        T = _log_int(rng, 1, min(65536 if not train else 8192, limit // (B * H * max(Dk, Dv))))
        return {"op": op, "B": B, "T": T + (T == 3072), "H": H, "Hk": Hk, "Dk": Dk, "Dv": Dv, "io": io,
                "ragged": rng.random() < 0.4, "state": rng.random() < 0.5, "train": train}
    if op == "rotary":
        B = rng.randint(1, 8)
        D = rng.choice([32, 64, 96, 128, 256])
        T = _log_int(rng, 1, min(65536, limit // (B * H * D)))
        return {"op": op, "B": B, "T": T + (T == 3072), "H": H, "Hk": Hk, "D": D,
                "R": rng.choice([D, D // 2, D // 4]), "io": io, "interleaved": rng.random() < 0.5,
                "scaling": rng.choice(["none", "linear", "stretched", "parts"]), "table": rng.choice([65536, 131072]),
                "train": train}
    B = rng.randint(1, 8)
    C = rng.choice([96, 384, 768, 1024, 1531, 1536, 2047, 2048, 4096, _log_int(rng, 64, 6000)])
    C += C == 3072
    T = _log_int(rng, 1, min(16384, limit // (B * C)))
    return {"op": op, "B": B, "T": T + (T == 3072), "C": C, "io": io, "gate": rng.choice(["token", "sequence", "none"]),
            "act": rng.choice(["none", "sigmoid", "silu"]), "post": rng.random() < 0.75, "scale": rng.random() < 0.5,
            "train": train}


# ---- inputs ---------------------------------------------------------------------------------


def _lengths(case):
    """Valid tokens of each sequence: in a ragged batch every fifth is empty, the next full, the others in between."""
    B, T = case["B"], case["T"]
    if not case["ragged"]:
        return [T] * B
    return [0 if b % 5 == 3 else T if b % 5 == 0 else max(1, (T * (37 + 11 * (b % 5))) // 97) for b in range(B)]


def frequencies(R, base, scaling, factor=8.0, trained=16384):
    """Angle per position of each of the R/2 pairs, in 64 bits. `linear` divides positions by
    `factor`; `stretched` raises the base so that the slowest pair is divided by it; `parts`
    divides the pairs that turn less than once over the trained length, keeps those that turn
    more than 32 times, and blends between."""
    e = torch.arange(0, R, 2, dtype=torch.float64) / R
    if scaling == "stretched" and R > 2:
        base = base * factor ** (R / (R - 2))
    f = base ** -e
    if scaling == "linear":
        return f / factor
    if scaling == "parts":
        turns = trained * f / (2 * math.pi)
        keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
        return f * keep + f / factor * (1 - keep)
    return f


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dt = DTYPES[case["io"]]

    def randn(*shape, dtype=dt, mul=1.0, add=0.0):
        return (torch.randn(shape, generator=g, device=dev) * mul + add).to(dtype)

    s = {"case": case}
    op = case["op"]
    if op in ("step", "attn"):
        B, H, Hk, Dk, Dv = (case[n] for n in ("B", "H", "Hk", "Dk", "Dv"))
        # memories of 32 to 4096 tokens over the heads
        span = torch.linspace(5, 12, H, dtype=torch.float64) if H > 1 else torch.tensor([8.0], dtype=torch.float64)
        s["log_decay"] = torch.log1p(-(2.0 ** -span)).float().to(dev)
        s["scale"] = Dk ** -0.5
    if op == "step":
        s["q"], s["k"], s["v"] = randn(B, H, Dk), randn(B, Hk, Dk), randn(B, Hk, Dv)
        n = case["slots"] or B
        s["state"] = randn(n, H, Dk, Dv, dtype=torch.float32, mul=4.0)
        s["slots"] = torch.randperm(n, generator=g, device=dev)[:B].int() if case["slots"] else None
    elif op == "attn":
        T = case["T"]
        s["q"], s["k"], s["v"] = randn(B, T, H, Dk), randn(B, T, Hk, Dk), randn(B, T, Hk, Dv)
        s["state"] = randn(B, H, Dk, Dv, dtype=torch.float32, mul=4.0) if case["state"] else None
        s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=dev) if case["ragged"] else None
        if case["train"]:
            s["do"] = randn(B, T, H, Dv)
            s["ds"] = randn(B, H, Dk, Dv, dtype=torch.float32)
            for n in ("q", "k", "v", "state"):
                if s[n] is not None:
                    s[n].requires_grad_(True)
    elif op == "rotary":
        B, T, H, Hk, D, R = (case[n] for n in ("B", "T", "H", "Hk", "D", "R"))
        s["q"], s["k"] = randn(B, T, H, D), randn(B, T, Hk, D)
        angle = torch.arange(case["table"], dtype=torch.float64, device=dev)[:, None] * frequencies(
            R, 10000.0, case["scaling"]).to(dev)
        s["table"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        start = torch.randint(0, case["table"] - T + 1, (B, 1), generator=g, device=dev)
        s["positions"] = (start + torch.arange(T, device=dev)).int()
        if case["train"]:
            s["dq"], s["dk"] = randn(B, T, H, D), randn(B, T, Hk, D)
            for n in ("q", "k"):
                s[n].requires_grad_(True)
    else:
        B, T, C = case["B"], case["T"], case["C"]
        s["x"], s["y"] = randn(B, T, C), randn(B, T, C, mul=0.5)
        s["gate"] = None if case["gate"] == "none" else randn(B, T if case["gate"] == "token" else 1, C)
        s["w_pre"] = randn(C, dtype=torch.float32, mul=0.1, add=1.0)
        s["w_post"] = randn(C, dtype=torch.float32, mul=0.1, add=1.0) if case["post"] else None
        s["scale"] = randn(C, dtype=torch.float32, mul=0.1, add=0.5) if case["scale"] else None
        if case["train"]:
            s["dr"], s["dh"] = randn(B, T, C), randn(B, T, C)
            for n in ("x", "y", "gate", "w_pre", "w_post", "scale"):
                if s[n] is not None:
                    s[n].requires_grad_(True)
    return s


# ---- plain forms, 32 bits -------------------------------------------------------------------


def _powers(log_decay, n):
    """exp(log_decay * n) for a whole-number tensor n, heads first; 0 where n is negative."""
    n = n.to(log_decay.dtype)
    ld = log_decay.reshape(-1, *([1] * n.dim()))
    return torch.where(n >= 0, torch.exp(ld * n.clamp(min=0)), torch.zeros((), device=n.device, dtype=ld.dtype))


def plain_attention(q, k, v, log_decay, scale, state, lengths, chunk=128):
    """Chunks of tokens: products within a chunk, and each chunk's entering state from those before it."""
    dt, dev = q.dtype, q.device
    B, T, H, Dk = q.shape
    G, Dv = H // k.shape[2], v.shape[3]
    t = torch.arange(T, device=dev)
    n = torch.full((B,), T, device=dev) if lengths is None else lengths.long()
    valid = (t[None, :] < n[:, None])[:, :, None, None]
    zero = torch.zeros((), device=dev)
    q, k, v = (torch.where(valid, x.float(), zero) for x in (q, k, v))
    k, v = (x.repeat_interleave(G, 2) if G > 1 else x for x in (k, v))
    nc = -(-T // chunk)
    qc, kc, vc = (torch.nn.functional.pad(x, (0, 0, 0, 0, 0, nc * chunk - T)).reshape(B, nc, chunk, H, -1)
                  .permute(0, 3, 1, 2, 4) for x in (q, k, v))  # [B, H, nc, chunk, D]
    i = torch.arange(chunk, device=dev)
    within = _powers(log_decay, i[:, None] - i[None, :])  # [H, chunk, chunk]
    o = torch.matmul(torch.matmul(qc, kc.transpose(-1, -2)) * within[None, :, None], vc)
    u = torch.matmul((kc * _powers(log_decay, chunk - 1 - i)[None, :, None, :, None]).transpose(-1, -2), vc)
    c = torch.arange(nc, device=dev)
    between = _powers(log_decay, (c[:, None] - 1 - c[None, :]) * chunk)  # [H, nc, nc]
    entering = torch.matmul(between[None], u.reshape(B, H, nc, Dk * Dv)).reshape(B, H, nc, Dk, Dv)
    if state is not None:
        entering = entering + _powers(log_decay, c * chunk)[None, :, :, None, None] * state.float()[:, :, None]
    o = (o + torch.matmul(qc, entering) * _powers(log_decay, i + 1)[None, :, None, :, None]) * scale
    o = o.permute(0, 2, 3, 1, 4).reshape(B, nc * chunk, H, Dv)[:, :T]
    o = torch.where(valid, o, zero).to(dt)
    left = _powers(log_decay, n[:, None] - 1 - t[None, :])  # [H, B, T]
    last = torch.matmul((k * left.permute(1, 2, 0)[..., None]).permute(0, 2, 3, 1), v.permute(0, 2, 1, 3))
    if state is not None:
        last = last + _powers(log_decay, n).t()[:, :, None, None] * state.float()
    return o, last


def plain_step(q, k, v, log_decay, state, scale, slots):
    G = q.shape[1] // k.shape[1]
    k, v = (x.float().repeat_interleave(G, 1) for x in (k, v))
    old = state if slots is None else state[slots.long()]
    new = old * torch.exp(log_decay)[None, :, None, None] + k[..., :, None] * v[..., None, :]
    o = (torch.matmul(q.float()[..., None, :], new)[..., 0, :] * scale).to(q.dtype)
    if slots is None:
        state.copy_(new)
    else:
        state[slots.long()] = new
    return o, state


def _plain_rotate(x, cos, sin, R, interleaved):
    z = x.float()
    if interleaved:
        a, b = z[..., 0:R:2], z[..., 1:R:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = z[..., :R // 2], z[..., R // 2:R]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, z[..., R:]], -1).to(x.dtype)


def plain_rotary(q, k, table, positions, interleaved):
    R = table.shape[1]
    row = table[positions.long()][:, :, None]
    cos, sin = row[..., :R // 2], row[..., R // 2:]
    return _plain_rotate(q, cos, sin, R, interleaved), _plain_rotate(k, cos, sin, R, interleaved)


def _plain_rms(z, w, eps):
    z = z * torch.rsqrt((z * z).mean(-1, keepdim=True) + eps)
    return z if w is None else z * w


def plain_norm(x, y, w_pre, w_post, gate, scale, act, eps):
    m = y.float() if w_post is None else _plain_rms(y.float(), w_post, eps)
    if gate is not None:
        a = gate.float()
        a = torch.sigmoid(a) if act == "sigmoid" else a * torch.sigmoid(a) if act == "silu" else a
        m = m * a
    if scale is not None:
        m = m * scale
    r = x.float() + m
    return r.to(x.dtype), _plain_rms(r, w_pre, eps).to(x.dtype)


# ---- one pass -------------------------------------------------------------------------------

EPS = 1e-6


def _ops():
    from sffft_amd import torch_ops  # noqa: F401  (registers torch.ops.sffft)

    return torch.ops.sffft


def run(s):
    case = s["case"]
    op = case["op"]
    if op == "step":
        a = (s["q"], s["k"], s["v"], s["log_decay"], s["state"], s["scale"], s["slots"])
        return (_ops().linear_attention_step(*a), s["state"]) if own else plain_step(*a)
    if op == "attn":
        a = (s["q"], s["k"], s["v"], s["log_decay"], s["scale"], s["state"], s["lengths"])
        out = _ops().linear_attention(*a) if own else plain_attention(*a)
        wanted, grads = ("q", "k", "v", "state"), ("do", "ds")
    elif op == "rotary":
        a = (s["q"], s["k"], s["table"], s["positions"], case["interleaved"])
        out = _ops().rotary(*a) if own else plain_rotary(*a)
        wanted, grads = ("q", "k"), ("dq", "dk")
    else:
        a = (s["x"], s["y"], s["w_pre"], s["w_post"], s["gate"], s["scale"], case["act"], EPS)
        out = _ops().block_norm(*a) if own else plain_norm(*a)
        wanted, grads = ("x", "y", "gate", "w_pre", "w_post", "scale"), ("dr", "dh")
    if not case["train"]:
        return tuple(out)
    leaves = [s[n] for n in wanted if s[n] is not None]
    return tuple(o.detach() for o in out) + torch.autograd.grad(tuple(out), leaves, [s[n] for n in grads])


# ---- what a pass cannot do without ----------------------------------------------------------


def work(case):
    e = 2 if case["io"] == "bf16" else 4
    op = case["op"]
    if op == "step":
        B, H, Hk, Dk, Dv = (case[n] for n in ("B", "H", "Hk", "Dk", "Dv"))
        return {"bytes": B * (8 * H * Dk * Dv + e * (H * Dk + Hk * Dk + Hk * Dv + H * Dv)) + 4 * H,
                "flops": 5 * B * H * Dk * Dv}
    if op == "attn":
        B, T, H, Hk, Dk, Dv = (case[n] for n in ("B", "T", "H", "Hk", "Dk", "Dv"))
        n = sum(_lengths(case))
        qkv, state = H * Dk + Hk * Dk + Hk * Dv, 4 * B * H * Dk * Dv
        has = 1 if case["state"] else 0
        # a recurrent step takes an update and a product of Dk x Dv; backwards the states again, their
        # gradients, and three products
        b = e * (n * qkv + B * T * H * Dv) + state * (1 + has) + 4 * H
        f = 4 * n * H * Dk * Dv
        if case["train"]:
            b += e * (n * (qkv + H * Dv) + B * T * qkv) + state * (1 + 2 * has)
            f += 10 * n * H * Dk * Dv
        return {"bytes": b, "flops": f}
    if op == "rotary":
        B, T, H, Hk, D, R = (case[n] for n in ("B", "T", "H", "Hk", "D", "R"))
        n = 2 if case["train"] else 1
        rows = min(B * T, case["table"])
        return {"bytes": n * (2 * e * B * T * (H + Hk) * D + 4 * rows * R + 4 * B * T),
                "flops": n * 3 * B * T * (H + Hk) * R}
    B, T, C = case["B"], case["T"], case["C"]
    gate = {"none": 0, "token": B * T * C, "sequence": B * C}[case["gate"]]
    vectors = 4 * C * (1 + case["post"] + case["scale"])
    b, f = e * (4 * B * T * C + gate) + vectors, 14 * B * T * C
    if case["train"]:
        b += e * (6 * B * T * C + 2 * gate) + 2 * vectors
        f += 40 * B * T * C
    return {"bytes": b, "flops": f}


# ---- the definitions in 64 bits -------------------------------------------------------------


def _exact_head(q, k, v, ld, scale, s0, do, ds, rows=2048):
    """One head of one sequence, every pair of tokens: o, last state, and for do, ds the gradients."""
    n = q.shape[0]
    t = torch.arange(n, dtype=torch.float64, device=q.device)
    o = torch.empty(n, v.shape[1], dtype=torch.float64, device=q.device)
    grads = None if do is None else [torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)]
    for a in range(0, n, rows):
        z = min(n, a + rows)
        gap = t[a:z, None] - t[None, :z]
        w = torch.where(gap >= 0, torch.exp(ld * gap), torch.zeros_like(gap)) * scale
        p = (q[a:z] @ k[:z].t()) * w
        o[a:z] = p @ v[:z]
        if grads:
            dp = (do[a:z] @ v[:z].t()) * w
            grads[0][a:z] = dp @ k[:z]
            grads[1][:z] += dp.t() @ q[a:z]
            grads[2][:z] += p.t() @ do[a:z]
    since = torch.exp(ld * (t + 1))[:, None]
    o += scale * since * (q @ s0)
    left = torch.exp(ld * (n - 1 - t))[:, None]
    last = (left * k).t() @ v + math.exp(float(ld) * n) * s0
    if grads:
        grads[0] += scale * since * (do @ s0.t())
        grads[1] += left * (v @ ds.t())
        grads[2] += left * (k @ ds)
        grads.append(scale * (since * q).t() @ do + math.exp(float(ld) * n) * ds)
    return o, last, grads


def _exact_attention(s):
    case = s["case"]
    B, T, H, Hk, Dk, Dv = (case[n] for n in ("B", "T", "H", "Hk", "Dk", "Dv"))
    if B * H * T * T > 3e11:
        return None
    d = {n: s[n].detach().double() for n in ("q", "k", "v", "state", "do", "ds") if s.get(n) is not None}
    new = lambda *shape: torch.zeros(shape, dtype=torch.float64, device="cuda")  # noqa: E731
    o, last = new(B, T, H, Dv), new(B, H, Dk, Dv)
    g = [new(B, T, H, Dk), new(B, T, Hk, Dk), new(B, T, Hk, Dv), new(B, H, Dk, Dv)] if case["train"] else None
    for b, n in enumerate(_lengths(case)):
        for h in range(H):
            hk = h // (H // Hk)
            s0 = d["state"][b, h] if "state" in d else new(Dk, Dv)
            do, ds = (d["do"][b, :n, h], d["ds"][b, h]) if g else (None, None)
            ob, lb, gb = _exact_head(d["q"][b, :n, h], d["k"][b, :n, hk], d["v"][b, :n, hk],
                                     s["log_decay"][h].double(), s["scale"], s0, do, ds)
            o[b, :n, h], last[b, h] = ob, lb
            if g:
                g[0][b, :n, h] = gb[0]
                g[1][b, :n, hk] += gb[1]
                g[2][b, :n, hk] += gb[2]
                g[3][b, h] = gb[3]
    return (o, last) + (tuple(g if case["state"] else g[:3]) if g else ())


def _exact_step(s):
    G = s["case"]["H"] // s["case"]["Hk"]
    state = s["state"].double()
    rows = torch.arange(s["case"]["B"], device="cuda") if s["slots"] is None else s["slots"].long()
    q = s["q"].double()
    k, v = (s[n].double().repeat_interleave(G, 1) for n in ("k", "v"))
    state[rows] = torch.exp(s["log_decay"].double())[None, :, None, None] * state[rows] + torch.einsum(
        "bhi,bhj->bhij", k, v)
    return s["scale"] * torch.einsum("bhi,bhij->bhj", q, state[rows]), state


def _exact_rotary(s):
    case = s["case"]
    R = case["R"]
    angle = s["positions"].double()[..., None, None] * frequencies(R, 10000.0, case["scaling"]).cuda()
    turn = torch.polar(torch.ones_like(angle), angle)

    def rotate(x, turn):
        x = x.detach().double()
        y = x.clone()
        first, second = (slice(0, R, 2), slice(1, R, 2)) if case["interleaved"] else (slice(0, R // 2), slice(R // 2, R))
        z = torch.complex(x[..., first], x[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        return y

    out = rotate(s["q"], turn), rotate(s["k"], turn)
    return out + (rotate(s["dq"], turn.conj()), rotate(s["dk"], turn.conj())) if case["train"] else out


def _exact_norm(s):
    """Forward and, by the chain rule written out, backward, in blocks of rows to bound the memory."""
    case = s["case"]
    B, T, C = case["B"], case["T"], case["C"]
    d = {n: (s[n].detach() if s.get(n) is not None else None)
         for n in ("x", "y", "gate", "w_pre", "w_post", "scale", "dr", "dh")}
    one = torch.ones(C, dtype=torch.float64, device="cuda")
    wq = d["w_pre"].double()
    wp = one if d["w_post"] is None else d["w_post"].double()
    sc = one if d["scale"] is None else d["scale"].double()
    new = lambda *shape: torch.zeros(shape, dtype=torch.float64, device="cuda")  # noqa: E731
    r, h = new(B, T, C), new(B, T, C)
    dx, dy, dg = new(B, T, C), new(B, T, C), new(*d["gate"].shape) if d["gate"] is not None else None
    dwq, dwp, dsc = new(C), new(C), new(C)
    for b in range(B):
        x, y = d["x"][b].double(), d["y"][b].double()
        sy = ((y ** 2).sum(-1, keepdim=True) / C + EPS) ** -0.5 if case["post"] else new(T, 1) + 1
        n = y * sy * wp
        g = one if d["gate"] is None else d["gate"][b].double()
        e = 1 / (1 + torch.exp(-g))
        a, da = {"none": (g, torch.ones_like(g)), "sigmoid": (e, e * (1 - e)),
                 "silu": (g * e, e * (1 + g * (1 - e)))}[case["act"] if d["gate"] is not None else "none"]
        r[b] = x + sc * a * n
        sr = ((r[b] ** 2).sum(-1, keepdim=True) / C + EPS) ** -0.5
        h[b] = r[b] * sr * wq
        if case["train"]:
            dh, hat = d["dh"][b].double(), r[b] * sr
            gh = dh * wq
            dr = d["dr"][b].double() + sr * (gh - hat * (gh * hat).sum(-1, keepdim=True) / C)
            dwq += (dh * hat).sum(0)
            dsc += (dr * a * n).sum(0)
            dx[b] = dr
            if dg is not None:
                dg[b] = (dr * sc * n * da).sum(0, keepdim=True) if case["gate"] == "sequence" else dr * sc * n * da
            dn = dr * sc * a
            if case["post"]:
                yh = y * sy
                dwp += (dn * yh).sum(0)
                gy = dn * wp
                dy[b] = sy * (gy - yh * (gy * yh).sum(-1, keepdim=True) / C)
            else:
                dy[b] = dn
    if not case["train"]:
        return r, h
    grads = [dx, dy] + ([dg] if dg is not None else []) + [dwq] + ([dwp] if case["post"] else []) + (
        [dsc] if case["scale"] else [])
    return (r, h) + tuple(grads)


def exact(case, seed):
    s = prepare(case, seed)
    return {"step": _exact_step, "attn": _exact_attention, "rotary": _exact_rotary, "norm": _exact_norm}[case["op"]](s)
