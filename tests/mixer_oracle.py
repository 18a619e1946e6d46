"""Plain 64-bit implementations of the operators beside the convolution, on the CPU: the recurrence
token by token, the rotation pair by pair, the norms as written. Test infrastructure only."""
import math

import torch


def attention(q, k, v, log_decay, scale, state=None, lengths=None):
    """(o, final state) of S_t = g S_{t-1} + k_t v_t^T, o_t = scale S_t^T q_t; tokens from lengths[b] on are
    left out and give 0. Differentiable."""
    q, k, v, log_decay = (x.double().cpu() if x.dtype != torch.float64 else x for x in (q, k, v, log_decay))
    B, T, H, Dk = q.shape
    G, Dv = H // k.shape[2], v.shape[3]
    g = torch.exp(log_decay)[:, None, None]
    o, last = [], []
    for b in range(B):
        n = T if lengths is None else int(lengths[b])
        S = torch.zeros(H, Dk, Dv, dtype=torch.float64) if state is None else state[b].double().cpu()
        rows = []
        for t in range(T):
            if t < n:
                kt, vt = (x[b, t].repeat_interleave(G, 0) for x in (k, v))
                S = g * S + kt[:, :, None] * vt[:, None, :]
                rows.append(scale * (q[b, t][:, None, :] @ S)[:, 0])
            else:
                rows.append(torch.zeros(H, Dv, dtype=torch.float64))
        o.append(torch.stack(rows))
        last.append(S)
    return torch.stack(o), torch.stack(last)


def attention_grads(q, k, v, log_decay, scale, go, gs, state=None, lengths=None):
    """(o, final, dq, dk, dv, d state) in 64 bits by automatic differentiation of the recurrence."""
    leaves = [x.detach().double().cpu().requires_grad_() for x in (q, k, v)]
    s0 = torch.zeros(q.shape[0], q.shape[2], q.shape[3], v.shape[3], dtype=torch.float64) if state is None else \
        state.detach().double().cpu()
    s0 = s0.clone().requires_grad_()
    o, last = attention(*leaves, log_decay.detach().double().cpu(), scale, s0, lengths)
    loss = 0.0
    if go is not None:
        keep = torch.ones(o.shape[:2], dtype=torch.bool)
        if lengths is not None:
            for b in range(len(keep)):
                keep[b, int(lengths[b]):] = False
        loss = loss + (o[keep] * go.detach().double().cpu()[keep]).sum()
    if gs is not None:
        loss = loss + (last * gs.detach().double().cpu()).sum()
    grads = torch.autograd.grad(loss, leaves + [s0], allow_unused=True)
    grads = [torch.zeros_like(x) if g is None else g for g, x in zip(grads, leaves + [s0])]
    return (o.detach(), last.detach(), *grads)


def attention_pairs(q, k, v, log_decay, scale, go, state, gs):
    """(o, final, dq, dk, dv, d state) in 64 bits from every pair of tokens, on the inputs' device: for lengths
    where the recurrence takes too long."""
    B, T, H, Dk = q.shape
    G = H // k.shape[2]
    d = [x.detach().double() for x in (q, k, v, go)]
    t = torch.arange(T, dtype=torch.float64, device=q.device)
    out = [torch.zeros(s, dtype=torch.float64, device=q.device) for s in (go.shape, gs.shape, q.shape, k.shape, v.shape, gs.shape)]
    gap = t[:, None] - t[None, :]
    for b in range(B):
        for h in range(H):
            ld, hk = log_decay[h].double(), h // G
            w = torch.where(gap >= 0, torch.exp(ld * gap.clamp(min=0)), torch.zeros_like(gap)) * scale
            qh, kh, vh, oh = d[0][b, :, h], d[1][b, :, hk], d[2][b, :, hk], d[3][b, :, h]
            s0, g1 = state[b, h].double(), gs[b, h].double()
            since, left = torch.exp(ld * (t + 1))[:, None], torch.exp(ld * (T - 1 - t))[:, None]
            p, r = (qh @ kh.t()) * w, (oh @ vh.t()) * w
            out[0][b, :, h] = p @ vh + scale * since * (qh @ s0)
            out[1][b, h] = (left * kh).t() @ vh + torch.exp(ld * T) * s0
            out[2][b, :, h] = r @ kh + scale * since * (oh @ s0.t())
            out[3][b, :, hk] += r.t() @ qh + left * (vh @ g1.t())
            out[4][b, :, hk] += p.t() @ oh + left * (kh @ g1)
            out[5][b, h] = scale * (since * qh).t() @ oh + torch.exp(ld * T) * g1
    return out


def rotary(x, table, positions, interleaved, inverse=False):
    """x [B, T, H, D] turned pair by pair; table [P, R] = cos | sin, positions [B, T] or None."""
    B, T, H, D = x.shape
    R = table.shape[1]
    y = x.detach().double().cpu().clone()
    table = table.double().cpu()
    for i in range(R // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
        p = torch.arange(T).expand(B, T) if positions is None else positions.long().cpu()
        c, s = table[p, i][..., None], table[p, R // 2 + i][..., None]
        if inverse:
            s = -s
        u, w = x[..., a].double().cpu(), x[..., b].double().cpu()
        y[..., a], y[..., b] = u * c - w * s, w * c + u * s
    return y


def block_norm(x, y, w_pre, w_post=None, gate=None, scale=None, activation="none", eps=1e-6):
    """(r, h) in 64 bits, differentiable; y None: (x, h)."""
    def norm(z):
        return z / torch.sqrt((z * z).mean(-1, keepdim=True) + eps)

    r = x
    if y is not None:
        m = y if w_post is None else norm(y) * w_post
        if gate is not None:
            act = {"none": lambda g: g, "sigmoid": lambda g: 1 / (1 + torch.exp(-g)),
                   "silu": lambda g: g / (1 + torch.exp(-g))}[activation]
            m = m * act(gate)
        if scale is not None:
            m = m * scale
        r = x + m
    return r, norm(r) * w_pre


def rel_l2(got, want):
    got, want = got.detach().double().cpu(), want.double().cpu()
    d, n = float((got - want).norm()), float(want.norm())
    return d / n if n else (0.0 if d == 0 else math.inf)
