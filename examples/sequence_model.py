"""A small sequence model that trains and generates with the framework's operators.

Its blocks mix the tokens by turns with linear attention (rotary positions, a decay for each head, key and value
heads shared by the query heads) and with the long convolution; between two blocks one operator gates and
normalises the block's output, adds it to the residual and normalises the sum. Training takes whole
sequences. Generation reads prompts of different lengths at once and goes on token by token: a linear
attention block keeps one state [Dk, Dv] a head, whatever the length, a convolution block the inputs so far.

    python examples/sequence_model.py [--steps N] [--generate N]

trains on sequences that mostly follow a fixed permutation of the tokens, and continues two of them.
"""
import argparse
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from sffft_amd import mixers, torch_ops  # noqa: E402

ops = torch.ops.sffft
BF16 = torch.bfloat16


def project(x, w):
    return F.linear(x, w.to(x.dtype))


class Attention(torch.nn.Module):
    """Linear attention over H heads, Hk of them with keys and values of their own."""

    def __init__(self, C, H, Hk, length):
        super().__init__()
        self.H, self.Hk, self.D = H, Hk, C // H
        self.w_in = torch.nn.Parameter(torch.randn((H + 2 * Hk) * self.D + C, C) * C ** -0.5)
        self.w_out = torch.nn.Parameter(torch.randn(C, C) * C ** -0.5)
        # heads that forget within a few tokens up to heads that remember the whole length
        self.register_buffer("log_decay", -torch.exp(torch.linspace(-0.5, -torch.log(torch.tensor(length)), H)))
        self.register_buffer("table", mixers.rotary_table(2 * length, self.D // 2))

    def heads(self, h, positions):
        """q, k, v [B, T, heads, D] and the gate, views of one projection; q and k are rotated."""
        nq, nk = self.H * self.D, self.Hk * self.D
        q, k, v, gate = project(h, self.w_in).split([nq, nk, nk, h.shape[-1]], -1)
        q, k, v = (x.unflatten(-1, (-1, self.D)) for x in (q, k, v))
        q, k = ops.rotary(q, k, self.table, positions)
        return q, k, v, gate

    def forward(self, h, lengths=None):
        q, k, v, gate = self.heads(h, None)
        o, state = ops.linear_attention(q, k, v, self.log_decay, self.D ** -0.5, None, lengths)
        return project(o.flatten(2), self.w_out), gate, state

    def step(self, h, positions, state):
        """One token of each sequence [B, 1, C]; the state is updated in place."""
        q, k, v, gate = self.heads(h, positions[:, None])
        o = ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], self.log_decay, state, self.D ** -0.5)
        return project(o.flatten(1)[:, None], self.w_out), gate


class Convolution(torch.nn.Module):
    """The long convolution of every channel with a filter of its own, up to `length` tokens."""

    def __init__(self, C, length):
        super().__init__()
        self.length = length
        self.w_in = torch.nn.Parameter(torch.randn(2 * C, C) * C ** -0.5)
        self.w_out = torch.nn.Parameter(torch.randn(C, C) * C ** -0.5)
        decay = torch.exp(-torch.arange(length) / torch.logspace(0, 2, C)[:, None])
        self.filter = torch.nn.Parameter(torch.randn(C, length) * decay / decay.norm(dim=1, keepdim=True))
        self.conv = torch_ops.LongConv()

    def forward(self, h, lengths=None):
        u, gate = project(h, self.w_in).chunk(2, -1)
        T = u.shape[1]
        u = F.pad(u.transpose(1, 2), (0, self.length - T)).contiguous()
        past = u
        if lengths is not None:  # what lies past a prompt's end is no token
            past = u * (torch.arange(self.length, device=u.device) < lengths[:, None])[:, None]
        y = self.conv(u, self.filter)[..., :T].transpose(1, 2).contiguous()
        return project(y, self.w_out), gate, past

    def step(self, h, positions, past):
        u, gate = project(h, self.w_in).chunk(2, -1)
        b = torch.arange(u.shape[0], device=u.device)
        past[b, :, positions] = u[:, 0]
        lag = positions[:, None] - torch.arange(self.length, device=u.device)
        k = self.filter[:, lag.clamp(min=0)].transpose(0, 1) * (lag >= 0)[:, None]  # [B, C, length]
        y = (k * past.float()).sum(-1).to(u.dtype)
        return project(y[:, None], self.w_out), gate


class Model(torch.nn.Module):
    def __init__(self, vocab=64, C=256, H=4, Hk=2, length=512, blocks=2):
        super().__init__()
        self.length = length
        self.embed = torch.nn.Parameter(torch.randn(vocab, C))
        self.head = torch.nn.Parameter(torch.zeros(vocab, C))
        self.mixers = torch.nn.ModuleList(
            m for _ in range(blocks) for m in (Attention(C, H, Hk, length), Convolution(C, length)))
        n = len(self.mixers)
        self.pre = torch.nn.Parameter(torch.ones(n + 1, C))  # of the input of each block, and of the head
        self.post = torch.nn.Parameter(torch.ones(n, C))  # of its output
        self.scale = torch.nn.Parameter(torch.full((n, C), 0.5))

    def run(self, tokens, mix):
        """mix(i, block, h) gives a block's output and gate."""
        if tokens.shape[1] > self.length:
            raise ValueError(f"at most {self.length} tokens, got {tokens.shape[1]}")
        x = F.embedding(tokens, self.embed.to(BF16))
        h = ops.pre_norm(x, self.pre[0])
        for i, block in enumerate(self.mixers):
            y, gate = mix(i, block, h)
            x, h = ops.block_norm(x, y, self.pre[i + 1], self.post[i], gate, self.scale[i], "silu")
        return project(h, self.head).float()

    def forward(self, tokens):
        """Logits [B, T, vocab] of tokens [B, T]."""
        return self.run(tokens, lambda i, block, h: block(h)[:2])

    def prompt(self, tokens, lengths):
        """Logits, and what each block keeps after lengths[b] tokens."""
        kept = []

        def mix(i, block, h):
            y, gate, state = block(h, lengths)
            kept.append(state)
            return y, gate

        return self.run(tokens, mix), kept

    def step(self, tokens, positions, kept):
        """Logits [B, vocab] of one token a sequence at its position; `kept` is updated."""
        return self.run(tokens[:, None], lambda i, block, h: block.step(h, positions, kept[i]))[:, 0]

    @torch.no_grad()
    def generate(self, tokens, lengths, n):
        """n more tokens, the likeliest each, of prompts tokens[b, :lengths[b]]; with the logits they were taken from."""
        shortest, longest = int(lengths.min()), int(lengths.max())
        if shortest < 1:
            raise ValueError("an empty prompt has no last token to go on from")
        if longest > tokens.shape[1] or longest + n - 1 > self.length:
            raise ValueError(f"prompts of {longest} tokens in {tokens.shape[1]} and {n} more: the blocks keep {self.length}")
        logits, kept = self.prompt(tokens, lengths)
        last = logits[torch.arange(tokens.shape[0], device=tokens.device), lengths.long() - 1]
        out, seen = [], []
        for i in range(n):
            seen.append(last)
            out.append(last.argmax(-1))
            if i + 1 < n:
                last = self.step(out[-1], lengths.long() + i, kept)
        return torch.stack(out, 1), torch.stack(seen, 1)


def sequences(batch, length, vocab, device, generator):
    """Each token follows its predecessor by a fixed permutation nine times in ten."""
    follow = torch.randperm(vocab, generator=torch.Generator().manual_seed(0))
    x = torch.randint(vocab, (batch, length), generator=generator)
    keep = torch.rand(batch, length, generator=generator) < 0.9
    for t in range(1, length):
        x[:, t] = torch.where(keep[:, t], follow[x[:, t - 1]], x[:, t])
    return x.to(device)


def train(model, steps, batch=8, vocab=64, seed=1):
    """The loss of each step."""
    device = model.embed.device
    generator = torch.Generator().manual_seed(seed)
    opt = torch.optim.AdamW(model.parameters(), lr=3e-3)
    losses = []
    for _ in range(steps):
        x = sequences(batch, model.length, vocab, device, generator)
        loss = F.cross_entropy(model(x)[:, :-1].flatten(0, 1), x[:, 1:].flatten())
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--steps", type=int, default=40)
    ap.add_argument("--generate", type=int, default=16)
    args = ap.parse_args()
    torch.manual_seed(0)
    model = Model().cuda()
    for i, loss in enumerate(train(model, args.steps)):
        if i % 10 == 0 or i + 1 == args.steps:
            print(f"step {i}: loss {loss:.3f}")
    prompts = sequences(2, 100, 64, "cuda", torch.Generator().manual_seed(2))
    lengths = torch.tensor([100, 37], dtype=torch.int32, device="cuda")
    tokens, _ = model.generate(prompts, lengths, args.generate)
    for b, n in enumerate(lengths.tolist()):
        print(f"prompt of {n} tokens ending {prompts[b, n - 4:n].tolist()}: {tokens[b].tolist()}")


if __name__ == "__main__":
    main()
