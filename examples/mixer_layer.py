"""A mixer layer with both its halves, trained and then run token by token: attention over the last tokens (`norm_rope`, `token_attention`)
beside the slot memory (`write_memory`, `read_snapshots`), and for generation their serving forms (`norm_rope_append`,
`token_attention_step` over ring caches; `StreamingScan`).

    python examples/mixer_layer.py            # train on a copying task, then generate; needs a B200

The task: random symbols, each sequence repeats what it said `LAG` tokens before, which the window reaches."""
import os
import sys

import torch
from torch import nn
from torch.nn import functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "smal-memory-llm_b200"))
import slotscan_b200 as S   # noqa: E402

VOCAB, LAG, WINDOW = 64, 5, 16


class MixerLayer(nn.Module):
    """y = x + out([attention over the last WINDOW tokens, read of the slot memory])."""

    def __init__(self, width=256, heads=4, kv_heads=2, dim=64, slots=32, block=8, positions=4096):
        super().__init__()
        self.H, self.KV, self.D, self.N, self.G = heads, kv_heads, dim, slots, block
        sizes = [(heads + 2 * kv_heads) * dim, 2 * heads * dim, heads * dim, 2 * heads]
        self.sizes = sizes
        self.inp = nn.Linear(width, sum(sizes), bias=False)            # q, k, v | slot key, slot value | read query | gate, forget
        self.out = nn.Linear(2 * heads * dim, width, bias=False)
        self.q_norm, self.k_norm = nn.Parameter(torch.ones(dim)), nn.Parameter(torch.ones(dim))
        self.log_sharp, self.log_temp = nn.Parameter(torch.full((heads,), 2.0)), nn.Parameter(torch.tensor(2.0))
        self.table = S.rope_table(positions, dim, device="cuda")       # not a buffer: it stays float32 when the layer becomes bfloat16

    def streams(self, x):
        """Everything that one projection gives; slices of it, read in place."""
        B, T, _ = x.shape
        token, slot, read, gates = self.inp(F.rms_norm(x, x.shape[-1:])).split(self.sizes, -1)
        q, k, v = token.view(B, T, -1, self.D).split((self.H, self.KV, self.KV), 2)
        sk, sv = slot.view(B, T, 2 * self.H, self.D).split(self.H, 2)
        gate, forget = gates.float().sigmoid().split(self.H, -1)
        return (q, k, v), (sk, sv, gate, 0.1 * forget), read.view(B, T, self.H, 1, self.D)

    def join(self, x, o, rd):
        B, T, _ = x.shape
        return x + self.out(torch.cat((o.reshape(B, T, -1), rd.to(x.dtype).reshape(B, T, -1)), -1))

    def read(self, rq, memory):
        sharp = self.log_sharp.exp().view(1, 1, self.H, 1).expand(rq.shape[:-1]).contiguous()
        return S.read_snapshots(rq, sharp, *memory, self.G)

    def forward(self, x):
        """Training, or a whole prompt: x (B, T, width)."""
        (q, k, v), (sk, sv, gate, forget), rq = self.streams(x)
        q, k = S.norm_rope(q, k, self.table, self.q_norm, self.k_norm)
        o = S.token_attention(q, k, v, window=WINDOW)
        memory = S.write_memory(sk, sv, gate, forget, self.N, self.log_temp.exp(), G=self.G, out_dtype=x.dtype)
        return self.join(x, o, self.read(rq, memory))


class Generation:
    """The state of one layer while it runs: ring caches of WINDOW rows, the memory as the running block reads it, the block's writes."""

    def __init__(self, layer, batch, dtype, device):
        self.layer, self.pos = layer, torch.zeros(batch, dtype=torch.int32, device=device)
        self.kc = torch.zeros(batch, WINDOW, layer.KV, layer.D, dtype=dtype, device=device)
        self.vc = torch.zeros_like(self.kc)
        self.scan = S.StreamingScan(layer.N, layer.log_temp.exp(), G=layer.G, out_dtype=dtype)
        z = torch.zeros(batch, 1, layer.H, layer.N, layer.D, dtype=torch.float32, device=device)
        self.memory, self.pending = S.writer_epilogue(z, z, dtype), []

    def _write(self, slot, dtype):
        """The block's writes; what the next block reads is the state that they leave."""
        self.scan.push(*slot)
        k, v = (t.view(self.pos.shape[0], 1, self.layer.H, self.layer.N, self.layer.D) for t in self.scan.state[:2])
        self.memory = S.writer_epilogue(k, v, dtype)

    @torch.no_grad()
    def prompt(self, x):
        """A prompt whose length is a multiple of the layer's block; the output of all its tokens."""
        layer, T = self.layer, x.shape[1]
        (q, k, v), slot, _ = layer.streams(x)
        n = min(T, WINDOW)                                             # the rows that the next tokens will see
        S.norm_rope_append(q[:, -n:], k[:, -n:], v[:, -n:], self.kc, self.vc, self.pos + (T - n), layer.table, layer.q_norm, layer.k_norm)
        self.pos += T
        self._write(slot, x.dtype)
        return layer(x)

    @torch.no_grad()
    def step(self, x):
        """The next token of every sequence, x (B, 1, width)."""
        layer = self.layer
        (q, k, v), slot, rq = layer.streams(x)
        q = S.norm_rope_append(q, k, v, self.kc, self.vc, self.pos, layer.table, layer.q_norm, layer.k_norm)
        o = S.token_attention_step(q, self.kc, self.vc, self.pos, window=WINDOW)
        y = layer.join(x, o, layer.read(rq, self.memory))
        self.pos += 1
        self.pending.append(slot)
        if len(self.pending) == layer.G:
            self._write([torch.cat(t, 1) for t in zip(*self.pending)], x.dtype)
            self.pending = []
        return y


class Model(nn.Module):
    def __init__(self, width=256, **kw):
        super().__init__()
        self.embed, self.layer = nn.Embedding(VOCAB, width), MixerLayer(width, **kw)
        self.head = nn.Linear(width, VOCAB, bias=False)

    def forward(self, tokens):
        return self.head(self.layer(self.embed(tokens)))


def sequences(batch, length, gen):
    """Symbols that repeat with period LAG."""
    first = torch.randint(VOCAB, (batch, LAG), generator=gen)
    return first.repeat(1, -(-length // LAG))[:, :length].cuda()


def train(model, steps=150, batch=16, length=128, seed=0):
    """The losses of the steps."""
    gen = torch.Generator().manual_seed(seed)
    opt = torch.optim.AdamW(model.parameters(), lr=2e-3)
    losses = []
    for _ in range(steps):
        tokens = sequences(batch, length + 1, gen)
        loss = F.cross_entropy(model(tokens[:, :-1])[:, LAG:].float().flatten(0, 1), tokens[:, 1 + LAG:].flatten())
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


@torch.no_grad()
def generate(model, prompt, n):
    """The n symbols that follow `prompt` (B, T), T a multiple of the block; greedy."""
    gen = Generation(model.layer, prompt.shape[0], model.head.weight.dtype, prompt.device)
    logits = model.head(gen.prompt(model.embed(prompt))[:, -1:])
    out = []
    for _ in range(n):
        out.append(logits.argmax(-1))
        logits = model.head(gen.step(model.embed(out[-1])))
    return torch.cat(out, 1)


def main():
    torch.manual_seed(0)
    model = Model().to("cuda", torch.bfloat16)
    losses = train(model)
    tokens = sequences(4, 64 + 40, torch.Generator().manual_seed(1))
    right = (generate(model, tokens[:, :64], 40) == tokens[:, 64:]).float().mean()
    print("loss %.3f -> %.3f over %d steps; %.0f%% of 40 generated symbols are the repeated ones" % (losses[0], losses[-1], len(losses), 100 * right))


if __name__ == "__main__":
    main()
