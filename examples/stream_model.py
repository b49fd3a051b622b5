"""A small sequence model over streams: signatures of windows of a path are the tokens, a block of attention and a gated
recurrence mixes them, trained end to end through the signatures, then run one window at a time.

    python examples/stream_model.py [--steps 30]

Synthetic data: paths of different lengths whose drift changes its sign now and then; the model tells each window's drift.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import pysiglib_amd as P  # noqa: E402
from pysiglib_amd import torch_api as A  # noqa: E402

CHANNELS, DEGREE, WINDOW = 3, 3, 16
WIDTH, HEADS, KV_HEADS, DIM = 256, 4, 2, 64
LONGEST = 512


class StreamModel(torch.nn.Module):
    def __init__(self, dtype=torch.bfloat16, device="cuda"):
        super().__init__()
        make = lambda a, b: torch.nn.Linear(a, b, dtype=dtype, device=device)       # noqa: E731
        self.dtype = dtype
        # the path's own small network: gradients reach it through the signature
        self.mix = torch.nn.Linear(CHANNELS, CHANNELS, bias=False, device=device)
        self.embed = make(P.sig_length(CHANNELS, DEGREE), WIDTH)
        self.qkv = make(WIDTH, (HEADS + 2 * KV_HEADS) * DIM)
        self.q_weight = torch.nn.Parameter(torch.ones(DIM, device=device))
        self.k_weight = torch.nn.Parameter(torch.ones(DIM, device=device))
        self.attended = make(HEADS * DIM, WIDTH)
        self.gates = make(WIDTH, 2 * WIDTH)
        self.remembered = make(WIDTH, WIDTH)
        self.answer = make(WIDTH, 1)
        self.cos, self.sin = P.rotary_tables(LONGEST, DIM, device=device)

    def tokens(self, windows):
        """(windows, WINDOW + 1, CHANNELS) -> (windows, WIDTH)."""
        return self.embed(A.sig(self.mix(windows), DEGREE).to(self.dtype))

    def parts(self, h, positions):
        rows = self.qkv(h).view(-1, HEADS + 2 * KV_HEADS, DIM)
        q, k = A.norm_rotary(rows[:, :HEADS], rows[:, HEADS:HEADS + KV_HEADS], self.q_weight, self.k_weight, self.cos, self.sin, positions)
        return q, k, rows[:, HEADS + KV_HEADS:]

    def decays(self, h):
        x, gate = self.gates(h).chunk(2, -1)
        return x, -torch.nn.functional.softplus(gate)

    def forward(self, windows, offsets, positions):
        """Streams packed behind each other: one answer for each window."""
        h = self.tokens(windows)
        q, k, v = self.parts(h, positions)
        h = h + self.attended(A.attention(q, k, v, offsets, offsets).flatten(1))
        x, log_decay = self.decays(h)
        h = h + self.remembered(A.linear_recurrence(x, log_decay, offsets=offsets)[0])
        return self.answer(h).squeeze(-1).float()

    def memory(self, streams):
        """What serving keeps for each stream: keys, values, how many of them, and the recurrence's state."""
        device = self.q_weight.device
        room = lambda: torch.zeros((streams, LONGEST, KV_HEADS, DIM), dtype=self.dtype, device=device)       # noqa: E731
        return dict(k=room(), v=room(), lengths=torch.zeros(streams, dtype=torch.int32, device=device),
                    state=torch.zeros((streams, WIDTH), device=device),
                    queries=torch.arange(streams + 1, dtype=torch.int32, device=device),
                    places=LONGEST * torch.arange(streams + 1, dtype=torch.int32, device=device))

    @torch.no_grad()
    def step(self, windows, memory):
        """The next window of each stream."""
        h = self.tokens(windows)
        q, k, v = self.parts(h, memory["lengths"])
        streams = torch.arange(len(windows), device=h.device)
        memory["k"][streams, memory["lengths"].long()] = k
        memory["v"][streams, memory["lengths"].long()] = v
        memory["lengths"] += 1
        out, _ = P.attention(q, memory["k"].flatten(0, 1), memory["v"].flatten(0, 1), memory["queries"], memory["places"],
                             k_lengths=memory["lengths"])
        h = h + self.attended(out.flatten(1))
        x, log_decay = self.decays(h)
        h = h + self.remembered(P.linear_recurrence_step(x, log_decay, memory["state"]))
        return self.answer(h).squeeze(-1).float()


def streams(count, gen, device="cuda"):
    """Windows of all streams behind each other, where the streams begin, each window's place in its own, and its drift."""
    lengths = torch.randint(5, 60, (count,), generator=gen)
    total = int(lengths.sum())
    offsets = torch.cat((torch.zeros(1, dtype=torch.long), lengths.cumsum(0)))
    positions = torch.arange(total) - offsets[:-1].repeat_interleave(lengths)
    drift = torch.where(torch.rand(total, generator=gen) < 0.2, -1.0, 1.0).cumprod(0)
    steps = 0.25 * torch.randn((total, WINDOW, CHANNELS), generator=gen)
    steps[..., 0] += 0.08 * drift[:, None]
    windows = torch.cat((torch.zeros(total, 1, CHANNELS), steps.cumsum(1)), 1)
    return windows.to(device), offsets.int().to(device), positions.int().to(device), drift.to(device)


def train(model, steps, gen, rate=3e-3, say=print):
    optimizer = torch.optim.Adam(model.parameters(), lr=rate)
    losses = []
    for step in range(steps):
        windows, offsets, positions, drift = streams(64, gen)
        loss = torch.nn.functional.binary_cross_entropy_with_logits(model(windows, offsets, positions), (drift + 1) / 2)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(float(loss.detach()))
        if step % 10 == 0 or step == steps - 1:
            say("step %d: loss %.4f" % (step, losses[-1]))
    return losses


@torch.no_grad()
def serve(model, gen):
    """Streams as a whole and window by window: the largest difference of their answers, and the answers' size."""
    windows, offsets, positions, _ = streams(16, gen)
    whole = model(windows, offsets, positions)
    starts, memory, worst = offsets[:-1].long(), model.memory(16), 0.0
    lengths = (offsets[1:] - offsets[:-1]).long()
    for t in range(int(lengths.max())):
        now = starts + torch.minimum(torch.full_like(lengths, t), lengths - 1)        # streams that ended repeat their last window
        difference = (model.step(windows[now], memory) - whole[now]).abs()
        worst = max(worst, float(difference[t < lengths].max()))
    return worst, float(whole.abs().mean())


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=30)
    args = parser.parse_args()
    torch.manual_seed(0)
    gen = torch.Generator().manual_seed(0)
    model = StreamModel()
    train(model, args.steps, gen)
    print("window by window against whole streams: largest difference %.4f, answers of size %.3f" % serve(model, gen))


if __name__ == "__main__":
    main()
