"""A decoding loop over a long context in the 4-bit key/value cache: the calls
of gofann_amd.kvcache as a serving program makes them.

    python -m gofann_amd.longcontext --context 65536 --steps 16

One attention layer with random weights: a prompt is written in chunks (each
chunk attends over everything before it), then every step appends one token a
sequence, chooses the blocks to read under a filter and attends over them.
Prints the mean time of a step, over all positions and over the chosen blocks,
and the share of the full attention's weight that the chosen blocks hold.
"""
from __future__ import annotations

import argparse
import time

import torch

from . import _lib
from .kvcache import KvBatch, KvCache


class Session:
    """Sequences of equal capacity whose pages are handed out in order."""

    def __init__(self, ctx: _lib.Context, *, sequences: int, capacity: int, kv_heads: int = 8,
                 dim: int = 128, page: int = 64, dtype: torch.dtype = torch.bfloat16):
        self.cache = KvCache.empty(ctx, pages=sequences * -(-capacity // page), kv_heads=kv_heads,
                                   dim=dim, page=page, dtype=dtype)
        dev = self.cache.device
        width = -(-capacity // page)
        self.table = torch.arange(sequences * width, dtype=torch.int32, device=dev).reshape(sequences, width)
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device=dev)
        self.sequences, self.capacity, self.filled = sequences, capacity, 0
        self.visible = torch.full((sequences, -(-capacity // 32)), -1, dtype=torch.int32, device=dev)

    def grow(self, tokens: int) -> KvBatch:
        """The batch of `tokens` further tokens of every sequence."""
        if self.filled + tokens > self.capacity:
            raise ValueError("the sequences are full")
        self.filled += tokens
        self.lengths.fill_(self.filled)
        n = self.sequences
        off = torch.arange(0, n * tokens + 1, tokens, dtype=torch.int32, device=self.table.device)
        return KvBatch(self.table, self.lengths, off, queries=n * tokens, max_queries=tokens,
                       max_length=self.filled, visible=self.visible)

    def hide(self, sequence: int, begin: int, end: int) -> None:
        """Positions [begin, end) of a sequence out of sight, in whole words of 32."""
        if begin % 32 or end % 32:
            raise ValueError("hidden spans start and end at multiples of 32")
        self.visible[sequence, begin // 32:end // 32] = 0

    def step(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, width: int = 0,
             lse: torch.Tensor | None = None) -> torch.Tensor:
        """Appends the tokens' keys and values and attends with their queries:
        over everything visible, or over the `width` blocks chosen for each.  A
        step that is refused leaves the sequences as long as they were."""
        tokens, rest = divmod(q.shape[0], self.sequences)
        if rest:
            raise ValueError("a step has as many tokens for each of the sequences")
        before = self.filled
        batch = self.grow(tokens)
        try:
            self.cache.append(batch, k, v)
            blocks = self.cache.select(batch, q, width) if width else None
            return self.cache.attend(batch, q, blocks=blocks, lse=lse)
        except Exception:
            # What was written lies past the end again; the next step's append
            # writes over it and renews its pages' boxes.
            self.filled = before
            self.lengths.fill_(before)
            raise


def main(argv=None) -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--context", type=int, default=32768)
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--sequences", type=int, default=4)
    ap.add_argument("--heads", type=int, default=32)
    ap.add_argument("--kv-heads", type=int, default=8)
    ap.add_argument("--dim", type=int, default=128)
    ap.add_argument("--width", type=int, default=64, help="blocks of 64 positions a token reads")
    ap.add_argument("--chunk", type=int, default=1024)
    a = ap.parse_args(argv)
    ctx = _lib.Context(0)
    s = Session(ctx, sequences=a.sequences, capacity=a.context + 2 * a.steps + 64, kv_heads=a.kv_heads,
                dim=a.dim)
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = lambda n, h: torch.randn(n, h, a.dim, device="cuda", generator=g).to(torch.bfloat16)  # noqa: E731
    done = 0
    torch.cuda.synchronize()
    began = time.perf_counter()
    while done < a.context:
        m = min(a.chunk, a.context - done)
        n = m * a.sequences
        s.step(rows(n, a.heads), rows(n, a.kv_heads), rows(n, a.kv_heads))
        done += m
    torch.cuda.synchronize()
    print(f"prompt: {a.sequences} x {a.context} positions in {time.perf_counter() - began:.3f} s", flush=True)
    if a.context >= 1024:
        s.hide(0, 256, 512)
    for width in (0, a.width):
        inputs = [(rows(a.sequences, a.heads), rows(a.sequences, a.kv_heads), rows(a.sequences, a.kv_heads))
                  for _ in range(a.steps)]
        torch.cuda.synchronize()
        began = time.perf_counter()
        for q, k, v in inputs:
            s.step(q, k, v, width)
        torch.cuda.synchronize()
        what = f"{width} blocks a token" if width else "all positions"
        print(f"step over {what}: {(time.perf_counter() - began) / a.steps * 1e6:.1f} us", flush=True)
    batch = KvBatch(s.table, s.lengths, max_length=s.filled, visible=s.visible)
    q = rows(a.sequences, a.heads)
    every = torch.empty(a.sequences, a.heads, device="cuda")
    some = torch.empty_like(every)
    s.cache.attend(batch, q, lse=every)
    s.cache.attend(batch, q, blocks=s.cache.select(batch, q, a.width), lse=some)
    print(f"weight in the chosen blocks: {torch.exp(some - every).mean().item():.3f} of all", flush=True)
    ctx.close()


if __name__ == "__main__":
    main()
