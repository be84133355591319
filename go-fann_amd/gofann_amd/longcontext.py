"""A decoding loop over a long context in the 4-bit key/value cache: the calls
of gofann_amd.kvcache as a serving program makes them.

    python -m gofann_amd.longcontext --context 65536 --steps 16

One attention layer with random weights: a prompt is written in chunks (each
chunk attends over everything before it), then every step appends one token a
sequence, chooses the blocks to read under a filter and attends over them; with
--draft every step drafts a tree of so many tokens, attends with it and keeps the
path that (random) answers accept.  Prints the mean time of a step, over all
positions, over the chosen blocks and with drafts, and the share of the full
attention's weight that the chosen blocks hold.
"""
from __future__ import annotations

import argparse
import time

import torch

from . import _lib
from .kvcache import KvBatch, KvCache, draft_accept, draft_tree


DEPTH = 8  # of a drafted tree that is kept, in main()


class Session:
    """Sequences of equal capacity whose pages are handed out in order."""

    pending = None  # a draft that is not settled: its batch, its parents, `filled` before it
    loose = False   # drafts were settled: the sequences may be shorter than `filled`

    def __init__(self, ctx: _lib.Context, *, sequences: int, capacity: int, kv_heads: int = 8,
                 dim: int = 128, page: int = 64, dtype: torch.dtype = torch.bfloat16):
        self.cache = KvCache.empty(ctx, pages=sequences * -(-capacity // page), kv_heads=kv_heads,
                                   dim=dim, page=page, dtype=dtype)
        dev = self.cache.device
        width = -(-capacity // page)
        self.table = torch.arange(sequences * width, dtype=torch.int32, device=dev).reshape(sequences, width)
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device=dev)
        # The sequences' lengths are the device's; `filled` is the most that any can have.
        self.sequences, self.capacity, self.filled = sequences, capacity, 0
        self.visible = torch.full((sequences, -(-capacity // 32)), -1, dtype=torch.int32, device=dev)

    def grow(self, tokens: int) -> KvBatch:
        """The batch of `tokens` further tokens of every sequence."""
        if self.pending is not None:
            raise ValueError("a draft is not settled")
        if self.filled + tokens > self.capacity and self.loose:
            # Only the device knows how many tokens of the drafts were kept: it is
            # asked, and waited for, where the bound would refuse.
            self.filled, self.loose = int(self.lengths.max()), False
        if self.filled + tokens > self.capacity:
            raise ValueError("the sequences are full")
        self.filled += tokens
        self.lengths += tokens
        n = self.sequences
        off = torch.arange(0, n * tokens + 1, tokens, dtype=torch.int32, device=self.table.device)
        return KvBatch(self.table, self.lengths, off, queries=n * tokens, max_queries=tokens,
                       max_length=self.filled, visible=self.visible)

    def _shrink(self, tokens: int) -> None:
        # What was written lies past the end again; the next append writes over
        # it and renews its pages' boxes.
        self.filled -= tokens
        self.lengths -= tokens

    def _tokens(self, q: torch.Tensor) -> int:
        tokens, rest = divmod(q.shape[0], self.sequences)
        if rest:
            raise ValueError("a step has as many tokens for each of the sequences")
        return tokens

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
        tokens = self._tokens(q)
        batch = self.grow(tokens)
        try:
            self.cache.append(batch, k, v)
            blocks = self.cache.select(batch, q, width) if width else None
            return self.cache.attend(batch, q, blocks=blocks, lse=lse)
        except Exception:
            self._shrink(tokens)
            raise

    def draft(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, parents: torch.Tensor,
              lse: torch.Tensor | None = None) -> torch.Tensor:
        """Appends a tree of drafted tokens to every sequence (the first of each
        is the one chosen last, parents as draft_tree takes them) and attends with
        them: each over what came before the draft, its ancestors and itself.  The
        sequences hold the whole draft until `settle`."""
        tokens = self._tokens(q)
        batch = self.grow(tokens)
        before = self.filled - tokens
        try:
            sees, _ = draft_tree(self.cache.ctx, batch, parents)
            self.cache.append(batch, k, v)
            out = self.cache.attend(batch, q, sees=sees, lse=lse)
        except Exception:
            self._shrink(tokens)
            raise
        self.pending = batch, parents, before
        return out

    def settle(self, drafted: torch.Tensor, chosen: torch.Tensor, width: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Keeps of the draft the path, of at most `width` tokens, that the answers
        `chosen` to its tokens accept (`drafted`: what each of them is).  Returns
        the path and the answer to its last token, which the next step begins with."""
        if self.pending is None:
            raise ValueError("there is no draft to settle")
        batch, parents, before = self.pending
        path, lengths, answer = draft_accept(self.cache.ctx, batch, parents, drafted, chosen, width)
        self.cache.keep(batch, path)
        self.lengths.copy_(lengths)
        self.filled = before + min(width, batch.max_queries)
        self.pending, self.loose = None, True
        return path, answer


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
    ap.add_argument("--draft", type=int, default=0, help="tokens of a drafted tree, in steps of their own")
    a = ap.parse_args(argv)
    ctx = _lib.Context(0)
    s = Session(ctx, sequences=a.sequences, capacity=a.context + (2 + DEPTH) * (a.steps + 1) + 64 + a.draft, kv_heads=a.kv_heads,
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
    if a.draft:
        n = a.sequences * a.draft
        whole = lambda top: torch.randint(0, top, (n,), device="cuda", generator=g, dtype=torch.int32)  # noqa: E731
        at = torch.arange(a.draft, device="cuda", dtype=torch.int32).repeat(a.sequences)
        inputs = [(rows(n, a.heads), rows(n, a.kv_heads), rows(n, a.kv_heads),
                   torch.div(at - 1, 3, rounding_mode="floor"), whole(4), whole(4)) for _ in range(a.steps + 1)]
        kept = torch.zeros(a.sequences, dtype=torch.int64, device="cuda")
        for i, (q, k, v, parents, drafted, chosen) in enumerate(inputs):
            if i == 1:  # the first step makes the workspace
                torch.cuda.synchronize()
                kept.zero_()
                began = time.perf_counter()
            s.draft(q, k, v, parents)
            kept += (s.settle(drafted, chosen, DEPTH)[0] >= 0).sum(1)
        torch.cuda.synchronize()
        print(f"step with {a.draft} drafted tokens: {(time.perf_counter() - began) / a.steps * 1e6:.1f} us, "
              f"{kept.double().mean().item() / a.steps:.2f} of them kept", flush=True)
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
