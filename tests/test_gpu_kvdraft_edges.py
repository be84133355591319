"""Edges of drafts, cross attention and reading back on the GPU: lengths next to
2^31, and row offsets that contradict a call's own bounds."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(gpu_ctx):
    return gpu_ctx


@pytest.mark.parametrize("page", [32, 64, 128, 256])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_reading_behind_a_length_next_to_2_to_the_31(ctx, page, dim):
    """The blocks that the longest draft of the call spans lie past position 2^31 for a sequence of
    such a length.  Its token has no page and is zero, and the others are what they are without it."""
    from gofann_amd import kvcache
    g = torch.Generator(device="cuda").manual_seed(page + dim)
    rnd = lambda lo, hi, *s: torch.randint(lo, hi, s, device="cuda", generator=g).to(torch.uint8)  # noqa: E731
    pages, heads, many = 4000 // page, 2, 3000
    cache = kvcache.KvCache(ctx, rnd(0, 256, pages, heads, page, dim // 2), rnd(123, 127, pages, heads, page, dim // 32),
                            rnd(0, 256, pages, heads, page // 8, 16, 8, dim // 32),
                            rnd(123, 127, pages, heads, page // 8, dim // 32, 8))
    dev = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    table = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(3, 1)
    alone = kvcache.KvBatch(table[:1], dev([many + 7]), dev([0, many]), queries=many, max_queries=many, max_length=many + 7)
    want = cache.read(alone)
    for far in (0x7FFFFF00, 0x7FFFFFFF, 0x7FFFFFFF - 5 * page):
        batch = kvcache.KvBatch(table, dev([far, many + 7, far]), dev([0, 1, 1 + many, 4 + many]), queries=many + 4,
                                max_queries=many, max_length=0x7FFFFF00)
        rows = [torch.full((many + 4, heads, dim), 9.0, dtype=cache.dtype, device="cuda") for _ in range(2)]
        cache.read(batch, k=rows[0], v=rows[1])
        for got, held in zip(rows, want):
            assert torch.equal(got[1:1 + many], held)
            assert (got[:1] == 0).all() and (got[1 + many:] == 0).all()
