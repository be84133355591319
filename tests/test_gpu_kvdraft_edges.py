"""Edges of drafts, cross attention and reading back on the GPU: lengths next to
2^31, and row offsets that contradict a call's own bounds."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_kvdraft_shapes import World

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


@pytest.mark.parametrize("how", ["cross", "draft"])
@pytest.mark.parametrize("dim,lens,new,group,most,per", [
    (128, [2500, 2300], [128, 100], 4, 96, 128),             # a grid of row tiles
    (128, [2400] * 60, [2] * 37 + [600] + [2] * 22, 4, 96, 128),  # counted through the sequences
    (128, [2400] * 60, [2] * 37 + [600] + [2] * 22, 4, 64, 32),
    (64, [2200] * 70, [1] * 5 + [300, 150] + [3] * 63, 2, 30, 32),
    (256, [2200] * 60, [3] * 59 + [200], 2, 60, 16),
])
def test_tokens_beyond_max_queries_are_left_out(ctx, dim, lens, new, group, most, per, how):
    """Offsets that give sequences more tokens than the call's bound: the row tiles that there is room
    for are right, and every other row is left as it is."""
    from gofann_amd import kvcache
    w = World(ctx, "bf16", dim, 64, 2, group, lens, new, seed=most)
    scale = 0.7 * dim ** -0.5
    call = (lambda b, **kw: w.cache.cross(b, w.q, scale=scale, **kw)) if how == "cross" else \
        (lambda b, **kw: w.cache.attend(b, w.q, scale=scale, sees=w.words, **kw))
    full_lse = torch.empty(w.n, 2 * group, device="cuda")
    full = call(w.batch, lse=full_lse)
    short = kvcache.KvBatch(w.table, w.batch._keep[1], w.batch._keep[2], queries=w.n, max_queries=most,
                            max_length=max(lens))
    room = -(-most * group // per) * per  # rows of a sequence
    nth = np.concatenate([np.arange(m) for m in new])
    row = torch.from_numpy(nth).cuda()[:, None, None] * group + torch.arange(group, device="cuda")
    there = (row < room).expand(w.n, 2, group).reshape(w.n, 2 * group)
    assert there.any() and not there.all()
    for _ in range(2):  # the second call finds the first one's notes in its scratch
        out, lse = torch.full_like(w.q, 99.0), torch.full_like(full_lse, 77.0)
        call(short, out=out, lse=lse)
        assert (out[~there] == 99.0).all() and (lse[~there] == 77.0).all()
        w.check(torch.where(there[..., None], out, full), torch.where(there, lse, full_lse), scale,
                None if how == "cross" else w.sees)
        call(w.batch)


@pytest.mark.parametrize("how", ["cross", "draft"])
@pytest.mark.parametrize("length,sequences", [(480_000, 1024), (470_000, 1000), (2000, 1024), (30_000, 200)])
def test_offsets_that_overlap_compute_nothing_out_of_place(ctx, how, length, sequences):
    """Every second sequence has all of the call's rows.  The longest count more tiles than 32 bits
    hold, where the bounds that the host goes by (rows in all) count a quarter of 2^30."""
    from gofann_amd import kvcache
    dim, heads, tokens, group, page = 64, 64, 64, 4, 256
    g = torch.Generator(device="cuda").manual_seed(length)
    rnd = lambda lo, hi, *s: torch.randint(lo, hi, s, device="cuda", generator=g).to(torch.uint8)  # noqa: E731
    cache = kvcache.KvCache(ctx, rnd(0, 256, 8, heads, page, dim // 2), rnd(123, 127, 8, heads, page, dim // 32),
                            rnd(0, 256, 8, heads, page // 8, 16, 8, dim // 32),
                            rnd(123, 127, 8, heads, page // 8, dim // 32, 8))
    dev = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    table = torch.full((sequences, -(-length // page)), -1, dtype=torch.int32, device="cuda")
    table[:, :8] = torch.arange(8, dtype=torch.int32, device="cuda")[:table.shape[1]]
    offsets = dev(([0, tokens] * sequences)[:sequences + 1])
    lengths = dev([length] * sequences)
    q = torch.randn(tokens, heads * group, dim, device="cuda", generator=g).to(cache.dtype)
    words = torch.full((tokens, tokens // 32), -1, dtype=torch.int32, device="cuda")
    call = (lambda b, **kw: cache.cross(b, q, **kw)) if how == "cross" else \
        (lambda b, **kw: cache.attend(b, q, sees=words, **kw))
    one = kvcache.KvBatch(table[:1], lengths[:1], dev([0, tokens]), queries=tokens, max_queries=tokens, max_length=length)
    want = call(one)
    around = torch.full((3, *q.shape), 99.0, dtype=q.dtype, device="cuda")
    lse = torch.full((3, tokens, heads * group), 77.0, device="cuda")
    for _ in range(2):
        bad = kvcache.KvBatch(table, lengths, offsets, queries=tokens, max_queries=tokens, max_length=length)
        call(bad, out=around[1], lse=lse[1])
        assert (around[::2] == 99.0).all() and (lse[::2] == 77.0).all()
        if length > 400_000:
            assert (around[1] == 99.0).all() and (lse[1] == 77.0).all()
        assert torch.equal(call(one), want)


@pytest.mark.parametrize("how", ["cross", "draft"])
@pytest.mark.parametrize("filt", [0.0, 0.5])
@pytest.mark.parametrize("dim,group,lens,new,tiles", [
    (256, 2, [700, 300, 500, 301, 640, 333, 450, 600], [300, 200, 300, 1, 17, 300, 0, 260], 380_000),
    (128, 4, [650] * 100, [1] * 50 + [600] + [3] * 49, 120_000),  # more sequences than are ordered by length
])
def test_bounds_past_a_count_of_tiles(ctx, dim, group, lens, new, tiles, filt, how):
    """A length's bound so loose that tiles are not counted: a row tile a workgroup."""
    from gofann_amd import kvcache
    w = World(ctx, "bf16", dim, 256, 64, group, lens, new, filt, seed=dim)
    pages = tiles // 8
    table = torch.full((len(lens), pages), -1, dtype=torch.int32, device="cuda")
    table[:, :w.table.shape[1]] = w.table
    row_tiles = -(-max(new) * group // 128)
    grid, slots = row_tiles * len(lens), sum(new) * group // 128 + len(lens)
    assert ((slots if 2 * slots <= grid else grid) + row_tiles) * 64 * tiles > 1 << 30
    w.batch = kvcache.KvBatch(table, w.batch._keep[1], w.batch._keep[2], queries=w.n, max_queries=max(new),
                              max_length=tiles * 32, visible=w.batch._keep[3])
    w.run(how, set(range(8)) | set(range(48, 53)))
