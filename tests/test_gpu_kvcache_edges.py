"""Edges of the 4-bit key/value cache on the GPU against its plain 64-bit
definition: filters that are slices, sequences longer than their page table,
batches of very unequal chunks, long chunks under filters and holes."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kv_reference as ref
from test_gpu_kvcache import check_attend, device_batch, device_cache, documents, rows, spread

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(gpu_ctx):
    return gpu_ctx


def with_filter(b: ref.Batch, visible: torch.Tensor, **kw):
    """The batch on the device under another filter tensor."""
    from gofann_amd import kvcache
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    return kvcache.KvBatch(dev(b.table), dev(np.array(b.lens, np.int32)), dev(b.offsets),
                           queries=b.queries, max_queries=max(b.new), max_length=max(b.lens),
                           visible=visible, **kw)


# ---- filters ------------------------------------------------------------------

@pytest.mark.parametrize("new", [[1, 1, 1], [1, 9, 3]])
@pytest.mark.parametrize("width", [1, 4, 16])
def test_a_sliced_filter_hides_what_lies_past_its_words(ctx, width, new):
    """Columns of a larger tensor whose other bits are all set: positions past
    the slice are hidden, in the last row as in the others."""
    lens = [200, 130, 490]
    b = ref.Batch(32, lens, new, seed=5, visible=lambda s, n, r: r.random(n) < 0.7)
    b.bits[:, 32 * width:] = False
    big = torch.full((3, 20), -1, dtype=torch.int32, device="cuda")
    part = big[:, 20 - width:]
    words = np.packbits(b.bits[:, :32 * width].reshape(3, width, 32), axis=-1, bitorder="little")
    part.copy_(torch.from_numpy(words.view(np.int32)[..., 0].copy()))
    c = ref.Cache(b.pages, 2, 32, 64, "bf16", seed=1)
    ref.fill(c, b, seed=2)
    q, q64 = rows(np.random.default_rng(3), b.queries, 6, 64, "bf16")
    d, db = device_cache(ctx, c), with_filter(b, part)
    lse = torch.empty((b.queries, 6), device="cuda")
    check_attend(d.attend(db, q, lse=lse), lse, *ref.attend(c, b, q64, 64 ** -0.5))
    got = d.select(db, q, 5)
    assert np.array_equal(got.cpu().numpy(), ref.select(c, b, q64, 5, 1, 2))
    check_attend(d.attend(db, q, blocks=got, lse=lse), lse,
                 *ref.attend(c, b, q64, 64 ** -0.5, got.cpu().numpy()))


def test_a_filter_without_words_hides_everything(ctx):
    b = ref.Batch(32, [70, 40], [1, 3], seed=5)
    c = ref.Cache(b.pages, 1, 32, 64, "bf16", seed=1)
    ref.fill(c, b, seed=2)
    q, _ = rows(np.random.default_rng(3), b.queries, 2, 64, "bf16")
    d, db = device_cache(ctx, c), with_filter(b, torch.empty((2, 0), dtype=torch.int32, device="cuda"))
    lse = torch.zeros((b.queries, 2), device="cuda")
    assert (d.attend(db, q, lse=lse) == 0).all() and torch.isneginf(lse).all()
    assert (d.select(db, q, 4) == -1).all()


# ---- sequences longer than their page table ------------------------------------

def cut(b: ref.Batch, width: int):
    """The batch with page tables of only `width` blocks."""
    b.table, b.width = np.ascontiguousarray(b.table[:, :width]), width
    return b


PAST = [
    # elem, dim, page, kv heads, group, lengths, new, table width
    ("bf16", 128, 64, 2, 4, [129, 200, 128], [1, 1, 1], 2),
    ("f16", 64, 32, 1, 3, [70, 100, 33], [9, 40, 2], 2),
    ("bf16", 256, 32, 1, 2, [90, 65], [30, 1], 2),
    ("bf16", 64, 64, 1, 1, [40, 3], [1, 3], 0),
]


@pytest.mark.parametrize("elem,dim,page,heads,group,lens,new,width", PAST)
def test_positions_past_the_page_table_are_holes(ctx, elem, dim, page, heads, group, lens, new, width):
    """Tokens there are written nowhere, and those that have a page keep their positions."""
    b = ref.Batch(page, lens, new, seed=dim)
    cut(b, width)
    c = ref.Cache(b.pages, heads, page, dim, elem, seed=1)
    old = ref.Batch(page, [min(n - m, width * page) for n, m in zip(lens, new)], [0] * len(new), pages=b.pages)
    old.table, old.width = b.table, width
    ref.fill(c, old, seed=2)
    r = np.random.default_rng(3)
    k, k64 = rows(r, b.queries, heads, dim, elem)
    v, v64 = rows(r, b.queries, heads, dim, elem)
    q, q64 = rows(r, b.queries, heads * group, dim, elem)
    d, db = device_cache(ctx, c), device_batch(b)
    kh = torch.full_like(k, 7.0)
    d.append(db, k, v, k_held=kh)
    touched = set()
    want = np.full(k64.shape, 7.0)
    for row, s, pos in b.tokens():
        if pos // page < width:
            want[row] = c.write(b.table[s, pos // page], pos % page, k64[row], v64[row])[0]
            touched.add((s, pos // page))
    for s, j in touched:
        c.renew_box(b.table[s, j], min(page, lens[s] - j * page))
    torch.cuda.synchronize()
    for name in c.NAMES:
        assert np.array_equal(getattr(d, name).cpu().numpy(), getattr(c, name)), name
    assert np.array_equal(kh.double().cpu().numpy(), want)
    lse = torch.empty((b.queries, heads * group), device="cuda")
    check_attend(d.attend(db, q, lse=lse), lse, *ref.attend(c, b, q64, dim ** -0.5))
    for n, first, last in ((1, 0, 1), (3, 1, 2)):
        got = d.select(db, q, n, first=first, last=last)
        assert np.array_equal(got.cpu().numpy(), ref.select(c, b, q64, n, first, last))
    check_attend(d.attend(db, q, blocks=got, lse=lse), lse,
                 *ref.attend(c, b, q64, dim ** -0.5, got.cpu().numpy()))


def test_a_token_past_the_table_leaves_the_cache_as_it_was(ctx):
    """Position 128 of a sequence with two pages of 64: position 127 keeps its key."""
    b = ref.Batch(64, [129], [1], seed=1)
    c = ref.Cache(b.pages, 2, 64, 128, "bf16", seed=1)
    ref.fill(c, b)
    cut(b, 2)
    d = device_cache(ctx, c)
    k, _ = rows(np.random.default_rng(2), 1, 2, 128, "bf16")
    d.append(device_batch(b), k, k)
    d.append(device_batch(b, one_token=True), k, k)
    torch.cuda.synchronize()
    for name in c.NAMES:
        assert np.array_equal(getattr(d, name).cpu().numpy(), getattr(c, name)), name


# ---- batches of very unequal chunks -------------------------------------------

MANY = [
    # elem, dim, page, kv heads, group, new tokens of the sequences, lengths beside them
    ("bf16", 128, 64, 2, 4, [1] * 9 + [70] + [0, 1, 3] + [1] * 8, 300),
    ("f16", 64, 32, 1, 7, [0, 0, 41] + [1] * 70 + [0], 90),
    ("bf16", 256, 64, 1, 3, [2] * 6 + [90] + [1] * 6, 200),
]


@pytest.mark.parametrize("elem,dim,page,heads,group,new,most", MANY)
@pytest.mark.parametrize("filtered", [False, True])
def test_a_chunk_beside_many_short_sequences(ctx, elem, dim, page, heads, group, new, most, filtered):
    """Few row tiles of many sequences: whole, listed and split under a far bound."""
    r = np.random.default_rng(4)
    lens = [n + int(r.integers(0, most)) for n in new]
    b = ref.Batch(page, lens, new, seed=dim, visible=(lambda s, n, g: g.random(n) < 0.6) if filtered else None)
    c = ref.Cache(b.pages, heads, page, dim, elem, seed=1)
    ref.fill(c, b, seed=2)
    q, q64 = rows(r, b.queries, heads * group, dim, elem)
    d = device_cache(ctx, c)
    lse = torch.full((b.queries, heads * group), 7.0, device="cuda")
    want = ref.attend(c, b, q64, dim ** -0.5)
    for bound in (max(lens), 1 << 21):
        check_attend(d.attend(device_batch(b, max_length=bound), q, lse=lse), lse, *want)
    blocks = d.select(device_batch(b), q, 4)
    check_attend(d.attend(device_batch(b), q, blocks=blocks, lse=lse), lse,
                 *ref.attend(c, b, q64, dim ** -0.5, blocks.cpu().numpy()))


def test_more_row_tiles_than_one_axis_of_a_grid(ctx):
    """65,000 sequences of one token beside one of 200."""
    from gofann_amd import kvcache
    n = 65_000
    d = kvcache.KvCache.empty(ctx, pages=300, kv_heads=1, dim=64, page=32)
    r = np.random.default_rng(1)
    for t in (d.k_codes, d.v_codes):
        t.random_(0, 256)
    for t in (d.k_scales, d.v_scales):
        t.random_(124, 128)
    new = np.ones(n + 1, np.int64)
    new[40_000] = 200
    lens = np.where(new == 1, r.integers(1, 65, n + 1), 256)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()  # noqa: E731
    table = r.integers(0, 300, (n + 1, 8))
    off = np.concatenate(([0], np.cumsum(new)))
    q, _ = rows(r, int(off[-1]), 1, 64, "bf16")
    lse = torch.full((int(off[-1]), 1), 1e9, device="cuda")
    out = d.attend(kvcache.KvBatch(dev(table), dev(lens), dev(off), queries=int(off[-1]), max_queries=200,
                                   max_length=256), q, lse=lse)
    # every token as a sequence of its own, no more than a launch takes at once
    seq = np.repeat(np.arange(n + 1), new)
    pos = lens[seq] - new[seq] + np.arange(int(off[-1])) - off[seq]
    for i in range(0, int(off[-1]), 40_000):
        j = min(i + 40_000, int(off[-1]))
        one = kvcache.KvBatch(dev(table[seq[i:j]]), dev(pos[i:j] + 1), max_length=256)
        each = torch.empty((j - i, 1), device="cuda")
        want = d.attend(one, q[i:j], lse=each)
        # one bf16 rounding of the weights and one of the result in each
        assert ((out[i:j].float() - want.float()).abs() <= 4 * 2.0 ** -8 * 12).all()
        assert (out[i:j].float() - want.float()).abs().mean() < 1e-2
        assert ((lse[i:j] - each).abs() <= 1e-4).all()


def test_row_tiles_of_rows_the_batch_does_not_have(ctx):
    """Offsets that leave rows out, before the first sequence and past the last."""
    from gofann_amd import kvcache
    new = [0, 1, 40, 1, 1, 1, 1, 1, 1, 1, 1, 1]
    b = ref.Batch(32, [n + 20 for n in new], new, seed=1)
    c = ref.Cache(b.pages, 1, 32, 64, "bf16", seed=1)
    ref.fill(c, b, seed=2)
    q, q64 = rows(np.random.default_rng(3), b.queries, 2, 64, "bf16")
    want = ref.attend(c, b, q64, 64 ** -0.5)
    big = torch.zeros((b.queries + 8, 2, 64), dtype=torch.bfloat16, device="cuda")
    big[3:3 + b.queries] = q
    db = kvcache.KvBatch(torch.from_numpy(b.table).cuda(), torch.tensor(b.lens, dtype=torch.int32, device="cuda"),
                         torch.from_numpy(b.offsets + 3).cuda(), queries=b.queries + 8, max_queries=40,
                         max_length=1 << 16)
    out = torch.full_like(big, 99.0)
    device_cache(ctx, c).attend(db, big, out=out)
    check_attend(out[3:3 + b.queries], None, want[0], None, want[2])
    assert (out[:3] == 99.0).all() and (out[3 + b.queries:] == 99.0).all()


def test_a_refused_step_of_the_example_is_as_if_never_made(ctx):
    from gofann_amd import _lib, longcontext
    r = np.random.default_rng(6)
    a, b = (longcontext.Session(ctx, sequences=2, capacity=200, kv_heads=2, dim=64, page=32) for _ in range(2))
    for tokens, width in ((70, 0), (9, 4), (1, 4)):
        q, k, v = (rows(r, 2 * tokens, h, 64, "bf16")[0] for h in (8, 2, 2))
        with pytest.raises(_lib.GofannError, match="width"):
            a.step(q + 1, k + 1, v + 1, 2)  # refused by the choice, once its tokens are written
        assert torch.equal(a.step(q, k, v, width), b.step(q, k, v, width))
        assert torch.equal(a.lengths, b.lengths)


# ---- scores of large magnitude -------------------------------------------------

@pytest.mark.parametrize("elem,dim,up", [("bf16", 64, 55), ("bf16", 256, 18), ("bf16", 64, 13), ("bf16", 128, 9),
                                         ("f16", 256, 13), ("f16", 64, 12), ("f16", 128, 8)])
@pytest.mark.parametrize("heads,group,new", [(1, 3, 1), (1, 3, 9), (8, 4, 1024)])
@pytest.mark.parametrize("sign,at", [(1, [10]), (1, [700]), (-1, [700]), (1, [31, 300])])
def test_attend_of_scores_far_past_the_others_is_a_choice(ctx, elem, dim, up, heads, group, new, sign, at):
    """Scores of up to 2^118, whose distance is infinite next to a weight's range:
    the highest position's values are the result, or the mean of two.  sign < 0:
    every score is as large, and negative."""
    n = 900 + new
    b = ref.Batch(64, [n], [new], seed=3)
    c = ref.Cache(b.pages, heads, 64, dim, elem)
    r = np.random.default_rng(5)
    c.k_scales[:], c.v_scales[:] = 127 + up, 127
    c.k_codes[:] = 0x77 if sign < 0 else 0                      # 6 or 0 in all channels
    c.v_codes[:] = r.integers(0, 256, c.v_codes.shape)
    for t in at:
        c.k_codes[b.table[0, t // 64], :, t % 64] = 0x66 if sign < 0 else 0x77   # 4 or 6
    v = np.mean([c.read(b.table[0, t // 64], t % 64)[1] for t in at], 0)
    mass = np.mean([np.abs(c.read(b.table[0, t // 64], t % 64)[1]) for t in at], 0)
    d, db = device_cache(ctx, c), device_batch(b)
    for x in (1.125, 1.359375, 1.734375, 1.984375):             # exact in both types
        q = torch.full((new, heads * group, dim), sign * x * 2.0 ** up, device="cuda").to(d.dtype)
        lse = torch.empty(new, heads * group, device="cuda")
        got = d.attend(db, q, lse=lse).double().cpu().numpy().reshape(new, heads, group, dim)
        u = ref.UNIT[elem]
        bound = 1.02 * u * (mass + np.abs(v)) + 2.0 ** -25
        assert (np.abs(got - v[None, :, None]) <= bound[None, :, None]).all(), x
        top = sign * (4 if sign < 0 else 6) * x * 4.0 ** up * dim ** 0.5 + np.log(len(at))
        # products and their sum exact, then four roundings in 32 bits
        assert (np.abs(lse.double().cpu().numpy() - top) <= 4 * 2.0 ** -23 * abs(top)).all()


# ---- long chunks ----------------------------------------------------------------

def sampled(b: ref.Batch, pick):
    """One-token sequences that are the picked rows of a batch."""
    tok = {row: (s, p) for row, s, p in b.tokens()}
    sub = ref.Batch(b.page, [max(0, tok[i][1] + 1) for i in pick], [1] * len(pick), pages=b.pages)
    sub.table = np.stack([b.table[tok[i][0]] for i in pick])
    sub.width, sub.visible = b.width, b.visible
    if b.visible is not None:
        sub.bits = np.stack([b.bits[tok[i][0]] for i in pick])
    return sub


def random_codes(c: ref.Cache, r):
    """Every position of the cache written."""
    for name in ("k_codes", "v_codes"):
        getattr(c, name)[:] = r.integers(0, 256, getattr(c, name).shape)
    for name in ("k_scales", "v_scales"):
        getattr(c, name)[:] = r.integers(124, 128, getattr(c, name).shape)


def garbage_where_nothing_is_seen(c: ref.Cache, b: ref.Batch):
    """Exponents of infinity and NaN at the positions that the filter hides."""
    for s, n in enumerate(b.lens):
        for t in range(n):
            pid = b.page_of(s, t // b.page)
            if pid >= 0 and not b.sees(s, t):
                c.k_scales[pid, :, t % b.page] = 255
                c.v_scales[pid, :, t % b.page // 8, :, t % 8] = 254


LONG = [
    # elem, dim, page, kv heads, group, lengths, new, filter, holes
    ("bf16", 128, 64, 8, 4, [1300, 500], [700, 400], documents, 0.0),
    ("bf16", 128, 32, 8, 3, [1300, 500], [1100, 400], None, 0.3),
    ("f16", 64, 256, 8, 5, [900, 300], [700, 300], documents, 0.2),
    ("f16", 256, 64, 8, 4, [1150], [1100], lambda s, n, r: r.random(n) < 0.5, 0.1),
    ("bf16", 256, 128, 8, 4, [1000, 200], [900, 200], documents, 0.0),
    ("bf16", 64, 32, 2, 20, [700, 100], [800, 100], None, 0.0),     # tokens before position 0
    ("f16", 128, 64, 8, 4, [1100], [1100], lambda s, n, r: np.zeros(n, bool), 0.0),
]


@pytest.mark.parametrize("elem,dim,page,heads,group,lens,new,filt,holes", LONG)
def test_long_chunks_under_filters_and_holes(ctx, elem, dim, page, heads, group, lens, new, filt, holes):
    assert sum(new) * group // 128 * heads >= 256, "not the kernel of long chunks"
    b = ref.Batch(page, lens, new, seed=dim, holes=holes, visible=filt)
    c = ref.Cache(b.pages, heads, page, dim, elem, seed=1)
    r = np.random.default_rng(4)
    random_codes(c, r)
    garbage_where_nothing_is_seen(c, b)
    q, _ = rows(r, b.queries, heads * group, dim, elem)
    d, db = device_cache(ctx, c), device_batch(b)
    lse = torch.full((b.queries, heads * group), 1e9, device="cuda")
    out = d.attend(db, q, lse=lse)
    assert torch.isfinite(out).all() and (lse < 1e8).all()
    first = new[0]
    pick = sorted({0, 1, 31, 32, 127, 300, first // 2, first - 1, first % b.queries, b.queries - 2, b.queries - 1})
    want = ref.attend(c, sampled(b, pick), q[pick].double().cpu().numpy(), dim ** -0.5)
    tok = {row: p for row, s, p in b.tokens()}
    empty = [i for i, row in enumerate(pick) if tok[row] < 0]
    for w, x in zip(want, (0.0, -np.inf, 0.0)):
        w[empty] = x
    check_attend(out[pick], lse[pick], *want)
    assert torch.equal(out, d.attend(db, q)), "two runs differ"
    odd = spread(torch.zeros_like(q))
    d.attend(db, spread(q), out=odd)
    assert torch.equal(out, odd), "strides change the result"
    swapped = torch.empty((heads * group, b.queries, dim), dtype=q.dtype, device="cuda").transpose(0, 1)
    d.attend(db, q.transpose(0, 1).contiguous().transpose(0, 1), out=swapped)
    assert torch.equal(out, swapped), "the order of tokens and heads changes the result"


@pytest.mark.parametrize("elem,dim,group,edge", [("bf16", 128, 4, [16, 17, 31, 32, 33]), ("f16", 64, 1, [63, 64, 65, 127, 128, 129])])
def test_sequences_of_about_the_rows_that_long_chunks_leave(ctx, elem, dim, group, edge):
    """64 rows and fewer go to the other kernel, 65 and more do not."""
    heads, page = 8, 64
    new = [4200 // group * 2] + edge + [1]
    lens = [new[0]] + [n + 150 for n in edge] + [200]
    assert sum(new) * group // 128 * heads >= 256
    b = ref.Batch(page, lens, new, seed=2)
    c = ref.Cache(b.pages, heads, page, dim, elem, seed=1)
    r = np.random.default_rng(4)
    random_codes(c, r)
    q, _ = rows(r, b.queries, heads * group, dim, elem)
    lse = torch.full((b.queries, heads * group), 1e9, device="cuda")
    out = torch.full_like(q, 99.0)
    device_cache(ctx, c).attend(device_batch(b), q, out=out, lse=lse)
    assert (out != 99.0).any(-1).all() and (lse < 1e8).all()
    pick = [0] + [int(b.offsets[s]) + i for s in range(1, len(new)) for i in {0, new[s] // 2, new[s] - 1}]
    want = ref.attend(c, sampled(b, pick), q[pick].double().cpu().numpy(), dim ** -0.5)
    check_attend(out[pick], lse[pick], *want)
