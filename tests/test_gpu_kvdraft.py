"""Drafts, cross attention and reading back over the 4-bit key/value cache on the
GPU against their plain 64-bit definition (kv_draft_reference): bits, paths and
bytes equal, attention within the error that its roundings allow."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kv_draft_reference as draft
import kv_reference as ref
from test_gpu_kvcache import check_attend, device_batch, device_cache, documents, rows, spread

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(gpu_ctx):
    return gpu_ctx


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def same_arrays(d, c):
    torch.cuda.synchronize()
    for name in c.NAMES:
        assert np.array_equal(getattr(d, name).cpu().numpy(), getattr(c, name)), name


# ---- trees --------------------------------------------------------------------

NEW = [[1, 1, 1], [7, 0, 40], [31, 32, 33, 1, 64, 65], [300, 2, 257], [1000]]


@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("bad", [0.0, 0.2])
def test_tree_bits_and_depths(ctx, new, bad):
    from gofann_amd import kvcache
    b = ref.Batch(32, [n + 5 for n in new], new)
    p = draft.trees(new, seed=len(new), bad=bad)
    sees, depths = kvcache.draft_tree(ctx, device_batch(b), dev(p))
    want, want_depths = draft.tree(new, p)
    assert np.array_equal(sees.cpu().numpy(), draft.words(want))
    assert np.array_equal(depths.cpu().numpy(), want_depths)


def test_tree_that_is_one_long_chain(ctx):
    from gofann_amd import kvcache
    n = 8192
    b = ref.Batch(32, [n], [n])
    sees, depths = kvcache.draft_tree(ctx, device_batch(b), torch.arange(-1, n - 1, dtype=torch.int32).cuda())
    assert torch.equal(depths.cpu(), torch.arange(n, dtype=torch.int32))
    assert np.array_equal(sees.cpu().numpy(), draft.words(np.tril(np.ones((n, n), bool))))


@pytest.mark.parametrize("words", [0, 1, 2, 5])
def test_tree_words_that_are_too_few_or_too_many(ctx, words):
    new = [70, 3]
    b = ref.Batch(32, [80, 3], new)
    p = draft.trees(new, seed=2)
    db, parents = device_batch(b), dev(p)
    sees = torch.full((73, words + 1), 7, dtype=torch.int32, device="cuda")
    depths = torch.full((73,), 7, dtype=torch.int32, device="cuda")
    ctx.check(ctx.lib.gofann_kv_draft_tree(ctx.handle, db.view, parents.data_ptr(), words,
                                           sees.data_ptr(), depths.data_ptr()))
    want, want_depths = draft.tree(new, p)
    flat = sees.cpu().numpy().reshape(-1)
    assert np.array_equal(flat[:73 * words].reshape(73, words), draft.words(want, words))
    assert (flat[73 * words:] == 7).all()
    assert np.array_equal(depths.cpu().numpy(), want_depths)
    if words == 5:
        ctx.check(ctx.lib.gofann_kv_draft_tree(ctx.handle, db.view, parents.data_ptr(), 0, None,
                                               depths.data_ptr()))


@pytest.mark.parametrize("new", NEW + [[0, 5]])
@pytest.mark.parametrize("width,bad", [(1, 0.0), (4, 0.1), (70, 0.0)])
def test_accepted_paths(ctx, new, width, bad):
    from gofann_amd import kvcache
    lens = [n + 11 for n in new]
    lens[0] = new[0] // 2  # more tokens than positions
    b = ref.Batch(32, lens, new)
    n = b.queries
    r = np.random.default_rng(width)
    p = draft.trees(new, seed=width, bad=bad)
    drafted = r.integers(0, 4, n).astype(np.int32)
    chosen = r.integers(0, 5, n).astype(np.int32)
    at = 0
    for m in new:  # mostly a child's
        for i in range(m - 1, 0, -1):
            if 0 <= p[at + i] < i and r.random() < 0.8:
                chosen[at + p[at + i]] = drafted[at + i]
        at += m
    got = kvcache.draft_accept(ctx, device_batch(b), dev(p), dev(drafted), dev(chosen), width)
    for g, w, name in zip(got, draft.accept(lens, new, p, drafted, chosen, width), ("path", "lengths", "next")):
        assert np.array_equal(g.cpu().numpy(), w), name


def test_accepted_chain_past_64_tokens(ctx):
    """A path through every 64 tokens, and one whose child lies far behind it."""
    from gofann_amd import kvcache
    n = 200
    b = ref.Batch(32, [n, n], [n, n])
    chain = np.arange(-1, n - 1)
    jump = np.zeros(n, int)
    jump[0], jump[190], jump[199] = -1, 0, 190
    p = np.concatenate((chain, jump)).astype(np.int32)
    tok = np.concatenate((np.arange(n), np.full(n, 9))).astype(np.int32)
    tok[n + 190] = tok[n + 199] = 5
    ans = np.concatenate((np.arange(1, n + 1), np.full(n, 5))).astype(np.int32)
    path, lengths, answer = kvcache.draft_accept(ctx, device_batch(b), dev(p), dev(tok), dev(ans), 256)
    want = draft.accept([n, n], [n, n], p, tok, ans, 256)
    assert np.array_equal(path.cpu().numpy(), want[0]) and list(want[0][1][:3]) == [0, 190, 199]
    assert lengths.tolist() == [200, 3] and answer.tolist() == [200, 5]


# ---- attention of drafts --------------------------------------------------------

DRAFT = [
    # elem, dim, page, kv heads, group, lengths, new, filter, holes
    ("bf16", 128, 64, 2, 4, [1, 31, 32, 33, 64, 65], [1, 5, 32, 2, 7, 9], None, 0),
    ("f16", 128, 64, 2, 8, [0, 5, 300], [0, 5, 12], None, 0),
    ("bf16", 64, 32, 3, 1, [97, 40], [33, 40], None, 0),
    ("bf16", 256, 128, 1, 16, [260, 130], [20, 3], None, 0),
    ("f16", 64, 256, 1, 7, [500, 90], [60, 30], None, 0),
    ("bf16", 128, 32, 1, 20, [75, 10], [1, 10], None, 0),
    ("f16", 256, 64, 2, 3, [90, 64], [37, 1], None, 0),
    ("bf16", 128, 64, 1, 4, [1200, 333, 100], [64, 33, 100], None, 0),
    ("bf16", 64, 32, 1, 40, [70], [13], None, 0),
    ("f16", 128, 64, 2, 4, [300, 90, 900], [30, 11, 64], documents, 0),
    ("bf16", 128, 64, 1, 5, [300, 90, 200], [70, 2, 40], documents, 0),
    ("bf16", 64, 32, 2, 2, [300, 90, 200], [90, 2, 40], documents, 0.3),
    ("f16", 256, 32, 1, 2, [300, 90], [40, 41], None, 0.4),
    ("bf16", 128, 64, 1, 2, [3, 40], [7, 40], None, 0),  # more tokens than positions
    ("bf16", 128, 64, 2, 8, [700, 700, 64], [130, 1, 64], None, 0),
]


@pytest.mark.parametrize("elem,dim,page,heads,group,lens,new,filt,holes", DRAFT)
def test_attend_of_drafts(ctx, elem, dim, page, heads, group, lens, new, filt, holes):
    b = ref.Batch(page, lens, new, seed=dim + group, holes=holes, visible=filt)
    c = ref.Cache(b.pages, heads, page, dim, elem, seed=1)
    draft.scatter(c, seed=2)
    sees, _ = draft.tree(new, draft.trees(new, seed=3, bad=0.05))
    sees[::5] &= np.random.default_rng(4).random(sees[::5].shape) < 0.5  # any bits will do
    q, q64 = rows(np.random.default_rng(3), b.queries, heads * group, dim, elem)
    scale = 0.6 * dim ** -0.5
    want = draft.attend(c, b, q64, scale, sees)
    d, db, bits = device_cache(ctx, c), device_batch(b), dev(draft.words(sees))
    lse = torch.full((b.queries, heads * group), 7.0, device="cuda")
    out = d.attend(db, q, scale=scale, sees=bits, lse=lse)
    check_attend(out, lse, *want)
    assert torch.equal(out, d.attend(db, q, scale=scale, sees=bits)), "two runs differ"
    odd = spread(torch.zeros_like(q))
    wide = torch.full((b.queries, bits.shape[1] + 3), -1, dtype=torch.int32, device="cuda")
    wide[:, 1:-2] = bits
    d.attend(db, spread(q), scale=scale, sees=wide[:, 1:-2], out=odd)
    assert torch.equal(out, odd), "strides change the result"


def test_a_draft_that_is_a_chain_sees_what_a_causal_call_sees(ctx):
    b = ref.Batch(64, [400, 90], [50, 33])
    c = ref.Cache(b.pages, 2, 64, 128, "bf16", seed=1)
    draft.scatter(c, seed=2)
    q, q64 = rows(np.random.default_rng(3), b.queries, 8, 128, "bf16")
    sees = np.tril(np.ones((50, 50), bool))
    sees = np.concatenate((sees, sees[:33]))
    d, db = device_cache(ctx, c), device_batch(b)
    lse = torch.empty((83, 8), device="cuda")
    want = ref.attend(c, b, q64, 128 ** -0.5)
    check_attend(d.attend(db, q, sees=dev(draft.words(sees)), lse=lse), lse, *want)


@pytest.mark.parametrize("words", [0, 1, 2])
def test_draft_tokens_past_the_words_are_not_seen(ctx, words):
    b = ref.Batch(32, [130, 60], [70, 60])
    c = ref.Cache(b.pages, 1, 32, 64, "f16", seed=1)
    draft.scatter(c, seed=2)
    q, q64 = rows(np.random.default_rng(3), b.queries, 6, 64, "f16")
    sees = np.ones((130, 32 * words), bool)
    d = device_cache(ctx, c)
    lse = torch.empty((130, 6), device="cuda")
    out = d.attend(device_batch(b), q, sees=dev(draft.words(sees, words)), lse=lse)
    check_attend(out, lse, *draft.attend(c, b, q64, 64 ** -0.5, sees))
    if words == 0:  # the second sequence is nothing but its draft
        assert (out[70:] == 0).all() and torch.isneginf(lse[70:]).all()


@pytest.mark.parametrize("elem,dim", [("bf16", 64), ("f16", 128), ("bf16", 256)])
@pytest.mark.parametrize("new", [9, 100])
def test_unseen_draft_tokens_need_not_be_written(ctx, elem, dim, new):
    """A padded draft: its last tokens have no keys yet, whatever lies there."""
    b = ref.Batch(32, [300], [new], seed=1)
    c = ref.Cache(b.pages, 2, 32, dim, elem, seed=1)
    draft.scatter(c, seed=2)
    real = new - new // 3
    for t in range(300 - new + real, 300):
        pid, at = b.table[0, t // 32], t % 32
        c.k_codes[pid, :, at] = c.v_codes[pid, :, at // 8, :, at % 8] = 0x7F
        c.k_scales[pid, :, at] = c.v_scales[pid, :, at // 8, :, at % 8] = 255 if t % 2 else 254
    sees, _ = draft.tree([new], draft.trees([new], seed=3))
    sees[:, real:] = False
    q, q64 = rows(np.random.default_rng(3), new, 8, dim, elem)
    clean = ref.Cache(b.pages, 2, 32, dim, elem, seed=1)
    draft.scatter(clean, seed=2)
    d = device_cache(ctx, c)
    lse = torch.empty((new, 8), device="cuda")
    out = d.attend(device_batch(b), q, sees=dev(draft.words(sees)), lse=lse)
    check_attend(out, lse, *draft.attend(clean, b, q64, dim ** -0.5, sees))


@pytest.mark.parametrize("filt,holes", [(None, 0), (documents, 0.2)])
def test_attend_of_drafts_to_listed_blocks(ctx, filt, holes):
    b = ref.Batch(32, [700, 65, 300], [24, 3, 40], seed=2, visible=filt, holes=holes)
    c = ref.Cache(b.pages, 2, 32, 64, "bf16", seed=1)
    old = ref.Batch(32, b.lens, [0, 0, 0], pages=b.pages, seed=2)
    old.table = b.table
    ref.fill(c, old, seed=2)
    sees, _ = draft.tree(b.new, draft.trees(b.new, seed=3))
    q, q64 = rows(np.random.default_rng(3), b.queries, 6, 64, "bf16")
    d, db, bits = device_cache(ctx, c), device_batch(b), dev(draft.words(sees))
    lse = torch.empty((b.queries, 6), device="cuda")
    blocks = d.select(db, q, 6, first=1, last=3)
    got = d.attend(db, q, sees=bits, blocks=blocks, lse=lse)
    check_attend(got, lse, *draft.attend(c, b, q64, 64 ** -0.5, sees, blocks.cpu().numpy()))
    r = np.random.default_rng(5)
    lists = np.stack([r.permutation(np.concatenate((np.arange(b.width), [-1, b.width, 2 ** 30])))[:4]
                      for _ in range(b.queries * 2)]).reshape(b.queries, 2, 4).astype(np.int32)
    got = d.attend(db, q, sees=bits, blocks=dev(lists), lse=lse)
    check_attend(got, lse, *draft.attend(c, b, q64, 64 ** -0.5, sees, lists))


@pytest.mark.parametrize("elem,dim,group,new", [("bf16", 128, 8, 40), ("f16", 64, 1, 17), ("bf16", 256, 4, 30),
                                               ("f16", 128, 4, 100), ("bf16", 128, 1, 300)])
def test_drafts_behind_a_long_context(ctx, elem, dim, group, new):
    """Positions cut over many workgroups and joined, with a bound on the length that is far off."""
    b = ref.Batch(64, [9001, new + 3, 2000], [new, new, 1], seed=9)
    c = ref.Cache(b.pages, 1, 64, dim, elem, seed=1)
    draft.scatter(c, seed=2, low=124, high=126)
    sees, _ = draft.tree(b.new, draft.trees(b.new, seed=3))
    q, q64 = rows(np.random.default_rng(3), b.queries, group, dim, elem)
    want = draft.attend(c, b, q64, dim ** -0.5, sees)
    lse = torch.empty((b.queries, group), device="cuda")
    d, bits = device_cache(ctx, c), dev(draft.words(sees))
    for most in (9001, 2 ** 20):
        out = d.attend(device_batch(b, max_length=most), q, sees=bits, lse=lse)
        check_attend(out, lse, *want)


# ---- cross attention --------------------------------------------------------------

CROSS = [
    # elem, dim, page, kv heads, group, lengths, new, filter, holes
    ("bf16", 128, 64, 2, 4, [1, 31, 0, 33, 64, 65], [1, 1, 1, 1, 1, 1], None, 0),
    ("f16", 64, 64, 5, 1, [300, 7, 151], [1, 1, 1], None, 0),
    ("f16", 64, 32, 3, 1, [97, 0, 40], [200, 9, 1], None, 0),
    ("bf16", 256, 128, 1, 16, [260, 130], [20, 3], None, 0),
    ("f16", 64, 256, 1, 7, [500, 1], [60, 130], None, 0),
    ("bf16", 128, 32, 1, 20, [75, 10], [1, 64], None, 0),
    ("f16", 256, 64, 2, 3, [90, 64], [137, 1], None, 0),
    ("bf16", 128, 64, 1, 4, [1200, 333, 100], [164, 33, 0], None, 0),
    ("f16", 128, 64, 2, 4, [300, 90, 900], [30, 11, 64], documents, 0),
    ("bf16", 64, 32, 2, 2, [300, 90, 200], [90, 2, 140], documents, 0.3),
    ("bf16", 128, 32, 8, 2, [500], [777], None, 0),
    ("f16", 128, 64, 1, 1, [5000, 70], [1, 1], None, 0),
]


@pytest.mark.parametrize("elem,dim,page,heads,group,lens,new,filt,holes", CROSS)
def test_cross_attention(ctx, elem, dim, page, heads, group, lens, new, filt, holes):
    b = ref.Batch(page, lens, new, seed=dim + group, holes=holes, visible=filt)
    c = ref.Cache(b.pages, heads, page, dim, elem, seed=1)
    draft.scatter(c, seed=2)
    q, q64 = rows(np.random.default_rng(3), b.queries, heads * group, dim, elem)
    scale = 0.6 * dim ** -0.5
    want = draft.attend(c, b, q64, scale)
    d, db = device_cache(ctx, c), device_batch(b)
    lse = torch.full((b.queries, heads * group), 7.0, device="cuda")
    out = d.cross(db, q, scale=scale, lse=lse)
    check_attend(out, lse, *want)
    assert torch.equal(out, d.cross(db, q, scale=scale)), "two runs differ"
    odd = spread(torch.zeros_like(q))
    d.cross(db, spread(q), scale=scale, out=odd)
    assert torch.equal(out, odd), "strides change the result"
    if all(m == 1 for m in new):
        assert torch.equal(out, d.cross(device_batch(b, one_token=True), q, scale=scale))
    far = d.cross(device_batch(b, max_length=2 ** 18), q, scale=scale, lse=lse)
    check_attend(far, lse, *want)


def test_cross_of_rows_that_no_sequence_has_leaves_them(ctx):
    from gofann_amd import kvcache
    b = ref.Batch(32, [70, 40], [3, 40])
    c = ref.Cache(b.pages, 1, 32, 64, "bf16", seed=1)
    draft.scatter(c)
    q, _ = rows(np.random.default_rng(3), 60, 2, 64, "bf16")
    table, off = dev(b.table), dev(b.offsets + 5)
    db = kvcache.KvBatch(table, dev(np.array(b.lens, np.int32)), off, queries=60, max_queries=40, max_length=70)
    d = device_cache(ctx, c)
    out = torch.full_like(q, 99.0)
    d.cross(db, q, out=out)
    assert (out[:5] == 99.0).all() and (out[48:] == 99.0).all() and (out[5:48] != 99.0).any(-1).all()
    out = torch.full_like(q, 99.0)
    d.attend(db, q, sees=torch.full((60, 2), -1, dtype=torch.int32, device="cuda"), out=out)
    assert (out[:5] == 99.0).all() and (out[48:] == 99.0).all() and (out[5:48] != 99.0).any(-1).all()


# ---- far scores, small weights, strange queries ---------------------------------------

@pytest.mark.parametrize("new,group", [(1, 4), (40, 4)])
@pytest.mark.parametrize("how", ["cross", "draft"])
def test_scores_far_apart(ctx, how, new, group):
    """A maximum that grows along the sequence, scores that underflow against it, and scaled
    scores past 2^22, where a score's own rounding is more than its weight."""
    b = ref.Batch(64, [640], [new], seed=1)
    c = ref.Cache(b.pages, 1, 64, 128, "bf16", seed=1)
    r = np.random.default_rng(2)
    for t in range(640):
        k = r.standard_normal((1, 128)) * 0.1
        k[0, 0] = t / 8.0 if t % 97 else -300.0
        c.write(b.table[0, t // 64], t % 64, k, r.standard_normal((1, 128)))
    q = torch.zeros(new, 4, 128, dtype=torch.bfloat16)
    q[:, 0, 0], q[:, 1, 0], q[:, 2, 1], q[:, 3, 0] = 30.0, -30.0, 1.0, 0.001
    sees = None if how == "cross" else np.ones((new, new), bool)
    want = draft.attend(c, b, q.double().numpy(), 1.0, sees)
    lse = torch.empty((new, 4), device="cuda")
    d, db = device_cache(ctx, c), device_batch(b)
    call = (lambda **kw: d.cross(db, q.cuda(), **kw)) if how == "cross" else \
        (lambda **kw: d.attend(db, q.cuda(), sees=dev(draft.words(sees)), **kw))
    check_attend(call(scale=1.0, lse=lse), lse, *want)
    # every score a multiple of 2^24: the largest one's positions alone have weight
    q[:] = 0
    q[:, :, 0] = 1.0
    out = call(scale=2.0 ** 24).double().cpu().numpy()
    k, v, _ = draft.dense(c, b, 0, 640)
    best = k[:, 0, 0] == k[:, 0, 0].max()
    mean = v[best, 0].mean(0)
    assert np.abs(out - mean).max() <= 2.0 ** -8 * (np.abs(v[best, 0]).max() + np.abs(mean).max())


@pytest.mark.parametrize("new", [2, 50])
def test_infinite_and_nan_queries_stay_in_their_rows(ctx, new):
    b = ref.Batch(64, [300], [new], seed=1)
    c = ref.Cache(b.pages, 1, 64, 128, "bf16", seed=1)
    draft.scatter(c)
    q, _ = rows(np.random.default_rng(2), new, 4, 128, "bf16")
    d, db = device_cache(ctx, c), device_batch(b)
    bits = torch.full((new, 2), -1, dtype=torch.int32, device="cuda")
    calls = (lambda: d.cross(db, q), lambda: d.attend(db, q, sees=bits))
    clean = [f() for f in calls]
    q[0, 1, 5] = float("nan")
    q[1, 2, 7] = float("inf")
    bad = torch.zeros(new, 4, dtype=torch.bool, device="cuda")
    bad[0, 1] = bad[1, 2] = True
    for f, was in zip(calls, clean):
        out = f()
        assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], was[~bad])


# ---- reading back ---------------------------------------------------------------------

READ = [
    ("bf16", 128, 64, 2, [1, 64, 65, 200], [1, 1, 1, 200], 0),
    ("f16", 128, 64, 3, [130, 7, 64], [130, 3, 0], 0),
    ("bf16", 64, 32, 1, [33, 70, 5], [2, 40, 9], 0.3),  # the last: more tokens than positions
    ("f16", 256, 128, 2, [129, 300], [2, 131], 0),
    ("bf16", 256, 256, 1, [257, 90], [17, 90], 0.4),
    ("f16", 64, 64, 2, [63, 1, 100], [1, 1, 100], 0),
]


@pytest.mark.parametrize("elem,dim,page,heads,lens,new,holes", READ)
def test_read(ctx, elem, dim, page, heads, lens, new, holes):
    b = ref.Batch(page, lens, new, seed=dim, holes=holes)
    c = ref.Cache(b.pages, heads, page, dim, elem, seed=1)
    draft.scatter(c, seed=2, low=110, high=138)
    want_k, want_v = np.zeros((b.queries, heads, dim)), np.zeros((b.queries, heads, dim))
    for row, s, pos in b.tokens():
        pid = b.page_of(s, pos // page) if pos >= 0 else -1
        if pid >= 0:
            want_k[row], want_v[row] = c.read(pid, pos % page)
    d, db = device_cache(ctx, c), device_batch(b)
    k, v = d.read(db)
    assert np.array_equal(k.double().cpu().numpy(), want_k) and np.array_equal(v.double().cpu().numpy(), want_v)
    odd = spread(torch.full_like(k, 3.0))
    assert d.read(db, v=odd)[0] is None
    assert torch.equal(odd, v)
    kk, vv = spread(torch.full_like(k, 3.0)), spread(torch.full_like(k, 3.0))
    d.read(db, k=kk, v=vv)
    assert torch.equal(kk, k) and torch.equal(vv, v)
    same_arrays(d, c)


def test_read_past_the_table_and_the_bound_gives_zeros(ctx):
    b = ref.Batch(32, [200, 100], [200, 60])
    c = ref.Cache(b.pages, 1, 32, 64, "bf16", seed=1)
    draft.scatter(c)
    d = device_cache(ctx, c)
    whole = d.read(device_batch(b))
    part = d.read(device_batch(b, max_length=90))
    for x, y in zip(whole, part):
        assert torch.equal(x[:90], y[:90]) and (y[90:200] == 0).all()
        assert torch.equal(x[200:250], y[200:250]) and (y[250:] == 0).all()
    b.table, b.width = np.ascontiguousarray(b.table[:, :2]), 2
    for x, y in zip(whole, d.read(device_batch(b))):
        assert torch.equal(x[:64], y[:64]) and (y[64:200] == 0).all()


def test_read_gives_what_append_held(ctx):
    b = ref.Batch(64, [150, 20], [100, 20])
    c = ref.Cache(b.pages, 2, 64, 128, "bf16", seed=1)
    r = np.random.default_rng(3)
    k, v = rows(r, 120, 2, 128, "bf16")[0], rows(r, 120, 2, 128, "bf16", 5.0)[0]
    kh, vh = torch.empty_like(k), torch.empty_like(v)
    d, db = device_cache(ctx, c), device_batch(b)
    d.append(db, k, v, k_held=kh, v_held=vh)
    got = d.read(db)
    assert torch.equal(got[0], kh) and torch.equal(got[1], vh)


# ---- keeping a path ---------------------------------------------------------------------

KEEP = [
    # elem, dim, page, heads, lengths, new, holes
    ("bf16", 128, 64, 2, [70, 64, 65, 200, 9], [10, 1, 2, 64, 9], 0),
    ("f16", 64, 32, 3, [130, 7, 64, 40], [100, 3, 0, 33], 0),
    ("bf16", 256, 128, 1, [129, 300], [40, 131], 0),
    ("f16", 128, 32, 1, [400, 90, 33], [300, 50, 33], 0.3),
    ("bf16", 64, 256, 1, [500, 3], [270, 7], 0),  # the last: more tokens than positions
]


@pytest.mark.parametrize("elem,dim,page,heads,lens,new,holes", KEEP)
@pytest.mark.parametrize("boxes", [True, False])
def test_keep(ctx, elem, dim, page, heads, lens, new, holes, boxes):
    from gofann_amd import kvcache
    b = ref.Batch(page, lens, new, seed=dim, holes=holes)
    r = np.random.default_rng(5)
    for width, share in ((5, 0.3), (16, 0.9), (300, 0.7), (300, 1.0)):
        c = ref.Cache(b.pages, heads, page, dim, elem, seed=1)
        draft.scatter(c, seed=width, low=118, high=132)
        path = np.full((len(new), width), -1, np.int32)
        for s, n in enumerate(new):
            some = np.nonzero(r.random(n) < share)[0][:width]
            path[s, :len(some)] = some
        d = device_cache(ctx, c)
        if not boxes:
            d = kvcache.KvCache(ctx, d.k_codes, d.k_scales, d.v_codes, d.v_scales, dtype=d.dtype)
        d.keep(device_batch(b), dev(path))
        torch.cuda.synchronize()
        draft.keep(c, b, path)
        for name in c.NAMES[:6 if boxes else 4]:
            assert np.array_equal(getattr(d, name).cpu().numpy(), getattr(c, name)), name


def test_keep_of_paths_that_end_early(ctx):
    """A path ends where it no longer ascends within the draft; nothing past that is moved."""
    paths = [[-1, 2, 3, 4, 5, 6], [3, 2, 4, 5, 6, 7], [0, 0, 1, 2, 3, 4], [1, 5, 40, 41, 42, 43],
             [2 ** 31 - 1, 1, 2, 3, 4, 5], [2, 7, -2 ** 31, 8, 9, 10], [0, 1, 2, 3, 4, 5], [9, 10, 11, 12, 13, 14]]
    b = ref.Batch(32, [40 + 9 * i for i in range(8)], [12] * 8)
    c = ref.Cache(b.pages, 2, 32, 64, "bf16", seed=1)
    draft.scatter(c)
    d = device_cache(ctx, c)
    path = np.array(paths, np.int32)
    d.keep(device_batch(b), dev(path))
    draft.keep(c, b, path)
    same_arrays(d, c)
    d.keep(device_batch(b), dev(path[:, :0]))  # nothing kept: only the boxes
    draft.keep(c, b, path[:, :0])
    same_arrays(d, c)


# ---- together ------------------------------------------------------------------------

@pytest.mark.parametrize("elem,dim,page,group", [("bf16", 128, 64, 4), ("f16", 64, 32, 3)])
def test_drafts_settle_into_what_their_tokens_alone_would_have_left(ctx, elem, dim, page, group):
    """Steps of drafts, each attended, accepted and kept, beside a cache that is given only the
    accepted tokens, in order: the same lengths, bytes, boxes and, of the next step's tokens, the
    same outputs of what a tree's path sees."""
    from gofann_amd import kvcache
    heads, seqs, cap = 2, 3, 400
    r = np.random.default_rng(8)
    width = -(-cap // page)
    table = np.arange(seqs * width, dtype=np.int32).reshape(seqs, width)
    one = ref.Cache(seqs * width, heads, page, dim, elem, seed=1)
    plain = device_cache(ctx, one)
    drafts = device_cache(ctx, one)
    t = dev(table)
    lengths = dev(np.zeros(seqs, np.int32))
    have = np.zeros(seqs, int)

    def batch(lens, off):
        return kvcache.KvBatch(t, lens, dev(np.array(off, np.int32)), queries=int(off[-1]),
                               max_queries=int(np.diff(off).max()), max_length=cap)

    for step in range(9):
        new = r.integers(1, 30, seqs)
        if step == 0:
            new[:] = [70, 33, 1]  # the prompts: chains that are accepted whole
        off = np.concatenate(([0], np.cumsum(new)))
        n = int(off[-1])
        parents = np.concatenate([np.arange(-1, m - 1) for m in new]) if step == 0 else draft.trees(list(new), seed=step)
        parents = parents.astype(np.int32)
        tok = r.integers(0, 3, n).astype(np.int32)
        ans = r.integers(0, 3, n).astype(np.int32)
        if step == 0:
            tok[:] = ans[:] = 1
        k, v, q = (rows(r, n, h, dim, elem)[0] for h in (heads, heads, heads * group))
        lengths += dev(new.astype(np.int32))
        db = batch(lengths, off)
        p = dev(parents)
        sees, depths = kvcache.draft_tree(ctx, db, p)
        drafts.append(db, k, v)
        out = drafts.attend(db, q, sees=sees)
        path, left, answer = kvcache.draft_accept(ctx, db, p, dev(tok), dev(ans), 80 if step == 0 else 6)
        drafts.keep(db, path)
        want = draft.accept(list(have + new), list(new), parents, tok, ans, 80 if step == 0 else 6)
        assert np.array_equal(path.cpu().numpy(), want[0]) and np.array_equal(left.cpu().numpy(), want[1])
        lengths.copy_(left)
        # the accepted ones alone, and their outputs in a causal call
        pick = [off[s] + i for s in range(seqs) for i in want[0][s] if i >= 0]
        count = (want[0] >= 0).sum(1)
        rows_of = torch.tensor(pick, device="cuda")
        only = batch(lengths, np.concatenate(([0], np.cumsum(count))))
        plain.append(only, k[rows_of].contiguous(), v[rows_of].contiguous())
        same = plain.attend(only, q[rows_of].contiguous())
        # both are within half a step of the sums, and those of the rounded weights
        tol = 6 * ref.UNIT[elem] * 6.0
        assert (same.double() - out[rows_of].double()).abs().max().item() <= tol
        have += count
        a, b_ = plain.read(batch(lengths, np.concatenate(([0], np.cumsum(have))))), \
            drafts.read(batch(lengths, np.concatenate(([0], np.cumsum(have)))))
        assert torch.equal(a[0], b_[0]) and torch.equal(a[1], b_[1])
        for s in range(seqs):
            for j in range(-(-int(have[s]) // page)):
                pid = table[s, j]
                assert torch.equal(plain.box[pid], drafts.box[pid]) and \
                    torch.equal(plain.box_scale[pid], drafts.box_scale[pid]), (step, s, j)
        assert depths.max().item() < new.max()


def _draft_world(ctx, new=(20, 7, 1)):
    lens = [700, 130, 1]
    b = ref.Batch(64, lens, list(new), seed=1)
    c = ref.Cache(b.pages, 2, 64, 128, "bf16", seed=1)
    draft.scatter(c)
    r = np.random.default_rng(1)
    k, v, q = (rows(r, b.queries, h, 128, "bf16")[0] for h in (2, 2, 8))
    p = draft.trees(b.new, seed=1)
    ints = [dev(x) for x in (p, r.integers(0, 2, b.queries).astype(np.int32),
                             r.integers(0, 2, b.queries).astype(np.int32))]
    return device_cache(ctx, c), device_batch(b), (k, v, q), ints


def test_graph_replays_equal_eager_drafts(gpu_ctx):
    """A whole step captured once, new inputs at each replay, eager work between them."""
    from gofann_amd import _lib, kvcache
    own = _lib.Context(0)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        own.bind_stream(side)
        d, db, (k, v, q), (parents, drafted, chosen) = _draft_world(own)

        def step():
            sees, depths = kvcache.draft_tree(own, db, parents)
            d.append(db, k, v)
            out = d.attend(db, q, sees=sees)
            every = d.cross(db, q)
            path, lengths, answer = kvcache.draft_accept(own, db, parents, drafted, chosen, 6)
            d.keep(db, path)
            kk, vv = d.read(db)
            return [sees, depths, out, every, path, lengths, answer, kk, vv, d.k_codes, d.v_codes, d.box]

        step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
        r = np.random.default_rng(11)
        for i in range(4):
            for t in (k, v, q):
                t.copy_(rows(r, *t.shape, "bf16")[0])
            parents.copy_(dev(draft.trees([20, 7, 1], seed=20 + i)))
            chosen.copy_(dev(r.integers(0, 2, 28).astype(np.int32)))
            graph.replay()
            side.synchronize()
            seen = [t.clone() for t in held]
            for a, e in zip(seen, step()):
                assert torch.equal(a, e)
            side.synchronize()
    own.close()


def test_calls_on_another_stream(gpu_ctx):
    from gofann_amd import _lib, kvcache
    own = _lib.Context(0)
    d, db, (k, v, q), (parents, drafted, chosen) = _draft_world(own)
    sees, _ = kvcache.draft_tree(own, db, parents)
    path, _, _ = kvcache.draft_accept(own, db, parents, drafted, chosen, 4)
    want = d.attend(db, q, sees=sees), d.cross(db, q), *d.read(db)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for call in (lambda: d.attend(db, q, sees=sees), lambda: d.cross(db, q), lambda: d.read(db),
                     lambda: d.keep(db, path), lambda: kvcache.draft_tree(own, db, parents),
                     lambda: kvcache.draft_accept(own, db, parents, drafted, chosen, 4)):
            with pytest.raises(_lib.GofannError, match="stream"):
                call()
        own.bind_stream(side)
        got = d.attend(db, q, sees=sees), d.cross(db, q), *d.read(db)
        side.synchronize()
    for a, e in zip(got, want):
        assert torch.equal(a, e)
    own.close()


def test_drafts_in_a_cache_past_four_gigabytes(ctx):
    from gofann_amd import kvcache
    d = kvcache.KvCache.empty(ctx, pages=150_000, kv_heads=8, dim=128)
    assert d.k_codes.numel() > 2 ** 32
    b = ref.Batch(64, [100], [40], pages=4, seed=1)
    c = ref.Cache(4, 8, 64, 128, "bf16")
    draft.scatter(c, seed=2)
    table = torch.from_numpy(np.where(b.table >= 0, b.table + 150_000 - 4, b.table)).cuda()
    for name in c.NAMES:
        getattr(d, name)[150_000 - 4:] = dev(getattr(c, name))
    db = device_batch(b)
    db._keep[0].copy_(table)
    q, q64 = rows(np.random.default_rng(3), 40, 16, 128, "bf16")
    sees, _ = draft.tree([40], draft.trees([40], seed=4))
    lse = torch.empty((40, 16), device="cuda")
    check_attend(d.attend(db, q, sees=dev(draft.words(sees)), lse=lse), lse,
                 *draft.attend(c, b, q64, 128 ** -0.5, sees))
    check_attend(d.cross(db, q, lse=lse), lse, *draft.attend(c, b, q64, 128 ** -0.5))
    k, v = d.read(db)
    small = device_cache(ctx, c).read(device_batch(b))
    assert torch.equal(k, small[0]) and torch.equal(v, small[1])
    path = np.array([[0, 3, 9, 30, 39, -1]], np.int32)
    d.keep(db, dev(path))
    draft.keep(c, b, path)
    torch.cuda.synchronize()
    for name in c.NAMES:
        assert np.array_equal(getattr(d, name)[150_000 - 4:].cpu().numpy(), getattr(c, name)), name


def test_session_with_drafts(ctx, capsys):
    """Drafts and steps of one token by turns, against what the cache then holds; refusals
    leave the sequences as they were."""
    from gofann_amd import longcontext
    r = np.random.default_rng(6)
    s = longcontext.Session(ctx, sequences=2, capacity=200, kv_heads=2, dim=64, page=32)
    c = ref.Cache(14, 2, 32, 64, "bf16")
    have = [40, 40]
    p0 = [rows(r, 80, h, 64, "bf16") for h in (8, 2, 2)]
    s.step(*(t for t, _ in p0))
    put = lambda b, pos, k, v: c.write(7 * b + pos // 32, pos % 32, k, v)  # noqa: E731
    for b in range(2):
        for i in range(40):
            put(b, i, p0[1][1][40 * b + i], p0[2][1][40 * b + i])
    for turn, n in enumerate((11, 1, 20, 7)):
        (q, q64), (k, k64), (v, v64) = (rows(r, 2 * n, h, 64, "bf16") for h in (8, 2, 2))
        p = draft.trees([n, n], seed=turn)
        tok, ans = (r.integers(0, 2, 2 * n).astype(np.int32) for _ in range(2))
        sees, _ = draft.tree([n, n], p)
        out = s.draft(q, k, v, dev(p))
        for b in range(2):
            for i in range(n):
                put(b, have[b] + i, k64[b * n + i], v64[b * n + i])
        b_ = ref.Batch(32, [h + n for h in have], [n, n], pages=14)
        b_.table, b_.width = np.arange(14, dtype=np.int32).reshape(2, 7), 7
        want = draft.attend(c, b_, q64, 64 ** -0.5, sees)
        check_attend(out, None, want[0], None, want[2])
        for bad in (lambda: s.draft(q, k, v, dev(p)), lambda: s.step(q, k, v), lambda: s.grow(1)):
            with pytest.raises(ValueError, match="settled"):
                bad()
        path, answer = s.settle(dev(tok), dev(ans), 4)
        want = draft.accept(b_.lens, [n, n], p, tok, ans, 4)
        assert np.array_equal(path.cpu().numpy(), want[0]) and np.array_equal(answer.cpu().numpy(), want[2])
        draft.keep(c, b_, want[0])
        have = list(want[1])
        assert s.lengths.tolist() == have and s.filled >= max(have)
        (q, q64), (k, k64), (v, v64) = (rows(r, 2, h, 64, "bf16") for h in (8, 2, 2))
        out = s.step(q, k, v)
        for b in range(2):
            put(b, have[b], k64[b], v64[b])
        have = [h + 1 for h in have]
        b_ = ref.Batch(32, have, [1, 1], pages=14)
        b_.table, b_.width = np.arange(14, dtype=np.int32).reshape(2, 7), 7
        want = ref.attend(c, b_, q64, 64 ** -0.5)
        check_attend(out, None, want[0], None, want[2])
    with pytest.raises(ValueError, match="no draft"):
        s.settle(dev(tok), dev(ans), 4)
    bound, lens = s.filled, s.lengths.tolist()
    with pytest.raises(ValueError):
        s.draft(q, k, v[:1], torch.full((2,), -1, dtype=torch.int32, device="cuda"))
    assert s.filled == bound and s.lengths.tolist() == lens and s.pending is None
    longcontext.main(["--context", "1500", "--steps", "2", "--sequences", "2", "--width", "8", "--draft", "13"])
    assert "13 drafted tokens" in capsys.readouterr().out
