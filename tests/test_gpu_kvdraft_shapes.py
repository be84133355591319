"""Drafts and cross attention over the 4-bit key/value cache at the sizes that its
kernels divide their work by: row tiles of 16, 32 and 128, tiles shared out over
sequences of very unequal lengths, lists of what a filter leaves, many sequences,
chunks that fill the chip.  Against 64-bit attention over what the cache holds."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kv_draft_reference as draft
import kv_reference as ref
from test_gpu_kvcache import TYPES

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(gpu_ctx):
    return gpu_ctx


class World:
    """A cache of random codes under sequences of given lengths and tokens, in pages of
    random order; a filter of runs (None: none), some pages missing."""

    def __init__(self, ctx, elem, dim, page, heads, group, lens, new, filt=0.0, holes=0.0, seed=1):
        from gofann_amd import kvcache
        r = np.random.default_rng(seed)
        self.elem, self.dim, self.heads, self.group, self.lens, self.new = elem, dim, heads, group, lens, new
        need = [-(-n // page) for n in lens]
        width, pages = max(need) + 1, sum(need) + 1
        order = r.permutation(pages)
        table = np.full((len(lens), width), -1, np.int32)
        at = 0
        for b, k in enumerate(need):
            table[b, :k] = order[at:at + k]
            at += k
        table[r.random(table.shape) < holes] = pages + 5
        g = torch.Generator(device="cuda").manual_seed(seed)
        rnd = lambda lo, hi, *s: torch.randint(lo, hi, s, device="cuda", generator=g).to(torch.uint8)  # noqa: E731
        self.cache = kvcache.KvCache(
            ctx, rnd(0, 256, pages, heads, page, dim // 2), rnd(123, 127, pages, heads, page, dim // 32),
            rnd(0, 256, pages, heads, page // 8, 16, 8, dim // 32),
            rnd(123, 127, pages, heads, page // 8, dim // 32, 8), dtype=TYPES[elem])
        dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        self.off = np.concatenate(([0], np.cumsum(new))).astype(np.int32)
        self.table, self.n = dev(table), int(self.off[-1])
        bits = None
        self.bits = np.ones((len(lens), width * page), bool)
        if filt:
            size = r.integers(1, 400, len(lens))
            for b in range(len(lens)):
                self.bits[b] = np.repeat(r.random(width * page // size[b] + 1) < filt, size[b])[:width * page]
            bits = dev(np.packbits(self.bits.reshape(len(lens), -1, 32), axis=-1,
                                   bitorder="little").view(np.int32)[..., 0])
        self.page, self.missing = page, table >= pages
        make = lambda off, q, most: kvcache.KvBatch(  # noqa: E731
            self.table, dev(np.array(lens, np.int32)), dev(off), queries=q, max_queries=most,
            max_length=max(lens), visible=bits)
        self.batch = make(self.off, self.n, max(new))
        whole = np.concatenate(([0], np.cumsum(lens))).astype(np.int32)
        held = make(whole, int(whole[-1]), max(lens))
        self.k, self.v = (x.double() for x in self.cache.read(held))
        self.starts = whole
        self.q = torch.randn(self.n, heads * group, dim, device="cuda", generator=g).to(TYPES[elem])
        self.parents = draft.trees(new, seed=seed)
        self.sees = draft.tree(new, self.parents)[0]
        self.words = dev(draft.words(self.sees))

    def check(self, out, lse, scale, sees=None, pick=None):
        """Against softmax over what each token may look at, within the error that 32-bit sums
        and roundings of weights and results to the element type allow."""
        H, G, D, u = self.heads, self.group, self.dim, ref.UNIT[self.elem]
        assert torch.isfinite(out).all()
        for b, (n, m) in enumerate(zip(self.lens, self.new)):
            if m == 0 or (pick is not None and b not in pick):
                continue
            there = self.bits[b, :n] & ~self.missing[b][np.arange(n) // self.page]
            ok = np.broadcast_to(there, (m, n)).copy()
            if sees is not None and n:
                t = np.arange(n) - (n - m)
                named = np.zeros((m, n), bool)
                inside = t >= 0
                named[:, inside] = sees[self.off[b]:self.off[b] + m][:, t[inside]]
                ok &= (t < 0) | named
            ok = torch.from_numpy(ok).cuda().repeat_interleave(G, 0)
            rows = slice(self.off[b], self.off[b] + m)
            k, v = self.k[self.starts[b]:self.starts[b] + n], self.v[self.starts[b]:self.starts[b] + n]
            for h in range(H):
                q = self.q[rows, h * G:(h + 1) * G].double().reshape(-1, D)
                s = (q @ k[:, h].T * scale).masked_fill(~ok, -np.inf) if n else q.new_zeros(len(q), 0)
                top = s.amax(-1, keepdim=True) if n else q.new_full((len(q), 1), -np.inf)
                none = torch.isinf(top)
                p = torch.exp(s - torch.where(none, torch.zeros_like(top), top))
                z = p.sum(-1, keepdim=True)
                p = p / torch.where(none, torch.ones_like(z), z)
                o = p @ v[:, h]
                mass = p @ v[:, h].abs()
                ds = (D + 8) * 2.0 ** -24 * scale * q.abs().sum(-1, keepdim=True) * 6 + 2.0 ** -21 * \
                    (1 + torch.where(none, torch.zeros_like(top), top).abs()) + n * 2.0 ** -24
                bound = 1.02 * u * (mass + o.abs()) + 4 * ds * mass
                if self.elem == "f16":
                    bound = bound + 2.0 ** -25 * (v[:, h].abs().sum(0) + 1)
                got = out[rows, h * G:(h + 1) * G].double().reshape(-1, D)
                off = (got - o).abs()
                assert (off <= bound).all(), (b, h, (off / bound).max().item())
                gl = lse[rows, h * G:(h + 1) * G].double().reshape(-1, 1)
                assert torch.equal(torch.isneginf(gl), none)
                want = top + torch.log(z)
                assert ((gl - want).abs()[~none] <= 1e-5 * (1 + want.abs()[~none])).all()

    def run(self, how, pick=None):
        scale = 0.7 * self.dim ** -0.5
        lse = torch.full((self.n, self.heads * self.group), 7.0, device="cuda")
        call = (lambda **kw: self.cache.cross(self.batch, self.q, scale=scale, **kw)) if how == "cross" else \
            (lambda **kw: self.cache.attend(self.batch, self.q, scale=scale, sees=self.words, **kw))
        out = call(lse=lse)
        assert torch.equal(out, call()), "two runs differ"
        self.check(out, lse, scale, None if how == "cross" else self.sees, pick)


def lengths(count, longest, seed=0, least=1):
    r = np.random.default_rng(seed)
    return [longest] + [int(least * (longest / least) ** r.random()) for _ in range(count - 1)]


@pytest.mark.parametrize("how", ["cross", "draft"])
@pytest.mark.parametrize("filt,holes", [(0.0, 0.0), (0.5, 0.2)])
@pytest.mark.parametrize("elem,dim,page,group,new,longest", [
    ("bf16", 128, 64, 4, 128, 2500),   # 128 rows a workgroup
    ("f16", 64, 32, 3, 171, 3000),     # 513 of them, the last tile nearly empty
    ("f16", 128, 128, 5, 77, 2300),
    ("bf16", 256, 64, 6, 64, 2200),
    ("f16", 256, 32, 2, 100, 9000),    # 32 rows of 256 channels
    ("bf16", 256, 64, 2, 30, 2500),    # 16 of them
    ("bf16", 64, 256, 2, 50, 2600),    # 32 rows
    ("bf16", 128, 32, 3, 9, 2400),
    ("f16", 128, 64, 1, 16, 2400),     # at most 16 rows
])
def test_unequal_sequences(ctx, elem, dim, page, group, new, longest, filt, holes, how):
    lens = lengths(6, longest, seed=new, least=new)
    r = np.random.default_rng(dim + new)
    counts = [new] + [int(r.integers(0, new + 1)) for _ in range(5)]
    if how == "cross":
        lens[2], lens[4] = 0, 1
    World(ctx, elem, dim, page, 2, group, lens, counts, filt, holes, seed=new).run(how)


@pytest.mark.parametrize("how", ["cross", "draft"])
@pytest.mark.parametrize("filt", [0.0, 0.4])
@pytest.mark.parametrize("elem,dim,heads,group,new,length", [
    ("bf16", 128, 4, 4, 128, 7001), ("f16", 64, 1, 7, 60, 40000), ("bf16", 256, 2, 8, 100, 9001),
    ("f16", 128, 8, 1, 40, 3000), ("bf16", 64, 20, 1, 20, 2200), ("f16", 256, 1, 4, 9, 70000),
])
def test_one_sequence(ctx, elem, dim, heads, group, new, length, filt, how):
    """Every row tile as long: parts that end with them; lists over more than one chunk of tiles."""
    World(ctx, elem, dim, 64, heads, group, [length], [new], filt, seed=new).run(how)


@pytest.mark.parametrize("how", ["cross", "draft"])
@pytest.mark.parametrize("elem,dim", [("bf16", 128), ("f16", 64)])
@pytest.mark.parametrize("filt", [0.0, 0.5])
def test_chunks_that_fill_the_chip(ctx, elem, dim, filt, how):
    """So many row tiles that each is a workgroup's, the longest sequences first."""
    new = [1100, 900, 1100, 0, 1000]
    lens = [1100, 1500, 1300, 50, 1001] if how == "draft" else [70, 900, 0, 50, 333]
    World(ctx, elem, dim, 64, 8, 4, lens, new, filt, seed=3).run(how)


@pytest.mark.parametrize("how", ["cross", "draft"])
@pytest.mark.parametrize("count,group,most", [(70, 4, 9), (200, 8, 40), (1030, 5, 5)])
@pytest.mark.parametrize("filt", [0.0, 0.5])
def test_many_sequences(ctx, count, group, most, filt, how):
    """More sequences than a wave has lanes, and more than tiles are shared out over."""
    r = np.random.default_rng(count)
    new = [most] + [int(r.integers(0, most + 1)) for _ in range(count - 1)]
    lens = [max(n, m) for n, m in zip(lengths(count, 2600, seed=count), new)]
    pick = set(range(12)) | set(range(60, 70)) | set(range(count - 8, count))
    World(ctx, "bf16", 64, 32, 1, group, lens, new, filt, seed=count).run(how, pick)


@pytest.mark.parametrize("how", ["cross", "draft"])
@pytest.mark.parametrize("dim,long", [(128, 600), (64, 130), (256, 300)])
def test_one_long_draft_among_many_short_ones(ctx, dim, long, how):
    """Row tiles counted through the sequences, where a grid of them would be mostly empty."""
    r = np.random.default_rng(dim)
    new = [1 + int(r.integers(0, 3)) for _ in range(60)]
    new[37] = long
    lens = [max(n, m) for n, m in zip(lengths(60, 2500, seed=dim), new)]
    World(ctx, "f16", dim, 64, 2, 3, lens, new, 0.0, seed=dim).run(how)


def test_short_calls_join_within_a_launch(ctx):
    for length in (1, 31, 33, 100, 500, 1000, 2048, 2049):
        for new in (1, 3, 20):
            if new <= length:
                World(ctx, "bf16", 128, 64, 2, 4, [length, new], [new, new], seed=length).run("draft")
                World(ctx, "f16", 64, 32, 2, 2, [length, 5], [new, 1], seed=length).run("cross")


def test_bounds_below_what_the_device_says_write_nothing_out_of_place(ctx):
    """max_queries below a sequence's tokens: what goes beyond is left out, as room for it is not there."""
    from gofann_amd import kvcache
    w = World(ctx, "bf16", 128, 64, 2, 4, [2500, 2300], [128, 100], seed=5)
    full = w.cache.cross(w.batch, w.q)
    short = kvcache.KvBatch(w.table, w.batch._keep[1], w.batch._keep[2], queries=w.n, max_queries=96,
                            max_length=2500)
    out = torch.full_like(w.q, 99.0)
    w.cache.cross(short, w.q, out=out)
    same = (out == 99.0).flatten(1).all(1) | ((out.float() - full.float()).abs() < 0.2).flatten(1).all(1)
    assert same.all()


@pytest.mark.parametrize("how", ["cross", "draft"])
@pytest.mark.parametrize("elem,dim,heads,group,length", [("bf16", 128, 2, 40, 3000), ("f16", 64, 1, 300, 2500),
                                                         ("bf16", 256, 1, 24, 2300), ("f16", 128, 1, 1024, 400)])
def test_one_token_each_under_many_heads(ctx, elem, dim, heads, group, length, how):
    """Rows of one token alone, without offsets, in every kind of row tile."""
    from gofann_amd import kvcache
    w = World(ctx, elem, dim, 64, heads, group, [length, 7, length // 2], [1, 1, 1], 0.6, seed=group)
    w.batch = kvcache.KvBatch(w.table, w.batch._keep[1], max_length=length, visible=w.batch._keep[3])
    w.run(how)


@pytest.mark.parametrize("how", ["cross", "draft"])
@pytest.mark.parametrize("dim,new,group", [(128, 40, 4), (128, 128, 4), (64, 130, 3), (256, 30, 2), (256, 200, 2)])
def test_far_scores_and_strange_queries_in_shared_tiles(ctx, how, dim, new, group):
    """Scaled scores past 2^22, and queries that hold an infinity or NaN, whose rows alone are lost."""
    w = World(ctx, "bf16", dim, 64, 2, group, [2600, 2500], [new, 3], seed=dim)
    call = (lambda q, **kw: w.cache.cross(w.batch, q, **kw)) if how == "cross" else \
        (lambda q, **kw: w.cache.attend(w.batch, q, sees=w.words, **kw))
    clean = call(w.q)
    q = w.q.clone()
    bad = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    for at, x in (((0, 1), float("nan")), ((1, 0), float("inf")), ((new, 2 * group - 1), float("-inf"))):
        q[(*at, 5)] = x
        bad[at] = True
    out = call(q)
    assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], clean[~bad])
    # one channel alone, of scores that are multiples of a large power of two: only the highest has weight
    q = torch.zeros_like(w.q)
    q[:, :, 0] = 1.0
    out = call(q, scale=2.0 ** 26)
    for b, n in enumerate(w.lens):
        k, v = w.k[w.starts[b]:w.starts[b] + n], w.v[w.starts[b]:w.starts[b] + n]
        for i in range(w.new[b]):
            ok = torch.ones(n, dtype=torch.bool, device="cuda")
            if how == "draft":
                ok[n - w.new[b]:] = torch.from_numpy(w.sees[w.off[b] + i][:w.new[b]]).cuda()
            for h in range(2):
                best = ok & (k[:, h, 0] == k[ok, h, 0].max())
                want = v[best, h].mean(0)
                off = (out[w.off[b] + i, h * group].double() - want).abs()
                # weights of one, an output's rounding, and sums of at most n values in 32 bits
                assert (off <= want.abs() * 2.0 ** -8 + v[best, h].abs().max() * n * 2.0 ** -23).all()


@pytest.mark.parametrize("dim,new", [(128, 30), (128, 128), (64, 1)])
def test_a_filter_without_words_hides_everything(ctx, dim, new):
    from gofann_amd import kvcache
    w = World(ctx, "f16", dim, 64, 2, 4, [2600, 200], [new, 1], seed=1)
    none = kvcache.KvBatch(w.table, w.batch._keep[1], w.batch._keep[2], queries=w.n, max_queries=new,
                           max_length=2600, visible=torch.empty((2, 0), dtype=torch.int32, device="cuda"))
    lse = torch.zeros((w.n, 8), device="cuda")
    assert (w.cache.cross(none, w.q, lse=lse) == 0).all() and torch.isneginf(lse).all()
    lse.zero_()
    assert (w.cache.attend(none, w.q, sees=w.words, lse=lse) == 0).all() and torch.isneginf(lse).all()


def test_graphs_of_shared_tiles_replay_after_larger_calls(gpu_ctx):
    """A captured call of shared tiles under a filter keeps its workspace while eager calls of other
    sizes, and a second graph, use the context between its replays."""
    from gofann_amd import _lib
    own = _lib.Context(0)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        own.bind_stream(side)
        some = World(own, "bf16", 128, 64, 2, 4, [3000, 500], [20, 9], 0.5, seed=1)
        more = World(own, "bf16", 128, 64, 2, 4, [2600, 2500, 900], [128, 100, 7], 0.5, seed=2)
        outs = [torch.empty_like(w.q) for w in (some, more)]
        call = lambda w, out: w.cache.attend(w.batch, w.q, sees=w.words, out=out)  # noqa: E731
        graphs = []
        for w, out in zip((some, more), outs):
            call(w, out)
            side.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                call(w, out)
            graphs.append(g)
        for i in range(4):
            for w, out, g in zip((some, more), outs, graphs):
                w.q.normal_()
                out.fill_(9.0)
                g.replay()
                side.synchronize()
                seen = out.clone()
                assert torch.equal(seen, call(w, out))
                more.cache.cross(more.batch, more.q)
            side.synchronize()
    own.close()
