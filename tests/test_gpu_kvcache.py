"""The 4-bit key/value cache on the GPU against its plain 64-bit definition
(kv_reference): quantized bytes, boxes and chosen blocks equal, attention
within the error that its roundings allow."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import torch

import kv_reference as ref

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def ctx(gpu_ctx):
    return gpu_ctx


def device_cache(ctx, c: ref.Cache):
    from gofann_amd import kvcache
    t = {n: torch.from_numpy(getattr(c, n)).cuda() for n in c.NAMES}
    return kvcache.KvCache(ctx, **t, dtype=TYPES[c.elem])


def device_batch(b: ref.Batch, one_token=False, max_length=None):
    from gofann_amd import kvcache
    dev = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    kw = dict(max_length=max(b.lens + [0]) if max_length is None else max_length, visible=dev(b.visible))
    lens = dev(np.array(b.lens, np.int32))
    if one_token:
        return kvcache.KvBatch(dev(b.table), lens, **kw)
    return kvcache.KvBatch(dev(b.table), lens, dev(b.offsets), queries=b.queries,
                           max_queries=max(b.new + [0]), **kw)


def rows(r, n, heads, dim, elem, magnitude=1.0):
    """Random rows of the element type, and the same in float64."""
    t = torch.from_numpy(magnitude * r.standard_normal((n, heads, dim))).to(TYPES[elem])
    return t.cuda(), t.double().numpy()


def spread(t, pad=3, shift=1):
    """The same rows at strides and addresses that no wide load fits."""
    n, h, d = t.shape
    big = torch.full((n, h, d + pad), 99.0, dtype=t.dtype, device=t.device).reshape(-1)
    big = torch.cat((big, big[:8]))
    view = big[shift:shift + n * h * (d + pad)].reshape(n, h, d + pad)[:, :, :d]
    view.copy_(t)
    return view


def check_attend(out, lse, want, want_lse, bound):
    o = out.double().cpu().numpy()
    assert np.isfinite(o).all()
    off = np.abs(o - want)
    assert (off <= bound).all(), f"{(off / np.maximum(bound, 1e-300)).max()} times the bound"
    if lse is not None:
        got = lse.double().cpu().numpy()
        empty = np.isinf(want_lse)
        assert np.array_equal(np.isneginf(got), empty)
        d = np.abs(got[~empty] - want_lse[~empty])
        assert (d <= 1e-5 * (1 + np.abs(want_lse[~empty]))).all(), d.max()


# ---- append ------------------------------------------------------------------

APPEND = [
    # elem, dim, page, heads, lengths, new
    ("bf16", 128, 64, 2, [1, 64, 65, 200], [1, 1, 1, 1]),
    ("f16", 128, 64, 3, [130, 7, 64], [130, 3, 64]),
    ("bf16", 64, 32, 1, [33, 70, 5], [2, 40, 5]),
    ("f16", 256, 128, 2, [129, 300], [2, 131]),
    ("bf16", 256, 256, 1, [257, 90], [17, 90]),
    ("f16", 64, 64, 2, [63, 1, 100], [1, 1, 0]),
]


@pytest.mark.parametrize("elem,dim,page,heads,lens,new", APPEND)
@pytest.mark.parametrize("plain_rows", [True, False])
def test_append_bytes_boxes_and_held_values(ctx, elem, dim, page, heads, lens, new, plain_rows):
    b = ref.Batch(page, lens, new, seed=dim + page, holes=0.0)
    c = ref.Cache(b.pages, heads, page, dim, elem, seed=3)
    old = ref.Batch(page, [n - m for n, m in zip(lens, new)], [0] * len(new), pages=b.pages)
    old.table, old.width = b.table, b.width
    ref.fill(c, old, seed=5)
    r = np.random.default_rng(7)
    k, k64 = rows(r, b.queries, heads, dim, elem)
    v, v64 = rows(r, b.queries, heads, dim, elem, 3.0)
    d = device_cache(ctx, c)
    kh, vh = torch.empty_like(k), torch.empty_like(v)
    if not plain_rows:
        k, v, kh, vh = spread(k), spread(v), spread(kh), spread(vh)
    d.append(device_batch(b), k, v, k_held=kh, v_held=vh)
    torch.cuda.synchronize()
    hk, hv = np.zeros_like(k64), np.zeros_like(v64)
    for row, s, pos in b.tokens():
        hk[row], hv[row] = c.write(b.table[s, pos // page], pos % page, k64[row], v64[row])
    for s, (n, m) in enumerate(zip(lens, new)):
        for j in range((n - m) // page, -(-n // page) if m else 0):
            c.renew_box(b.table[s, j], min(page, n - j * page))
    for name in c.NAMES:
        got = getattr(d, name).cpu().numpy()
        assert np.array_equal(got, getattr(c, name)), name
    assert np.array_equal(kh.double().cpu().numpy(), hk)
    assert np.array_equal(vh.double().cpu().numpy(), hv)


@pytest.mark.parametrize("elem", ["bf16", "f16"])
def test_append_of_extreme_values(ctx, elem):
    """Halfway values, zeros of both signs, the type's least and largest, NaN and infinities."""
    dim, page = 64, 32
    b = ref.Batch(page, [12], [12], seed=1)
    c = ref.Cache(b.pages, 1, page, dim, elem)
    x = np.zeros((12, 1, dim))
    half = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    x[0, 0, :8], x[0, 0, 8:16] = half, -half
    x[1, 0, :] = -0.0
    t = TYPES[elem]
    big, small = torch.finfo(t).max, torch.finfo(t).tiny
    x[2, 0, 0], x[2, 0, 40] = big, -big
    x[3, 0, 0], x[3, 0, 1] = small, -small
    x[4, 0, 5], x[4, 0, 6] = np.nan, 2.0
    x[5, 0, 5], x[5, 0, 6], x[5, 0, 40] = np.inf, 1.0, -np.inf
    x[6, 0, :] = np.nan
    x[7, 0, :32] = 6.0 * 2.0 ** -5
    x[8, 0, :32] = 6.0 * 2.0 ** -5 + 2.0 ** -9
    x[9, 0, 3] = -1.0
    x[10, 0, ::3] = 2.0 ** -20
    x[11, 0, :] = np.linspace(-7, 7, dim)
    xt = torch.from_numpy(x).to(t)
    x64 = xt.double().numpy()
    d = device_cache(ctx, c)
    held = torch.empty_like(xt.cuda())
    d.append(device_batch(b), xt.cuda(), -xt.cuda(), k_held=held)
    torch.cuda.synchronize()
    for row, s, pos in b.tokens():
        c.write(b.table[s, 0], pos, x64[row], -x64[row])
    c.renew_box(b.table[0, 0], 12)
    assert np.array_equal(d.k_scales.cpu().numpy(), c.k_scales)
    codes = d.k_codes.cpu().numpy()
    pid = b.table[0, 0]
    # the sign of a NaN's zero is open
    keep = ~np.isnan(x64[:, 0]).reshape(12, -1, 2).any(-1)
    assert np.array_equal(codes[pid, 0, :12][keep], c.k_codes[pid, 0, :12][keep])
    assert np.isfinite(held.double().cpu().numpy()).all()
    nan = np.isnan(x64[:, 0])
    assert (held.double().cpu().numpy()[:, 0][nan] == 0).all()
    assert np.array_equal(d.box.cpu().numpy()[pid], c.box[pid])
    assert np.array_equal(d.box_scale.cpu().numpy()[pid], c.box_scale[pid])


def test_append_in_pieces_equals_append_at_once(ctx):
    from gofann_amd import kvcache
    dim, page, heads = 128, 64, 2
    b = ref.Batch(page, [150], [150], seed=2)
    c = ref.Cache(b.pages, heads, page, dim, "bf16")
    r = np.random.default_rng(3)
    k, _ = rows(r, 150, heads, dim, "bf16")
    v, _ = rows(r, 150, heads, dim, "bf16")
    once, pieces = device_cache(ctx, c), device_cache(ctx, c)
    once.append(device_batch(b), k, v)
    table = torch.from_numpy(b.table).cuda()
    at = 0
    for m in (1, 62, 1, 1, 70, 15):
        length = torch.tensor([at + m], dtype=torch.int32, device="cuda")
        off = torch.tensor([0, m], dtype=torch.int32, device="cuda")
        pieces.append(kvcache.KvBatch(table, length, off, queries=m, max_queries=m, max_length=150),
                      k[at:at + m], v[at:at + m])
        at += m
    torch.cuda.synchronize()
    for name in c.NAMES:
        assert torch.equal(getattr(once, name), getattr(pieces, name)), name


def test_append_leaves_holes_and_negative_positions_alone(ctx):
    """A token without a page, or before position 0, is written nowhere."""
    dim, page = 128, 32
    b = ref.Batch(page, [70, 3], [70, 5], seed=4)
    b.table[0, 1] = b.pages  # a hole
    c = ref.Cache(b.pages, 1, page, dim, "f16")
    r = np.random.default_rng(5)
    k, k64 = rows(r, 75, 1, dim, "f16")
    v, v64 = rows(r, 75, 1, dim, "f16")
    d = device_cache(ctx, c)
    d.append(device_batch(b), k, v)
    torch.cuda.synchronize()
    for row, s, pos in b.tokens():
        pid = b.page_of(s, pos // page) if pos >= 0 else -1
        if pid >= 0:
            c.write(pid, pos % page, k64[row], v64[row])
    for s, j, n in ((0, 0, 32), (0, 2, 6), (1, 0, 3)):
        c.renew_box(b.table[s, j], n)
    for name in c.NAMES:
        assert np.array_equal(getattr(d, name).cpu().numpy(), getattr(c, name)), name


# ---- attend ------------------------------------------------------------------

def documents(b, n, r):
    """A filter of runs, as documents are; sequence 1 sees nothing."""
    if b == 1:
        return np.zeros(n, bool)
    keep = np.zeros(n, bool)
    at = 0
    while at < n:
        size = int(r.integers(1, 90))
        keep[at:at + size] = r.random() < 0.5
        at += size
    return keep


ATTEND = [
    # elem, dim, page, kv heads, group, lengths, new, filter, holes
    ("bf16", 128, 64, 2, 4, [1, 31, 32, 33, 64, 65], [1] * 6, None, 0),
    ("f16", 128, 64, 2, 8, [0, 5, 300], [1, 1, 1], None, 0),
    ("bf16", 64, 32, 3, 1, [97, 40], [1, 1], None, 0),
    ("bf16", 256, 128, 1, 16, [260, 130], [1, 1], None, 0),
    ("f16", 64, 256, 1, 7, [500, 20], [5, 3], None, 0),
    ("bf16", 128, 32, 1, 20, [75, 10], [1, 2], None, 0),
    ("f16", 256, 64, 2, 3, [90, 64], [17, 1], None, 0),
    ("bf16", 128, 64, 1, 4, [200, 33, 100], [33, 33, 0], None, 0),
    ("bf16", 64, 32, 1, 40, [70], [3], None, 0),
    ("f16", 128, 64, 2, 4, [300, 90, 200], [1, 1, 1], documents, 0),
    ("bf16", 128, 64, 1, 5, [300, 90, 200], [9, 2, 40], documents, 0),
    ("bf16", 64, 32, 2, 2, [300, 90, 200], [9, 2, 40], documents, 0.3),
    ("f16", 256, 32, 1, 2, [300, 90], [1, 1], None, 0.4),
    ("bf16", 128, 64, 1, 2, [3, 40], [7, 40], None, 0),  # more tokens than positions
]


@pytest.mark.parametrize("elem,dim,page,heads,group,lens,new,filt,holes", ATTEND)
def test_attend(ctx, elem, dim, page, heads, group, lens, new, filt, holes):
    b = ref.Batch(page, lens, new, seed=dim + group, holes=holes, visible=filt)
    c = ref.Cache(b.pages, heads, page, dim, elem, seed=1)
    ref.fill(c, b, seed=2, magnitude=2.0)
    q, q64 = rows(np.random.default_rng(3), b.queries, heads * group, dim, elem)
    scale = 1.3 * dim ** -0.5
    want = ref.attend(c, b, q64, scale)
    d, db = device_cache(ctx, c), device_batch(b)
    lse = torch.full((b.queries, heads * group), 7.0, device="cuda")
    out = d.attend(db, q, scale=scale, lse=lse)
    check_attend(out, lse, *want)
    assert torch.equal(out, d.attend(db, q, scale=scale)), "two runs differ"
    odd = spread(torch.zeros_like(q))
    d.attend(db, spread(q), scale=scale, out=odd)
    assert torch.equal(out, odd), "strides change the result"
    if all(m == 1 for m in new):
        assert torch.equal(out, d.attend(device_batch(b, one_token=True), q, scale=scale))


@pytest.mark.parametrize("elem,dim,group", [("bf16", 128, 8), ("f16", 64, 1), ("bf16", 256, 4)])
def test_attend_split_over_a_long_context(ctx, elem, dim, group):
    """Positions cut over many workgroups and joined, with a bound on the length that is far off."""
    b = ref.Batch(64, [3001, 17], [1, 1], seed=9)
    c = ref.Cache(b.pages, 1, 64, dim, elem, seed=1)
    ref.fill(c, b, seed=2)
    q, q64 = rows(np.random.default_rng(3), b.queries, group, dim, elem, 3.0)
    want = ref.attend(c, b, q64, dim ** -0.5)
    lse = torch.empty((2, group), device="cuda")
    d = device_cache(ctx, c)
    for most in (3001, 2 ** 20):
        out = d.attend(device_batch(b, max_length=most), q, lse=lse)
        check_attend(out, lse, *want)


@pytest.mark.parametrize("elem,dim,group,heads", [("bf16", 128, 4, 8), ("f16", 64, 3, 8), ("bf16", 256, 4, 8)])
def test_attend_of_long_chunks(ctx, elem, dim, group, heads):
    """Enough rows that every wave has row tiles of its own: chunks of unequal lengths."""
    new = [1100, 901, 64, 1000] if dim != 256 else [900, 300, 64, 900]
    lens = [1100, 920, 300, 1003] if dim != 256 else [900, 310, 300, 903]
    b = ref.Batch(64, lens, new, seed=9)
    c = ref.Cache(b.pages, heads, 64, dim, elem, seed=1)
    r = np.random.default_rng(4)
    # every position written at once: the same few rows over and over
    some = r.standard_normal((37, heads, dim))
    one = ref.Cache(1, heads, 64, dim, elem)
    pos = 0
    for s, n in enumerate(lens):
        for t in range(n):
            pid, at = b.table[s, t // 64], t % 64
            if pos < 37:
                one.write(0, pos, some[pos], some[36 - pos])
            i = pos % 37 if pos >= 37 else pos
            c.k_codes[pid, :, at] = one.k_codes[0, :, i]
            c.k_scales[pid, :, at] = one.k_scales[0, :, i]
            c.v_codes[pid, :, at // 8, :, at % 8] = one.v_codes[0, :, i // 8, :, i % 8]
            c.v_scales[pid, :, at // 8, :, at % 8] = one.v_scales[0, :, i // 8, :, i % 8]
            pos += 1
    q, q64 = rows(r, b.queries, heads * group, dim, elem, 2.0)
    d = device_cache(ctx, c)
    lse = torch.empty((b.queries, heads * group), device="cuda")
    out = d.attend(device_batch(b), q, lse=lse)
    # a sample of the rows, each with its own limit, as one-token batches
    pick = [0, 1, 63, 64, 255, 256, new[0] - 1, new[0], new[0] + 5, new[0] + new[1] - 1,
            b.queries - 1, b.queries - 900]
    tok = {row: (s, p) for row, s, p in b.tokens()}
    sub = ref.Batch(64, [tok[i][1] + 1 for i in pick], [1] * len(pick), pages=b.pages)
    sub.table = np.stack([b.table[tok[i][0]] for i in pick])
    sub.width = b.width
    want = ref.attend(c, sub, q64[pick], dim ** -0.5)
    check_attend(out[pick], lse[pick], *want)


def test_attend_of_a_mixed_batch(ctx):
    """Long chunks that fill the chip beside sequences of one and of a few tokens."""
    new = [2100, 1, 5, 2049, 0, 17]
    lens = [2100, 300, 5, 2060, 90, 400]
    heads, group, dim = 8, 2, 64
    b = ref.Batch(32, lens, new, seed=9)
    c = ref.Cache(b.pages, heads, 32, dim, "bf16", seed=1)
    r = np.random.default_rng(4)
    for name in ("k_codes", "v_codes"):
        getattr(c, name)[:] = r.integers(0, 256, getattr(c, name).shape)
    for name in ("k_scales", "v_scales"):
        getattr(c, name)[:] = r.integers(124, 128, getattr(c, name).shape)
    q, q64 = rows(r, b.queries, heads * group, dim, "bf16")
    d = device_cache(ctx, c)
    lse = torch.full((b.queries, heads * group), 7.0, device="cuda")
    out = torch.full_like(q, 99.0)
    d.attend(device_batch(b), q, out=out, lse=lse)
    tok = {row: (s, p) for row, s, p in b.tokens()}
    pick = [0, 1, 2099, 2100, 2101, 2105, 2106, 2107, 3000, 4154, 4155, 4160, 4171]
    sub = ref.Batch(32, [tok[i][1] + 1 for i in pick], [1] * len(pick), pages=b.pages)
    sub.table = np.stack([b.table[tok[i][0]] for i in pick])
    sub.width = b.width
    want = ref.attend(c, sub, q64[pick], dim ** -0.5)
    check_attend(out[pick], lse[pick], *want)
    assert (out != 99.0).any(-1).all() and (lse != 7.0).all()


def test_attend_scores_far_apart(ctx):
    """A maximum that grows along the sequence, and scores that underflow against it."""
    b = ref.Batch(64, [640], [1], seed=1)
    c = ref.Cache(b.pages, 1, 64, 128, "bf16", seed=1)
    r = np.random.default_rng(2)
    for t in range(640):
        k = r.standard_normal((1, 128)) * 0.1
        k[0, 0] = t / 8.0 if t % 97 else -300.0
        c.write(b.table[0, t // 64], t % 64, k, r.standard_normal((1, 128)))
    q = torch.zeros(1, 4, 128, dtype=torch.bfloat16)
    q[0, 0, 0], q[0, 1, 0], q[0, 2, 1], q[0, 3, 0] = 30.0, -30.0, 1.0, 0.001
    want = ref.attend(c, b, q.double().numpy(), 1.0)
    lse = torch.empty((1, 4), device="cuda")
    check_attend(device_cache(ctx, c).attend(device_batch(b), q.cuda(), scale=1.0, lse=lse), lse, *want)


@pytest.mark.parametrize("heads,group,new", [(1, 3, 1), (1, 3, 9), (8, 4, 1024)])
@pytest.mark.parametrize("dim", [64, 256])
def test_attend_f16_keeps_a_tail_of_small_weights(ctx, dim, heads, group, new):
    """One position's weight of 1 over thousands of 2^-25.5, which f16 alone would
    round to nothing: the small ones have all of the values, so their sum is the
    result.  In one launch, in splits and in long chunks."""
    n = 3000 + new
    b = ref.Batch(64, [n], [new], seed=3)
    c = ref.Cache(b.pages, heads, 64, dim, "f16")
    c.k_scales[:], c.v_scales[:], c.k_codes[:] = 127, 127, 0
    c.v_codes[:] = 0x77                                  # 6, 6
    pid = b.table[0, 10 // 64]
    c.k_codes[pid, :, 10, 0] = 7                         # a key of (6, 0, ..), its value 0
    c.v_codes[pid, :, 10 // 8, :, 10 % 8] = 0
    x = torch.tensor(25.5 * np.log(2.0) / 6, dtype=torch.float16)
    q = torch.zeros(new, heads * group, dim, dtype=torch.float16, device="cuda")
    q[:, :, 0] = x
    w = np.exp(-6.0 * float(x))
    many = n - new + np.arange(new, dtype=np.float64)    # small ones of each token
    z = 1 + many * w
    want = 6 * many * w / z
    lse = torch.empty(new, heads * group, device="cuda")
    out = device_cache(ctx, c).attend(device_batch(b), q, scale=1.0, lse=lse)
    # A weight is off by 2^-25 of at least 2^7 at the maximum, the result by half
    # an f16 unit; sums in 32 bits by 2^-24 a term, exponentials by 2^-21 of 18.
    bound = 2.0 ** -32 * 6 * many + 2.0 ** -25 + want * (2.0 ** -11 + (n + 64) * 2.0 ** -24 + 2.0 ** -16)
    off = np.abs(out.double().cpu().numpy() - want[:, None, None])
    assert (off <= bound[:, None, None]).all(), (off / bound[:, None, None]).max()
    got = lse.double().cpu().numpy()
    assert np.abs(got - (6.0 * float(x) + np.log(z))[:, None]).max() < 1e-4


def test_attend_infinite_and_nan_queries_stay_in_their_rows(ctx):
    b = ref.Batch(64, [100, 70], [1, 1], seed=1)
    c = ref.Cache(b.pages, 1, 64, 128, "bf16", seed=1)
    ref.fill(c, b)
    q, q64 = rows(np.random.default_rng(2), 2, 4, 128, "bf16")
    d, db = device_cache(ctx, c), device_batch(b)
    clean = d.attend(db, q)
    q[0, 1, 5] = float("nan")
    q[1, 2, 7] = float("inf")
    out = d.attend(db, q)
    bad = torch.zeros(2, 4, dtype=torch.bool, device="cuda")
    bad[0, 1] = bad[1, 2] = True
    assert torch.isnan(out[bad]).all()
    assert torch.equal(out[~bad], clean[~bad])


# ---- select and block lists --------------------------------------------------

SELECT = [
    # elem, dim, page, kv heads, group, lengths, new, width, first, last, filter, holes
    ("bf16", 128, 32, 2, 4, [1, 33, 900, 1500], [1] * 4, 8, 1, 2, None, 0),
    ("f16", 64, 32, 1, 1, [700, 1000], [1, 1], 5, 0, 0, None, 0),
    ("bf16", 256, 64, 1, 2, [1000, 40], [3, 2], 6, 1, 1, None, 0),
    ("f16", 128, 32, 2, 3, [600, 90], [5, 2], 7, 2, 3, None, 0),
    ("bf16", 64, 32, 1, 8, [600, 90, 300], [3, 2, 0], 64, 1, 2, None, 0),
    ("bf16", 128, 32, 1, 16, [640], [2], 4, 0, 4, None, 0),
    ("f16", 128, 32, 1, 20, [640], [2], 4, 1, 1, None, 0),
    ("bf16", 64, 64, 1, 40, [640], [1], 3, 1, 0, None, 0),
    ("bf16", 128, 32, 2, 4, [900, 300, 500], [4, 1, 1], 6, 1, 2, documents, 0.2),
    ("bf16", 64, 32, 1, 2, [2, 50], [5, 50], 3, 1, 1, None, 0),  # tokens before position 0
]


@pytest.mark.parametrize("elem,dim,page,heads,group,lens,new,width,first,last,filt,holes", SELECT)
def test_select(ctx, elem, dim, page, heads, group, lens, new, width, first, last, filt, holes):
    b = ref.Batch(page, lens, new, seed=dim + group, holes=holes, visible=filt)
    c = ref.Cache(b.pages, heads, page, dim, elem, seed=1)
    r = np.random.default_rng(4)
    c.box = np.sort(r.integers(-127, 128, c.box.shape), axis=2)[:, :, ::-1].astype(np.int8).copy()
    c.box_scale = r.integers(118, 124, c.box_scale.shape).astype(np.uint8)
    q, q64 = rows(r, b.queries, heads * group, dim, elem)
    d, db = device_cache(ctx, c), device_batch(b)
    got = d.select(db, q, width, first=first, last=last)
    want = ref.select(c, b, q64, width, first, last)
    assert np.array_equal(got.cpu().numpy(), want)
    assert torch.equal(got, d.select(db, spread(q), width, first=first, last=last))


@pytest.mark.parametrize("blocks,width", [(700, 40), (2100, 700), (9000, 64)])
def test_select_of_many_blocks_with_ties(ctx, blocks, width):
    """Scores that repeat: the lowest blocks of the last score are taken."""
    b = ref.Batch(32, [blocks * 32], [1], seed=3)
    c = ref.Cache(b.pages, 1, 32, 64, "bf16", seed=1)
    r = np.random.default_rng(4)
    kinds = np.sort(r.integers(-127, 128, (13, 1, 2, 64)), axis=2)[:, :, ::-1].astype(np.int8)
    c.box = kinds[r.integers(0, 13, b.pages)].copy()
    c.box_scale[:] = 120
    q, q64 = rows(r, 1, 2, 64, "bf16")
    got = device_cache(ctx, c).select(device_batch(b), q, width)
    assert np.array_equal(got.cpu().numpy(), ref.select(c, b, q64, width, 1, 2))


@pytest.mark.parametrize("up", [118, -110])
@pytest.mark.parametrize("new", [1, 3])
def test_select_of_queries_and_boxes_far_from_one(ctx, up, new):
    """Queries near the end of bf16's range against boxes at its other end: the
    scores lie in the middle, the integer product times one power alone does not."""
    b = ref.Batch(32, [32 * 40], [new], seed=3)
    c = ref.Cache(b.pages, 1, 32, 64, "bf16", seed=1)
    r = np.random.default_rng(4)
    c.box = np.sort(r.integers(-127, 128, c.box.shape), axis=2)[:, :, ::-1].astype(np.int8).copy()
    c.box_scale = (127 - up + r.integers(-2, 3, c.box_scale.shape)).astype(np.uint8)
    q, _ = rows(r, new, 2, 64, "bf16", 1.0)
    q = (q.float() * 2.0 ** up).to(torch.bfloat16)
    got = device_cache(ctx, c).select(device_batch(b), q, 9)
    assert np.array_equal(got.cpu().numpy(), ref.select(c, b, q.double().cpu().numpy(), 9, 1, 2))


def test_select_of_zero_and_nonfinite_queries(ctx):
    b = ref.Batch(32, [800], [3], seed=3)
    c = ref.Cache(b.pages, 1, 32, 128, "bf16", seed=1)
    ref.fill(c, b)
    q, _ = rows(np.random.default_rng(4), 3, 2, 128, "bf16")
    q[0] = 0
    q[1, 0, 3], q[1, 1, 4] = float("nan"), float("inf")
    q[2, 0, 5] = float("-inf")
    got = device_cache(ctx, c).select(device_batch(b), q, 6)
    assert np.array_equal(got.cpu().numpy(), ref.select(c, b, q.double().cpu().numpy(), 6, 1, 2))


LISTED = [
    ("bf16", 128, 64, 2, 4, [700, 65, 5], [1, 1, 1], None, 0),
    ("f16", 64, 32, 1, 7, [300, 100], [6, 1], None, 0),
    ("bf16", 256, 32, 1, 20, [300, 100], [2, 1], None, 0),
    ("bf16", 128, 32, 2, 3, [300, 90, 250], [4, 1, 3], documents, 0.2),
    ("f16", 128, 128, 1, 40, [600], [2], None, 0),
]


@pytest.mark.parametrize("elem,dim,page,heads,group,lens,new,filt,holes", LISTED)
def test_attend_to_listed_blocks(ctx, elem, dim, page, heads, group, lens, new, filt, holes):
    """Lists in any order, with gaps, blocks past the token's own and past the table."""
    b = ref.Batch(page, lens, new, seed=dim + group, holes=holes, visible=filt)
    c = ref.Cache(b.pages, heads, page, dim, elem, seed=1)
    ref.fill(c, b, seed=2)
    r = np.random.default_rng(5)
    q, q64 = rows(r, b.queries, heads * group, dim, elem)
    width = 5
    lists = np.stack([r.permutation(np.concatenate((np.arange(b.width), [-1, -5, b.width, 2 ** 30])))[:width]
                      for _ in range(b.queries * heads)]).reshape(b.queries, heads, width).astype(np.int32)
    lists[0, 0] = -1
    want = ref.attend(c, b, q64, dim ** -0.5, lists)
    lse = torch.empty((b.queries, heads * group), device="cuda")
    out = device_cache(ctx, c).attend(device_batch(b), q, blocks=torch.from_numpy(lists).cuda(), lse=lse)
    check_attend(out, lse, *want)


def test_all_blocks_listed_equal_no_list(ctx):
    b = ref.Batch(64, [1000, 130], [1, 1], seed=1)
    c = ref.Cache(b.pages, 2, 64, 128, "bf16", seed=1)
    ref.fill(c, b)
    q, q64 = rows(np.random.default_rng(2), 2, 8, 128, "bf16")
    d, db = device_cache(ctx, c), device_batch(b)
    blocks = d.select(db, q, b.width)
    want = ref.attend(c, b, q64, 128 ** -0.5)
    check_attend(d.attend(db, q, blocks=blocks), None, want[0], None, want[2])
    check_attend(d.attend(db, q), None, want[0], None, want[2])


# ---- machines ----------------------------------------------------------------

def test_cache_past_four_gigabytes(ctx):
    """Pages whose codes lie past 2^32 bytes."""
    from gofann_amd import kvcache
    d = kvcache.KvCache.empty(ctx, pages=150_000, kv_heads=8, dim=128)
    assert d.k_codes.numel() > 2 ** 32
    b = ref.Batch(64, [100], [100], pages=4, seed=1)
    small = ref.Cache(4, 8, 64, 128, "bf16")
    r = np.random.default_rng(2)
    k, k64 = rows(r, 100, 8, 128, "bf16")
    v, v64 = rows(r, 100, 8, 128, "bf16")
    for row, s, pos in b.tokens():
        small.write(b.table[s, pos // 64], pos % 64, k64[row], v64[row])
    for j, n in ((0, 64), (1, 36)):
        small.renew_box(b.table[0, j], n)
    db = device_batch(b)
    far = np.where(b.table >= 0, b.table + 150_000 - 4, b.table)
    db._keep[0].copy_(torch.from_numpy(far))
    d.append(db, k, v)
    q, q64 = rows(r, 100, 16, 128, "bf16")
    assert np.array_equal(d.select(db, q, 2, first=0, last=1).cpu().numpy(),
                          ref.select(small, b, q64, 2, 0, 1))
    want = ref.attend(small, b, q64, 128 ** -0.5)
    check_attend(d.attend(db, q), None, want[0], None, want[2])


def _step_world(ctx, seed=1):
    b = ref.Batch(64, [700, 130, 1], [1, 1, 1], seed=seed)
    c = ref.Cache(b.pages, 2, 64, 128, "bf16", seed=1)
    ref.fill(c, b)
    r = np.random.default_rng(seed)
    t = [rows(r, 3, h, 128, "bf16")[0] for h in (2, 2, 8)]
    return device_cache(ctx, c), device_batch(b, one_token=True), t


def test_calls_on_another_stream(gpu_ctx):
    from gofann_amd import _lib
    own = _lib.Context(0)
    d, db, (k, v, q) = _step_world(own)
    d.append(db, k, v)
    want = d.attend(db, q, blocks=d.select(db, q, 4))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        with pytest.raises(_lib.GofannError, match="stream"):
            d.attend(db, q)
        own.bind_stream(side)
        d.append(db, k, v)
        got = d.attend(db, q, blocks=d.select(db, q, 4))
        side.synchronize()
    assert torch.equal(want, got)
    own.close()


def test_graph_replays_equal_eager_steps(gpu_ctx):
    """A step captured once: append, select and attend, new inputs at each replay."""
    from gofann_amd import _lib
    own = _lib.Context(0)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        own.bind_stream(side)
        d, db, (k, v, q) = _step_world(own)
        blocks = torch.empty((3, 2, 4), dtype=torch.int32, device="cuda")
        out = torch.empty_like(q)

        def step():
            d.append(db, k, v)
            d.select(db, q, 4, out=blocks)
            d.attend(db, q, blocks=blocks, out=out)
            d.attend(db, q, out=dense)

        dense = torch.empty_like(q)
        step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        r = np.random.default_rng(11)
        for _ in range(4):
            for t in (k, v, q):
                t.copy_(rows(r, *t.shape, "bf16")[0])
            graph.replay()
            side.synchronize()
            seen = [t.clone() for t in (out, dense, blocks, d.k_codes, d.box)]
            step()
            side.synchronize()
            for a, e in zip(seen, (out, dense, blocks, d.k_codes, d.box)):
                assert torch.equal(a, e)
    own.close()


def test_workspace_too_small_under_capture_is_an_error(gpu_ctx):
    from gofann_amd import _lib
    own = _lib.Context(0)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        own.bind_stream(side)
        d, db, (k, v, q) = _step_world(own)
        out = torch.empty_like(q)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            d.append(db, k, v)  # needs none
            with pytest.raises(_lib.GofannError, match="before capturing"):
                d.attend(db, q, out=out)  # 700 positions in splits
        graph.replay()
        side.synchronize()
        d.attend(db, q, out=out)
        side.synchronize()
    own.close()


def test_session_of_the_example(ctx, capsys):
    """Prompt in chunks, then steps, against one attention over all of it."""
    from gofann_amd import longcontext
    r = np.random.default_rng(6)
    s = longcontext.Session(ctx, sequences=2, capacity=200, kv_heads=2, dim=64, page=32)
    c = ref.Cache(14, 2, 32, 64, "bf16")
    at, last = 0, None
    s.hide(1, 32, 96)
    for tokens, width in ((70, 0), (50, 7), (1, 0), (1, 3)):
        q, q64 = rows(r, 2 * tokens, 8, 64, "bf16")
        k, k64 = rows(r, 2 * tokens, 2, 64, "bf16")
        v, v64 = rows(r, 2 * tokens, 2, 64, "bf16")
        out = s.step(q, k, v, width)
        for b in range(2):
            for i in range(tokens):
                pos = at + i
                c.write(7 * b + pos // 32, pos % 32, k64[b * tokens + i], v64[b * tokens + i])
        at += tokens
        b = ref.Batch(32, [at, at], [tokens, tokens], pages=14,
                      visible=lambda i, n, _: ~((i == 1) & (np.arange(n) >= 32) & (np.arange(n) < 96)))
        b.table = np.arange(14, dtype=np.int32).reshape(2, 7)
        b.width = 7
        for j in range(14):
            n = min(32, at - 32 * (j % 7))
            if n > 0:
                c.renew_box(j, n)
        blocks = ref.select(c, b, q64, width, 1, 2) if width else None
        want = ref.attend(c, b, q64, 64 ** -0.5, blocks)
        check_attend(out, None, want[0], None, want[2])
    with pytest.raises(ValueError):
        s.grow(100)
    longcontext.main(["--context", "1500", "--steps", "2", "--sequences", "2", "--width", "8"])
    assert "8 blocks a token" in capsys.readouterr().out


# ---- refusals ----------------------------------------------------------------

def test_refusals_at_the_c_entry(ctx):
    from gofann_amd import _lib as L
    d, db, (k, v, q) = _step_world(ctx)
    lib, h = ctx.lib, ctx.handle
    out = torch.empty_like(q)
    rq = lambda t: L.KvRows(t.data_ptr(), t.stride(0), t.stride(1))  # noqa: E731
    blocks = torch.empty((3, 2, 4), dtype=torch.int32, device="cuda")

    def changed(view, **kw):
        w = type(view).from_buffer_copy(view)
        for n, x in kw.items():
            setattr(w, n, x)
        return w

    def attend(cache=d.view, batch=db.view, heads=8, scale=0.1, blk=None, width=0, rows_q=None, rows_o=None):
        return lib.gofann_kv_attention(h, cache, batch, rows_q or rq(q), heads, scale, blk, width,
                                       rows_o or rq(out), None)

    def select(cache=d.view, width=4, first=1, last=2, heads=8, dst=blocks.data_ptr()):
        return lib.gofann_kv_select(h, cache, db.view, rq(q), heads, width, first, last, dst)

    assert attend() == L.OK and select() == L.OK
    inv, uns = L.ERR_INVALID, L.ERR_UNSUPPORTED
    for rc, kw in [(uns, dict(dim=96)), (uns, dict(page_size=48)), (uns, dict(elem=L.ELEM_F32)),
                   (inv, dict(kv_heads=0)), (inv, dict(k_codes=None)), (inv, dict(v_scales=None)),
                   (inv, dict(k_codes=d.k_codes.data_ptr() + 8)), (inv, dict(box_scale=None)),
                   (uns, dict(pages=2 ** 31))]:
        assert attend(cache=changed(d.view, **kw)) == rc, kw
        assert ctx.last_error().startswith("kv_attention: ")
    for rc, kw in [(inv, dict(lengths=None)), (inv, dict(page_table=None)), (inv, dict(table_stride=1)),
                   (inv, dict(queries=2)), (uns, dict(sequences=70000)), (uns, dict(max_length=2 ** 31))]:
        assert attend(batch=changed(db.view, **kw)) == rc, kw
    for s in (0.0, -1.0, float("nan"), float("inf")):
        assert attend(scale=s) == inv
    for n in (0, 7):
        assert attend(heads=n) == inv and select(heads=n) == inv
    assert attend(blk=blocks.data_ptr(), width=0) == inv
    assert attend(rows_q=L.KvRows(None, 1, 1)) == inv
    assert attend(rows_o=L.KvRows(out.data_ptr() + 1, 1024, 128)) == inv
    assert select(width=0) == inv and select(width=2) == inv and select(dst=None) == inv
    assert select(cache=changed(d.view, box=None, box_scale=None)) == inv
    assert lib.gofann_kv_append(h, d.view, db.view, rq(k), None, None, None) == inv
    assert lib.gofann_kv_append(None, d.view, db.view, rq(k), rq(v), None, None) == inv
    assert lib.gofann_kv_append(h, None, db.view, rq(k), rq(v), None, None) == inv
    assert attend(batch=changed(db.view, queries=0, sequences=0)) == L.OK  # nothing to do
    torch.cuda.synchronize()
