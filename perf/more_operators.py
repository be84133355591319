"""Drafts and encoders over the 4-bit key/value cache, as cases to be timed:
attention for trees of drafted tokens, what settles such a draft once the model
has answered it, cross attention to an encoder's states, and the cache read back.

The cache is paged and holds a token's key and value in groups of 32 channels,
each channel as one of +-{0, .5, 1, 1.5, 2, 3, 4, 6} times the group's power of
two; `page_table[b][j]` is the page of positions [j P, (j+1) P) of sequence b:
  k_codes  [pages][kv_heads][P][dim/2]            low nibble: even channel
  k_scales [pages][kv_heads][P][dim/32]           exponent + 127
  v_codes  [pages][kv_heads][P/8][16][8][dim/32]  unit u of 16 holds channels
           [u dim/16, (u+1) dim/16) of the eight tokens one after another
  v_scales [pages][kv_heads][P/8][dim/32][8]
  box      [pages][kv_heads][2][dim] int8: most and least of the page's keys
           a channel, rounded outwards, times 2^(box_scale - 127)

A draft is a sequence's last `query_offsets[b+1] - query_offsets[b]` positions.
`parents[i]` is the draft's token before token i, by its index in the draft and
below i; a token with none is a root.  Token 0 is the one that the model chose
last.

`kind` picks the path:
  tree    attention of a draft's tokens over all positions before the draft and
          over those of the draft that `sees` names, one bit each: a token's
          ancestors and itself; a filter's clear bits are left out
  settle  a draft in the cache of one layer, but for its attention: the bits and
          depths of its tree, its keys and values appended, the path that the
          model's answers accept, and that path's tokens moved to the positions
          right behind the sequence's earlier ones, boxes renewed
  cross   attention of tokens over all positions of a sequence that they are no
          part of
  read    the values that the cache holds of each sequence's last tokens
"""
from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
LIMITS = {"bf16": (-125, 125), "f16": (-23, 13)}  # a group's exponents
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
KEEP = 0.6  # share of the positions that a filter leaves


def listed():
    return [
        # an interactive user's draft of a few tokens, latency alone
        dict(name="tree_one", kind="tree", elem="bf16", batch=1, tokens=25, heads=8, group=4,
             dim=128, page=64, shortest=2100, longest=2100, filter=False),
        # a server's drafts, sequences of all lengths, a filter on their positions
        dict(name="tree_serve", kind="tree", elem="bf16", batch=32, tokens=16, heads=8, group=4,
             dim=128, page=64, shortest=500, longest=16000, filter=True),
        # wide trees and many query heads to a key/value head: bound by the products
        dict(name="tree_wide", kind="tree", elem="bf16", batch=8, tokens=63, heads=8, group=8,
             dim=128, page=64, shortest=4000, longest=30000, filter=False),
        # one draft behind one long context
        dict(name="tree_long", kind="tree", elem="bf16", batch=1, tokens=60, heads=8, group=8,
             dim=128, page=128, shortest=200001, longest=200001, filter=False),
        # small heads, an odd group, small pages
        dict(name="tree_small", kind="tree", elem="f16", batch=19, tokens=40, heads=2, group=7,
             dim=64, page=32, shortest=300, longest=9001, filter=False),
        # a decoding step over an encoder's states, a query head for each key/value head
        dict(name="cross_step", kind="cross", elem="f16", batch=48, tokens=1, heads=20, group=1,
             dim=64, page=64, shortest=300, longest=1500, filter=False),
        # prompts of different lengths over encoded documents, some of them hidden
        dict(name="cross_prompt", kind="cross", elem="bf16", batch=6, tokens=701, heads=8, group=4,
             dim=128, page=64, shortest=900, longest=7000, filter=True),
        # a few tokens of wide heads over long encodings
        dict(name="cross_wide", kind="cross", elem="bf16", batch=10, tokens=9, heads=2, group=8,
             dim=256, page=64, shortest=2000, longest=20000, filter=False),
        # an interactive user's draft settled
        dict(name="settle_one", kind="settle", elem="bf16", batch=1, tokens=25, heads=8, dim=128,
             page=64, shortest=2100, longest=2100, width=10),
        # a server's drafts settled
        dict(name="settle_serve", kind="settle", elem="bf16", batch=64, tokens=40, heads=8, dim=128,
             page=64, shortest=200, longest=3000, width=10),
        # a few tokens looked at again
        dict(name="read_tail", kind="read", elem="bf16", batch=30, tokens=17, heads=8, dim=128,
             page=64, shortest=100, longest=2000),
        # whole sequences taken out of the cache
        dict(name="read_whole", kind="read", elem="f16", batch=5, tokens=6001, heads=8, dim=128,
             page=64, shortest=6001, longest=6001),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "tree", "cross", "cross", "cross", "settle", "read"])
    c = dict(kind=kind, elem=rng.choice(["bf16", "f16"]), heads=rng.choice([1, 2, 3, 4, 8]),
             dim=rng.choice([64, 128, 128, 256]), page=rng.choice([32, 64, 64, 128]))
    c["batch"] = _log(rng, 1, 64)
    if kind == "read":
        c["tokens"] = _log(rng, 1, max(2, 30_000 // c["batch"]))
        c["longest"] = c["tokens"] + rng.randint(0, 2000)
        c["shortest"] = max(c["tokens"], _log(rng, 10, c["longest"]))
        return c
    if kind == "settle":
        c["tokens"] = _log(rng, 2, 128)
        c["longest"] = c["tokens"] + _log(rng, 10, 4000)
        c["shortest"] = max(c["tokens"], _log(rng, 10, c["longest"]))
        c["width"] = _log(rng, 2, 24)
        return c
    c["group"] = rng.choice([1, 2, 3, 4, 5, 8, 16])
    c["tokens"] = (_log(rng, 2, 128) if kind == "tree"
                   else rng.choice([1, 1, _log(rng, 2, max(3, 4000 // c["batch"]))]))
    # positions that a pass reads and pairs that it computes, both below the largest listed
    most = 1_600_000 * 128 // (c["batch"] * c["heads"] * c["dim"])
    most = min(most, 7 * 10 ** 8 * 128 // (c["batch"] * c["tokens"] * c["heads"] * c["group"] * c["dim"]))
    c["longest"] = c["tokens"] + _log(rng, 60, max(100, min(most, 200_000)))
    c["shortest"] = max(c["tokens"] if kind == "tree" else 1, _log(rng, 30, c["longest"]))
    c["filter"] = rng.random() < 0.4
    return c


def _lengths(c):
    """Every sequence's length, spread over the case's range, and its new tokens."""
    r = random.Random("%s %s %s" % (c["batch"], c["longest"], c["tokens"]))
    n = c["batch"]
    lens = [c["longest"]] + [_log(r, c["shortest"], c["longest"]) for _ in range(n - 1)]
    new = [c["tokens"]] + [r.randint(1 + c["tokens"] // 2, c["tokens"]) if c["tokens"] > 1 else 1
                           for _ in range(n - 1)]
    return lens, new


# ---- the plain forms ---------------------------------------------------------------------

def _pow2(e):
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _exponent(amax, top):
    """The least x with amax <= top 2^x, for top in (0.5, 1]."""
    m, x = torch.frexp(amax)
    return x + (m > top).to(torch.int32)


def _codes(x, elem):
    """4-bit codes [..][dim] (one a byte) and the groups' exponents [..][dim/32] of finite rows."""
    g = x.float().reshape(*x.shape[:-1], -1, 32)
    a = g.abs()
    amax = a.amax(-1)
    lo, hi = LIMITS[elem]
    e = torch.where(amax > 0, _exponent(amax, 0.75) - 3, torch.full_like(amax, lo, dtype=torch.int32))
    e = e.clamp(lo, hi)
    a = a * _pow2(-e)[..., None]
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5)
            + (a >= 3.5) + (a > 5))
    code = code | (torch.signbit(g).to(torch.uint8) << 3)
    return code.reshape(x.shape), e


def _values(codes, e):
    """What codes [..][dim] in groups of exponents [..][dim/32] stand for, in 32 bits."""
    table = torch.tensor([*GRID, *[-v for v in GRID]], device=codes.device)
    v = table[codes.long()].reshape(*codes.shape[:-1], -1, 32)
    return (v * _pow2(e)[..., None]).reshape(codes.shape)


def _pack(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _unpack(b):
    return torch.stack((b & 15, b >> 4), -1).flatten(-2)


def _pages_k(s, pid):
    """Keys [.., kv_heads, P, dim] of pages."""
    return _values(_unpack(s["k_codes"][pid]), s["k_scales"][pid].to(torch.int32) - 127)


def _pages_v(s, pid):
    c, e = s["v_codes"][pid], s["v_scales"][pid].to(torch.int32) - 127
    c = c.transpose(-3, -2).flatten(-2)      # [.., P/8, 8, 16 units of bytes]
    c = c.flatten(-3, -2)                    # [.., P, dim/2]
    e = e.transpose(-2, -1).flatten(-3, -2)  # [.., P, dim/32]
    return _values(_unpack(c), e)


def _where(s):
    """Sequence, position and index in its sequence of every token of the call."""
    off, lens = s["query_offsets"].long(), s["lengths"].long()
    i = torch.arange(s["queries"], device=off.device)
    seq = torch.searchsorted(off, i, right=True) - 1
    nth = i - off[seq]
    return seq, lens[seq] - (off[seq + 1] - off[seq]) + nth, nth


def _bits(words, n):
    """Words [..][w] as truth values [..][n]."""
    b = (words[..., None] >> torch.arange(32, device=words.device, dtype=torch.int32)) & 1
    return b.flatten(-2)[..., :n].bool()


def _words(bits):
    """Truth values [..][32 w] as words [..][w]."""
    w = (bits.unflatten(-1, (-1, 32)).long() << torch.arange(32, device=bits.device)).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def _visible(s, positions):
    """The filter's bits [batch][positions], True without one."""
    if s["visible"] is None:
        return torch.ones(s["page_table"].shape[0], positions, dtype=torch.bool, device=DEV)
    return _bits(s["visible"], positions)


def _softmax(x):
    """Rows of scores, -inf where masked; a row of nothing gives zeros."""
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    return p / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _plain_attend(s):
    c = s["case"]
    H, G, D = c["heads"], c["group"], c["dim"]
    B, T = c["batch"], s["max_queries"]
    seq, _, nth = _where(s)
    table = s["page_table"].long().clamp(min=0)
    k = _pages_k(s, table).transpose(1, 2).flatten(2, 3)  # [B, H, positions, D]
    v = _pages_v(s, table).transpose(1, 2).flatten(2, 3)
    L = k.shape[2]
    q = torch.zeros(B, T, H * G, D, device=DEV)
    q[seq, nth] = s["q"].float()
    q = q.reshape(B, T, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, T * G, D)
    x = torch.matmul(q, k.transpose(2, 3)) * s["scale"]
    t = torch.arange(L, device=DEV)
    lens, off = s["lengths"].long(), s["query_offsets"].long()
    ok = ((t < lens[:, None]) & _visible(s, L))[:, None]  # [B, 1 or T, L]
    if c["kind"] == "tree":
        sees = torch.zeros(B, T, s["sees"].shape[1] * 32, dtype=torch.bool, device=DEV)
        sees[seq, nth] = _bits(s["sees"], sees.shape[2])
        start = (lens - (off[1:] - off[:-1]))[:, None, None]
        nth_of = (t - start).clamp(0, sees.shape[2] - 1).expand(B, T, L)
        ok = ok & ((t < start) | torch.gather(sees, 2, nth_of))
    ok = ok.expand(B, T, L)
    x = x.reshape(B, H, T, G, L).masked_fill(~ok[:, None, :, None], -math.inf)
    o = torch.matmul(_softmax(x).reshape(B, H, T * G, L), v)
    o = o.reshape(B, H, T, G, D).permute(0, 2, 1, 3, 4).reshape(B, T, H * G, D)
    return o[seq, nth].to(s["q"].dtype)


def _renew_boxes(s, first, lens, most):
    """Boxes of the pages, at most `most` of a sequence, that hold positions [first, lens)."""
    P = s["case"]["page"]
    block = first[:, None] // P + torch.arange(most, device=DEV)
    b, j = torch.nonzero(block * P < lens[:, None], as_tuple=True)
    block = block[b, j]
    pid = s["page_table"].long()[b, block]
    k = _pages_k(s, pid)
    there = (block[:, None] * P + torch.arange(P, device=DEV)) < lens[b][:, None]
    there = there[:, None, :, None]
    hi = torch.where(there, k, torch.full_like(k, -math.inf)).amax(2)
    lo = torch.where(there, k, torch.full_like(k, math.inf)).amin(2)
    amax = torch.maximum(hi.abs(), lo.abs()).amax(-1)
    e = torch.where(amax > 0, _exponent(amax, 127 / 128) - 7, torch.full_like(amax, -125, dtype=torch.int32))
    e = e.clamp(-125, 125)
    inv = _pow2(-e)[..., None]
    s["box"][pid] = torch.stack((torch.ceil(hi * inv), torch.floor(lo * inv)), 2).to(torch.int8)
    s["box_scale"][pid] = (e + 127).to(torch.uint8)


def _plain_settle(s):
    c, P, T, width = s["case"], s["case"]["page"], s["max_queries"], s["case"]["width"]
    seq, pos, nth = _where(s)
    lens, off = s["lengths"].long(), s["query_offsets"].long()
    new = off[1:] - off[:-1]
    start = lens - new
    # Ancestors as a matrix [B, T, T]: parents taken twice as far each time.
    B = c["batch"]
    padded = torch.full((3, B, T), -1, dtype=torch.long, device=DEV)
    padded[:, seq, nth] = torch.stack((s["parents"], s["drafted"], s["chosen"])).long()
    parents, drafted, chosen = padded
    j = torch.arange(T, device=DEV)
    there = j < new[:, None]
    ancestors = ((parents[..., None] == j) | (j[:, None] == j)).float()
    for _ in range((T - 1).bit_length()):
        ancestors = (torch.matmul(ancestors, ancestors) > 0).float()
    ancestors = ancestors.bool() & there[..., None]
    words = (T + 31) // 32
    sees = _words(torch.nn.functional.pad(ancestors, (0, 32 * words - T)))[seq, nth]
    depths = (ancestors.sum(-1) - 1)[seq, nth].to(torch.int32)
    # Keys and values.
    pid, at = s["page_table"].long()[seq, pos // P], pos % P
    kc, ke = _codes(s["k"], c["elem"])
    vc, ve = _codes(s["v"], c["elem"])
    s["k_codes"][pid, :, at] = _pack(kc)
    s["k_scales"][pid, :, at] = (ke + 127).to(torch.uint8)
    s["v_codes"][pid, :, at // 8, :, at % 8] = _pack(vc).reshape(*vc.shape[:2], 16, -1)
    s["v_scales"][pid, :, at // 8, :, at % 8] = (ve + 127).to(torch.uint8)
    _renew_boxes(s, start, lens, T // P + 2)
    # The answer to token i accepts the first of its children that drafted it; a token is on
    # the path where that holds for it and all of its ancestors but token 0.
    child = (parents[:, None] == j[:, None]) & (drafted[:, None] == chosen[..., None]) & there[:, None]
    first = torch.where(child, j, T).amin(-1)                       # [B, T], T: none
    good = (torch.gather(first, 1, parents.clamp(min=0)) == j) & (parents >= 0)
    good[:, 0] = True
    on = (good[:, None] | ~ancestors).all(-1) & there
    order = torch.sort(torch.where(on, j, T), dim=-1)[0]
    order = torch.nn.functional.pad(order, (0, max(0, width - T)), value=T)[:, :width]
    path = torch.where(order < T, order, torch.full_like(order, -1))
    count = (path >= 0).sum(-1)
    answer = torch.gather(chosen, 1, torch.gather(path, 1, (count - 1)[:, None]))[:, 0]
    # The path's tokens moved together, all of them read before any is written.
    b, i = torch.nonzero(path >= 0, as_tuple=True)
    src, dst = start[b] + path[b, i], start[b] + i
    table = s["page_table"].long()
    p0, a0, p1, a1 = table[b, src // P], src % P, table[b, dst // P], dst % P
    s["k_codes"][p1, :, a1] = s["k_codes"][p0, :, a0]
    s["k_scales"][p1, :, a1] = s["k_scales"][p0, :, a0]
    s["v_codes"][p1, :, a1 // 8, :, a1 % 8] = s["v_codes"][p0, :, a0 // 8, :, a0 % 8]
    s["v_scales"][p1, :, a1 // 8, :, a1 % 8] = s["v_scales"][p0, :, a0 // 8, :, a0 % 8]
    _renew_boxes(s, start, start + count, T // P + 2)
    return {"sees": sees, "depths": depths, "path": path.to(torch.int32),
            "lengths": (start + count).to(torch.int32), "next": answer.to(torch.int32), **_arrays(s)}


def _plain_read(s):
    P = s["case"]["page"]
    seq, pos, _ = _where(s)
    pid, at = s["page_table"].long()[seq, pos // P], pos % P
    dt = TYPES[s["case"]["elem"]]
    k = _values(_unpack(s["k_codes"][pid, :, at]), s["k_scales"][pid, :, at].to(torch.int32) - 127)
    v = _values(_unpack(s["v_codes"][pid, :, at // 8, :, at % 8].flatten(2)),
                s["v_scales"][pid, :, at // 8, :, at % 8].to(torch.int32) - 127)
    return {"k": k.to(dt), "v": v.to(dt)}


# ---- inputs ------------------------------------------------------------------------------

_ARRAYS = ("k_codes", "k_scales", "v_codes", "v_scales", "box", "box_scale")


def _arrays(s):
    return {n: s[n] for n in _ARRAYS}


def _drafts(new, seed):
    """Trees of so many tokens, what they drafted, and the model's answer to each token: mostly
    one of its children, drawn from few tokens, so that siblings have drafted the same."""
    r = random.Random(seed)
    parents, drafted, chosen = [], [], []
    for n in new:
        p = [-1] + [r.randint(max(0, (i - 1) // 2 - 2), i - 1) for i in range(1, n)]
        d = [r.randint(0, 7) for _ in range(n)]
        a = [r.randint(0, 9) for _ in range(n)]
        for i in range(n - 1, 0, -1):
            if r.random() < 0.85:
                a[p[i]] = d[i]
        parents += p
        drafted += d
        chosen += a
    return parents, drafted, chosen


def _sees(new, parents):
    """The bits of every token's ancestors and itself, in words."""
    words, rows, at = (max(new) + 31) // 32, [], 0
    for n in new:
        m = []
        for i in range(n):
            p = parents[at + i]
            m.append((m[p] if p >= 0 else 0) | 1 << i)
        rows += [[x >> 32 * w & 0xFFFFFFFF for w in range(words)] for x in m]
        at += n
    return torch.tensor(rows, dtype=torch.int64).to(torch.int32)


def prepare(case, seed):
    """A cache with the sequences' tokens in it, in pages of random order, and what the call
    brings.  Keys have a part that a run of positions shares (what a text is about there), a
    constant part with a few strong channels, and noise; queries ask for some run's part."""
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    H, D, P, elem = c["heads"], c["dim"], c["page"], c["elem"]
    lens, new = _lengths(c)
    need = [-(-n // P) for n in lens]
    W, pages = max(need), sum(need) + 3
    order = torch.randperm(pages, device=DEV, generator=g).to(torch.int32).cpu()
    table = torch.full((c["batch"], W), -1, dtype=torch.int32)
    n = 0
    for b, k in enumerate(need):
        table[b, :k] = order[n:n + k]
        n += k
    randn = lambda *shape: torch.randn(*shape, device=DEV, generator=g)  # noqa: E731
    base = 0.5 * randn(H, D) * (1 + 6 * (torch.rand(H, D, device=DEV, generator=g) < 0.04))
    topics = randn(64, H, D)
    s = dict(case=c, page_table=table.to(DEV), pages=pages,
             lengths=torch.tensor(lens, dtype=torch.int32, device=DEV),
             query_offsets=torch.tensor([sum(new[:i]) for i in range(len(new) + 1)],
                                        dtype=torch.int32, device=DEV),
             queries=sum(new), max_queries=max(new), max_length=max(lens), scale=D ** -0.5,
             visible=None,
             k_codes=torch.empty(pages, H, P, D // 2, dtype=torch.uint8, device=DEV),
             k_scales=torch.empty(pages, H, P, D // 32, dtype=torch.uint8, device=DEV),
             v_codes=torch.empty(pages, H, P // 8, 16, 8, D // 32, dtype=torch.uint8, device=DEV),
             v_scales=torch.empty(pages, H, P // 8, D // 32, 8, dtype=torch.uint8, device=DEV),
             box=torch.empty(pages, H, 2, D, dtype=torch.int8, device=DEV),
             box_scale=torch.empty(pages, H, dtype=torch.uint8, device=DEV))
    step = max(1, (1 << 27) // (H * P * D))
    for i in range(0, pages, step):
        m = min(step, pages - i)
        about = topics[torch.randint(0, 64, (m,), device=DEV, generator=g)]
        x = base[None, :, None] + about[:, :, None] + 0.7 * randn(m, H, P, D)
        kc, e = _codes(x, elem)
        s["k_codes"][i:i + m] = _pack(kc)
        s["k_scales"][i:i + m] = (e + 127).to(torch.uint8)
        x = _values(kc, e)
        hi, lo = x.amax(2), x.amin(2)
        e = _exponent(torch.maximum(hi, -lo).amax(-1), 127 / 128) - 7
        inv = _pow2(-e)[..., None]
        s["box"][i:i + m] = torch.stack((torch.ceil(hi * inv), torch.floor(lo * inv)), 2).to(torch.int8)
        s["box_scale"][i:i + m] = (e + 127).to(torch.uint8)
        vc, e = _codes(randn(m, H, P, D) + 0.3, elem)
        vc = _pack(vc).reshape(m, H, P // 8, 8, 16, D // 32)
        s["v_codes"][i:i + m] = vc.transpose(3, 4)
        s["v_scales"][i:i + m] = (e + 127).to(torch.uint8).reshape(m, H, P // 8, 8, -1).transpose(3, 4)
    N, dt = s["queries"], TYPES[elem]
    if c["kind"] == "read":
        return s
    about = topics[torch.randint(0, 64, (N,), device=DEV, generator=g)]
    parents, drafted, chosen = _drafts(new, seed)
    if c["kind"] == "settle":
        for name, x in (("parents", parents), ("drafted", drafted), ("chosen", chosen)):
            s[name] = torch.tensor(x, dtype=torch.int32).to(DEV)
        s["k"] = (base + about + 0.7 * randn(N, H, D)).to(dt)
        s["v"] = (randn(N, H, D) + 0.3).to(dt)
        return s
    if c["kind"] == "tree":
        s["sees"] = _sees(new, parents).to(DEV)
    s["q"] = (0.5 * about.repeat_interleave(c["group"], 1) + randn(N, H * c["group"], D)).to(dt)
    if c["filter"]:  # documents of a sequence are kept or left out as a whole
        t = torch.arange(W * P, device=DEV)
        size = torch.randint(40, 700, (c["batch"], 1), device=DEV, generator=g)
        keep = torch.rand(c["batch"], W * P // 40 + 1, device=DEV, generator=g) < KEEP
        s["visible"] = _words(torch.gather(keep, 1, t // size))
    return s


_ctx = None


def _handles(s):
    """The framework's handles of a state, made once as a program keeps them."""
    global _ctx
    if "cache" not in s:
        pkg = str(Path(__file__).resolve().parent.parent / "go-fann_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from gofann_amd import _lib, kvcache
        if _ctx is None:
            _ctx = _lib.Context(0)
        s["cache"] = kvcache.KvCache(_ctx, *[s[n] for n in _ARRAYS[:4]], box=s["box"],
                                     box_scale=s["box_scale"], dtype=TYPES[s["case"]["elem"]])
        s["batch"] = kvcache.KvBatch(s["page_table"], s["lengths"], s["query_offsets"],
                                     queries=s["queries"], max_queries=s["max_queries"],
                                     max_length=s["max_length"], visible=s["visible"])
        s["kvcache"] = kvcache
    return s["cache"], s["batch"], s["kvcache"]


def run(state):
    s, kind = state, state["case"]["kind"]
    if not own:
        return {"tree": _plain_attend, "cross": _plain_attend, "settle": _plain_settle,
                "read": _plain_read}[kind](s)
    cache, batch, kvcache = _handles(s)
    if kind == "tree":
        return cache.attend(batch, s["q"], scale=s["scale"], sees=s["sees"])
    if kind == "cross":
        return cache.cross(batch, s["q"], scale=s["scale"])
    if kind == "read":
        k, v = cache.read(batch)
        return {"k": k, "v": v}
    sees, depths = kvcache.draft_tree(cache.ctx, batch, s["parents"])
    cache.append(batch, s["k"], s["v"])
    path, lengths, answer = kvcache.draft_accept(cache.ctx, batch, s["parents"], s["drafted"],
                                                 s["chosen"], s["case"]["width"])
    cache.keep(batch, path)
    return {"sees": sees, "depths": depths, "path": path, "lengths": lengths, "next": answer,
            **_arrays(s)}


def work(case):
    c = case
    H, D, P = c["heads"], c["dim"], c["page"]
    lens, new = _lengths(c)
    N = sum(new)
    token = H * (D // 2 + D // 32)  # a key or a value of one position, all heads
    if c["kind"] == "read":
        return {"bytes": N * 2 * (token + 2 * H * D), "flops": N * 2 * H * D}
    words = (max(new) + 31) // 32
    if c["kind"] == "settle":
        # the keys of every page that a draft falls in are read again for its box
        pages = sum((n - 1) // P - (n - m) // P + 1 for n, m in zip(lens, new))
        return {"bytes": N * (2 * H * D * 2 + 2 * token + 12 + 4 + 4 * words)
                + pages * (P * token + H * (2 * D + 1)) + len(lens) * 4 * (c["width"] + 2),
                "flops": N * 2 * H * D * 4 + pages * P * H * D * 2}
    Hq, keep = H * c["group"], KEEP if c["filter"] else 1.0
    extra = 2 * N * Hq * D * 2 + (sum(lens) // 8 if c["filter"] else 0)
    pairs = sum(m * n for n, m in zip(lens, new))
    if c["kind"] == "tree":
        extra += N * 4 * words
        pairs -= sum(m * (m - 1) for m in new)  # itself at least
    return {"bytes": int(keep * sum(lens)) * 2 * token + extra, "flops": int(keep * pairs * Hq * D * 4)}


# ---- the definition in 64 bits -----------------------------------------------------------

def _number(c):
    """A code's value from its sign, exponent and mantissa bits."""
    c = c.to(torch.int64)
    ex, man = (c >> 1) & 3, (c & 1).double()
    mag = torch.where(ex == 0, 0.5 * man, (1 + 0.5 * man) * torch.pow(2.0, (ex - 1).double()))
    return torch.where((c & 8) != 0, -mag, mag)


def _exact_kv(s, b, t):
    """Keys and values [..][H][D] of positions t of sequence b in 64 bits."""
    D, P = s["case"]["dim"], s["case"]["page"]
    pid, at = s["page_table"][b].long()[t // P], t % P
    ch = torch.arange(D, device=DEV)
    shift = (ch % 2) * 4
    k = _number((s["k_codes"][pid, :, at][..., ch // 2].long() >> shift) & 15)
    k *= torch.pow(2.0, s["k_scales"][pid, :, at][..., ch // 32].double() - 127)
    unit, inside = ch // (D // 16), ch % (D // 16)
    v = s["v_codes"][pid, :, at // 8, :, at % 8].flatten(2)[..., unit * (D // 32) + inside // 2]
    v = _number((v.long() >> shift) & 15)
    v *= torch.pow(2.0, s["v_scales"][pid, :, at // 8, :, at % 8][..., ch // 32].double() - 127)
    return k, v


def _exact_attend(s):
    c = s["case"]
    H, G, D = c["heads"], c["group"], c["dim"]
    out = torch.zeros(s["queries"], H * G, D, dtype=torch.float64, device=DEV)
    off = s["query_offsets"].tolist()
    for b, n in enumerate(s["lengths"].tolist()):
        i, j = off[b], off[b + 1]
        ok = torch.ones(j - i, n, dtype=torch.bool, device=DEV)
        if c["kind"] == "tree":
            t = torch.arange(j - i, device=DEV)
            ok[:, n - (j - i):] = (s["sees"][i:j].long()[:, t // 32] >> (t % 32)) & 1 == 1
        if s["visible"] is not None:
            t = torch.arange(n, device=DEV)
            ok &= (s["visible"][b].long()[t // 32] >> (t % 32)) & 1 == 1
        ok = ok.repeat_interleave(G, 0)
        k, v = _exact_kv(s, b, torch.arange(n, device=DEV))
        for h in range(H):
            q = s["q"][i:j, h * G:(h + 1) * G].double().reshape(-1, D)
            x = torch.where(ok, q @ k[:, h].T * s["scale"], -1e300)
            p = torch.exp(x - x.max(-1, keepdim=True)[0]) * ok
            z = p.sum(-1, keepdim=True)
            p = torch.where(z > 0, p / torch.where(z > 0, z, 1.0), torch.zeros_like(p))
            out[i:j, h * G:(h + 1) * G] = (p @ v[:, h]).reshape(j - i, G, D)
    return out


def _exact_settle(s):
    """Token by token; what the cache holds then is whole numbers."""
    c = s["case"]
    new = [b - a for a, b in zip(s["query_offsets"].tolist(), s["query_offsets"].tolist()[1:])]
    parents, drafted, chosen = (s[n].tolist() for n in ("parents", "drafted", "chosen"))
    depths, path, lengths, answer, at = [], [], [], [], 0
    for n, length in zip(new, s["lengths"].tolist()):
        for i in range(n):
            d, p = 0, parents[at + i]
            while p >= 0:
                d, p = d + 1, parents[at + p]
            depths.append(d)
        walk = [0]
        while len(walk) < c["width"]:
            at_most = [j for j in range(walk[-1] + 1, n)
                       if parents[at + j] == walk[-1] and drafted[at + j] == chosen[at + walk[-1]]]
            if not at_most:
                break
            walk.append(at_most[0])
        path.append(walk + [-1] * (c["width"] - len(walk)))
        lengths.append(length - n + len(walk))
        answer.append(chosen[at + walk[-1]])
        at += n
    whole = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    return {"sees": _sees(new, parents).to(DEV), "depths": whole(depths), "path": whole(path),
            "lengths": whole(lengths), "next": whole(answer), **{n: None for n in _ARRAYS}}


def _exact_read(s):
    off = s["query_offsets"].tolist()
    rows = [_exact_kv(s, b, torch.arange(n - (off[b + 1] - off[b]), n, device=DEV))
            for b, n in enumerate(s["lengths"].tolist())]
    return {"k": torch.cat([k for k, _ in rows]), "v": torch.cat([v for _, v in rows])}


def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _exact_attend, "cross": _exact_attend, "settle": _exact_settle,
            "read": _exact_read}[case["kind"]](s)
