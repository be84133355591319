"""The operators of the 4-bit key/value cache, as cases to be timed: writing
tokens into it, attention over it, and attention over the blocks of it that a
cheap score selects for each query.

The cache is paged.  `page_table[b][j]` is the page that holds the positions
[j P, (j+1) P) of sequence b, `lengths[b]` its positions, the last
`query_offsets[b+1] - query_offsets[b]` of which are this call's tokens.  A
token's key and its value are held in groups of 32 channels, each channel as
one of +-{0, .5, 1, 1.5, 2, 3, 4, 6} times the group's power of two:
  k_codes  [pages][kv_heads][P][dim/2]            low nibble: even channel
  k_scales [pages][kv_heads][P][dim/32]           exponent + 127
  v_codes  [pages][kv_heads][P/8][16][8][dim/32]  unit u of 16 holds channels
           [u dim/16, (u+1) dim/16) of the eight tokens one after another
  v_scales [pages][kv_heads][P/8][dim/32][8]
  box      [pages][kv_heads][2][dim] int8: most and least of the page's keys
           a channel, rounded outwards, times 2^(box_scale - 127)

`kind` picks the path:
  append   new tokens' keys and values quantized into their pages, the boxes
           of the pages they fall in, and the values that the cache then holds
  attend   attention of new tokens over all positions up to their own, those
           whose bit in `visible` is clear left out
  select   per token and key/value head the `width` blocks to read: the first,
           the last and those whose box has the highest products with a query
  sparse   select, then attention over the selected blocks
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
        # one decoding step of a server: every sequence's newest token
        dict(name="append_step", kind="append", elem="bf16", batch=64, tokens=1, heads=8, dim=128,
             page=64, shortest=200, longest=3000),
        # prompts of different lengths written behind what is there already
        dict(name="append_prompt", kind="append", elem="f16", batch=5, tokens=4001, heads=8,
             dim=128, page=64, shortest=4100, longest=9000),
        # an interactive user's next token, latency alone
        dict(name="attend_one", kind="attend", elem="bf16", batch=1, tokens=1, heads=8, group=4,
             dim=128, page=64, shortest=1999, longest=1999, filter=False),
        # a server's decoding step, sequences of all lengths, a filter on their positions
        dict(name="attend_serve", kind="attend", elem="bf16", batch=48, tokens=1, heads=8, group=4,
             dim=128, page=64, shortest=500, longest=16000, filter=True),
        # one long context, the whole chip on one token
        dict(name="attend_long", kind="attend", elem="bf16", batch=1, tokens=1, heads=8, group=8,
             dim=128, page=128, shortest=500001, longest=500001, filter=False),
        # drafts of up to five tokens to be verified, small heads, an odd group
        dict(name="attend_draft", kind="attend", elem="f16", batch=19, tokens=5, heads=2, group=7,
             dim=64, page=32, shortest=300, longest=9001, filter=False),
        # one key/value head under many query heads, wide heads
        dict(name="attend_wide", kind="attend", elem="bf16", batch=20, tokens=1, heads=1, group=16,
             dim=256, page=64, shortest=2000, longest=33000, filter=False),
        # a chunk of a long prompt over what was written before it, causal
        dict(name="attend_chunk", kind="attend", elem="bf16", batch=1, tokens=2048, heads=8, group=4,
             dim=128, page=64, shortest=16390, longest=16390, filter=False),
        # the choice of blocks of a decoding step over long contexts
        dict(name="select_step", kind="select", elem="bf16", batch=16, tokens=1, heads=8, group=4,
             dim=128, page=64, shortest=20000, longest=131072, filter=False, width=64),
        # a single user's token over a long context, by 4096 of its positions
        dict(name="sparse_one", kind="sparse", elem="bf16", batch=1, tokens=1, heads=8, group=4,
             dim=128, page=64, shortest=131000, longest=131000, filter=False, width=64),
        # a server's decoding step over long contexts with a filter
        dict(name="sparse_serve", kind="sparse", elem="f16", batch=12, tokens=1, heads=8, group=8,
             dim=128, page=64, shortest=9000, longest=100000, filter=True, width=48),
        # a chunk of a prompt, each of its tokens over its own blocks
        dict(name="sparse_chunk", kind="sparse", elem="bf16", batch=2, tokens=300, heads=4, group=8,
             dim=128, page=64, shortest=20000, longest=40000, filter=False, width=24),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "select",
                       "sparse", "sparse"])
    c = dict(kind=kind, elem=rng.choice(["bf16", "f16"]), heads=rng.choice([1, 2, 3, 4, 8]),
             dim=rng.choice([64, 128, 128, 256]), page=rng.choice([32, 64, 64, 128]))
    c["batch"] = _log(rng, 1, 64)
    if kind == "append":
        c["tokens"] = rng.choice([1, _log(rng, 2, max(3, 16_000 // c["batch"]))])
        c["longest"] = c["tokens"] + _log(rng, 10, 4000)
        c["shortest"] = max(c["tokens"], _log(rng, 10, c["longest"]))
        return c
    c["group"] = rng.choice([1, 2, 3, 4, 5, 8, 16, 20])
    tokens = (1600 if kind == "attend" else 200) // c["batch"]
    c["tokens"] = rng.choice([1, 1, _log(rng, 2, max(3, tokens))])
    # positions that a pass reads and pairs that it computes, both below the largest listed
    most = 2_400_000 * 128 // (c["batch"] * c["heads"] * c["dim"])
    most = min(most, 10 ** 9 * 128 // (c["batch"] * c["tokens"] * c["heads"] * c["group"] * c["dim"]))
    c["longest"] = c["tokens"] + _log(rng, 100, max(200, min(most, 400_000)))
    c["shortest"] = max(c["tokens"], _log(rng, 30, c["longest"]))
    c["filter"] = rng.random() < 0.4
    if kind != "attend":
        rows = c["batch"] * c["tokens"] * c["heads"] * c["page"] * c["dim"]
        c["width"] = _log(rng, 4, max(5, min(64, 400_000_000 // rows)))
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
    """4-bit codes [..][dim] (one a byte) and the groups' exponents [..][dim/32]."""
    g = x.float().reshape(*x.shape[:-1], -1, 32)
    g = torch.where(torch.isnan(g), torch.zeros_like(g), g)
    a = g.abs()
    amax = torch.where(torch.isinf(a), torch.zeros_like(a), a).amax(-1)
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


def _pages_k(s, pid, h=None):
    """Keys of pages: [.., kv_heads, P, dim], or [.., P, dim] of heads `h`."""
    at = (pid,) if h is None else (pid, h)
    return _values(_unpack(s["k_codes"][at]), s["k_scales"][at].to(torch.int32) - 127)


def _pages_v(s, pid, h=None):
    at = (pid,) if h is None else (pid, h)
    c, e = s["v_codes"][at], s["v_scales"][at].to(torch.int32) - 127
    c = c.transpose(-3, -2).flatten(-2)      # [.., P/8, 8, 16 units of bytes]
    c = c.flatten(-3, -2)                    # [.., P, dim/2]
    e = e.transpose(-2, -1).flatten(-3, -2)  # [.., P, dim/32]
    return _values(_unpack(c), e)


def _where(s):
    """Sequence, position and index in its sequence of every new token."""
    off, lens = s["query_offsets"].long(), s["lengths"].long()
    i = torch.arange(s["queries"], device=off.device)
    seq = torch.searchsorted(off, i, right=True) - 1
    nth = i - off[seq]
    return seq, lens[seq] - (off[seq + 1] - off[seq]) + nth, nth


def _visible(s, positions):
    """Bits [batch][positions] of the filter, True without one."""
    if s["visible"] is None:
        return torch.ones(s["page_table"].shape[0], positions, dtype=torch.bool, device=DEV)
    w = s["visible"]
    bits = (w[..., None] >> torch.arange(32, device=w.device, dtype=torch.int32)) & 1
    return bits.flatten(1)[:, :positions].bool()


def _plain_append(s):
    c, P = s["case"], s["case"]["page"]
    seq, pos, _ = _where(s)
    pid, at = s["page_table"].long()[seq, pos // P], pos % P
    kc, ke = _codes(s["k"], c["elem"])
    vc, ve = _codes(s["v"], c["elem"])
    s["k_codes"][pid, :, at] = _pack(kc)
    s["k_scales"][pid, :, at] = (ke + 127).to(torch.uint8)
    s["v_codes"][pid, :, at // 8, :, at % 8] = _pack(vc).reshape(*vc.shape[:2], 16, -1)
    s["v_scales"][pid, :, at // 8, :, at % 8] = (ve + 127).to(torch.uint8)
    lens = s["lengths"].long()
    new = (s["query_offsets"][1:] - s["query_offsets"][:-1]).long()
    j = torch.arange(s["max_queries"] // P + 2, device=DEV)
    block = (lens - new)[:, None] // P + j
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
    dt = TYPES[c["elem"]]
    return {"k": _values(kc, ke).to(dt), "v": _values(vc, ve).to(dt),
            **{n: s[n] for n in ("k_codes", "k_scales", "v_codes", "v_scales", "box", "box_scale")}}


def _softmax(x):
    """Rows of scores, -inf where masked; a row of nothing gives zeros."""
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    return p / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _plain_attend(s):
    c = s["case"]
    H, G, D = c["heads"], c["group"], c["dim"]
    B, T = c["batch"], s["max_queries"]
    seq, pos, nth = _where(s)
    table = s["page_table"].long().clamp(min=0)
    k = _pages_k(s, table).transpose(1, 2).flatten(2, 3)  # [B, H, positions, D]
    v = _pages_v(s, table).transpose(1, 2).flatten(2, 3)
    L = k.shape[2]
    q = torch.zeros(B, T, H * G, D, device=DEV)
    q[seq, nth] = s["q"].float()
    last = torch.full((B, T), -1, dtype=torch.long, device=DEV)
    last[seq, nth] = pos
    q = q.reshape(B, T, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, T * G, D)
    x = torch.matmul(q, k.transpose(2, 3)) * s["scale"]
    ok = (torch.arange(L, device=DEV) <= last[..., None]) & _visible(s, L)[:, None]  # [B, T, L]
    x = x.reshape(B, H, T, G, L).masked_fill(~ok[:, None, :, None], -math.inf)
    o = torch.matmul(_softmax(x).reshape(B, H, T * G, L), v)
    o = o.reshape(B, H, T, G, D).permute(0, 2, 1, 3, 4).reshape(B, T, H * G, D)
    return o[seq, nth].to(s["q"].dtype)


def _plain_select(s):
    c = s["case"]
    H, G, D, P = c["heads"], c["group"], c["dim"], c["page"]
    B, T, W = c["batch"], s["max_queries"], s["page_table"].shape[1]
    seq, pos, nth = _where(s)
    q = torch.zeros(B, T, H * G, D, device=DEV)
    q[seq, nth] = s["q"].float()
    q = q.reshape(B, T, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, T * G, D)
    amax = q.abs().amax(-1, keepdim=True)
    e = torch.where(amax > 0, torch.frexp(amax)[1] - 7, torch.full_like(amax, -125, dtype=torch.int32))
    e = e.clamp(-125, 125)
    q = torch.round(q * _pow2(-e)).clamp(-127, 127)
    page = s["page_table"].long().clamp(min=0)
    box = s["box"][page].float().permute(3, 0, 2, 4, 1)  # [2, B, H, D, W]
    x = torch.matmul(q.clamp(min=0), box[0]) + torch.matmul(q.clamp(max=0), box[1])  # whole numbers
    x = x * _pow2(e) * _pow2(s["box_scale"][page].to(torch.int32) - 127).transpose(1, 2)[:, :, None]
    x = x.reshape(B, H, T, G, W).amax(3)
    last = torch.full((B, T), -1, dtype=torch.long, device=DEV)
    last[seq, nth] = pos
    t = torch.arange(W * P, device=DEV)
    ok = (t <= last[..., None]) & _visible(s, W * P)[:, None]
    ok = ok.reshape(B, T, W, P).any(-1)
    j = torch.arange(W, device=DEV)
    blocks = last[..., None] // P + 1
    must = (j < s["first"]) | (j >= blocks - s["last"])
    x = x.masked_fill(must[:, None], math.inf).masked_fill(~ok[:, None], -math.inf)
    got = torch.sort(x, dim=-1, descending=True, stable=True)
    n = min(c["width"], W)
    at = torch.where(torch.isinf(got[0]) & (got[0] < 0), torch.full_like(got[1], W), got[1])[..., :n]
    at = torch.sort(at, dim=-1)[0]
    at = torch.nn.functional.pad(at, (0, c["width"] - n), value=W)
    at = torch.where(at == W, torch.full_like(at, -1), at)
    return at.transpose(1, 2)[seq, nth].to(torch.int32)


def _plain_sparse(s):
    c = s["case"]
    H, G, D, P = c["heads"], c["group"], c["dim"], c["page"]
    blocks = _plain_select(s)
    seq, pos, _ = _where(s)
    N, S = blocks.shape[0], blocks.shape[2]
    at = blocks.long().clamp(min=0)
    page = s["page_table"].long()[seq[:, None, None], at].clamp(min=0)
    h = torch.arange(H, device=DEV)[None, :, None].expand_as(page)
    k = _pages_k(s, page, h).flatten(2, 3)  # [N, H, S P, D]
    v = _pages_v(s, page, h).flatten(2, 3)
    t = (at[..., None] * P + torch.arange(P, device=DEV)).flatten(2)
    ok = (t <= pos[:, None, None]) & (blocks >= 0)[..., None].expand(N, H, S, P).flatten(2)
    if s["visible"] is not None:
        ok &= (s["visible"][seq[:, None, None], t // 32] >> (t % 32)) & 1 == 1
    x = torch.matmul(s["q"].float().reshape(N, H, G, D), k.transpose(2, 3)) * s["scale"]
    o = torch.matmul(_softmax(x.masked_fill(~ok[:, :, None], -math.inf)), v)
    return {"blocks": blocks, "out": o.reshape(N, H * G, D).to(s["q"].dtype)}


# ---- inputs ------------------------------------------------------------------------------

def prepare(case, seed):
    """A cache with the sequences' earlier tokens in it, in pages of random order, and
    this call's tokens.  Keys have a part that a run of positions shares (what a text
    is about there), a constant part with a few strong channels, and noise; queries ask
    for some run's part."""
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
             first=1, last=2, visible=None,
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
    if c["kind"] == "append":
        about = topics[torch.randint(0, 64, (N,), device=DEV, generator=g)]
        s["k"] = (base + about + 0.7 * randn(N, H, D)).to(dt)
        s["v"] = (randn(N, H, D) + 0.3).to(dt)
        return s
    about = topics[torch.randint(0, 64, (N,), device=DEV, generator=g)]
    s["q"] = (0.5 * about.repeat_interleave(c["group"], 1) + randn(N, H * c["group"], D)).to(dt)
    if c["filter"]:  # documents of a sequence are kept or left out as a whole
        t = torch.arange(W * P, device=DEV)
        size = torch.randint(40, 700, (c["batch"], 1), device=DEV, generator=g)
        keep = torch.rand(c["batch"], W * P // 40 + 1, device=DEV, generator=g) < KEEP
        keep = torch.gather(keep, 1, t // size).reshape(c["batch"], -1, 32).long()
        word = (keep << torch.arange(32, device=DEV)).sum(-1)
        s["visible"] = torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32)
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
        s["cache"] = kvcache.KvCache(_ctx, s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"],
                                     box=s["box"], box_scale=s["box_scale"],
                                     dtype=TYPES[s["case"]["elem"]])
        s["batch"] = kvcache.KvBatch(s["page_table"], s["lengths"], s["query_offsets"],
                                     queries=s["queries"], max_queries=s["max_queries"],
                                     max_length=s["max_length"], visible=s["visible"])
    return s["cache"], s["batch"]


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "select": _plain_select,
                "sparse": _plain_sparse}[c["kind"]](s)
    cache, batch = _handles(s)
    if c["kind"] == "append":
        k, v = torch.empty_like(s["k"]), torch.empty_like(s["v"])
        cache.append(batch, s["k"], s["v"], k_held=k, v_held=v)
        return {"k": k, "v": v,
                **{n: s[n] for n in ("k_codes", "k_scales", "v_codes", "v_scales", "box", "box_scale")}}
    if c["kind"] == "attend":
        return cache.attend(batch, s["q"], scale=s["scale"])
    blocks = cache.select(batch, s["q"], c["width"], first=s["first"], last=s["last"])
    if c["kind"] == "select":
        return blocks
    return {"blocks": blocks, "out": cache.attend(batch, s["q"], scale=s["scale"], blocks=blocks)}


def work(case):
    c = case
    H, D, P = c["heads"], c["dim"], c["page"]
    lens, new = _lengths(c)
    N = sum(new)
    token = H * (D // 2 + D // 32)  # a key or a value of one position, all heads
    if c["kind"] == "append":
        pages = sum((n - 1) // P - (n - m) // P + 1 for n, m in zip(lens, new))
        return {"bytes": N * (2 * H * D * 2 * 2 + 2 * token) + pages * H * (2 * D + 1),
                "flops": N * 2 * H * D * 4}
    Hq, keep = H * c["group"], KEEP if c["filter"] else 1.0
    qo = N * Hq * D * 2
    bits = sum(lens) // 8 if c["filter"] else 0
    if c["kind"] == "attend":
        pairs = sum(m * n - m * (m - 1) // 2 for n, m in zip(lens, new))
        return {"bytes": int(keep * sum(lens)) * 2 * token + 2 * qo + bits,
                "flops": int(keep * pairs * Hq * D * 4)}
    blocks = [-(-n // P) for n in lens]
    w = {"bytes": sum(blocks) * H * (2 * D + 1) + qo + N * H * c["width"] * 4 + bits,
         "flops": sum(b * m for b, m in zip(blocks, new)) * Hq * D * 2}
    if c["kind"] == "sparse":
        per = [min(c["width"] * P, n) for n in lens]
        w["bytes"] += sum(min(n, m * k) for n, m, k in zip(lens, new, per)) * 2 * token + qo
        w["flops"] += int(keep * sum(m * k for m, k in zip(new, per)) * Hq * D * 4)
    return w


# ---- the definition in 64 bits -----------------------------------------------------------

def _number(c):
    """A code's value from its sign, exponent and mantissa bits."""
    c = c.to(torch.int64)
    ex, man = (c >> 1) & 3, (c & 1).double()
    mag = torch.where(ex == 0, 0.5 * man, (1 + 0.5 * man) * torch.pow(2.0, (ex - 1).double()))
    return torch.where((c & 8) != 0, -mag, mag)


def _exact_kv(s, b, n, only=None):
    """Keys and values [n][H][D] of sequence b's first n positions in 64 bits."""
    D, P = s["case"]["dim"], s["case"]["page"]
    table = s["page_table"][b].long()
    t = torch.arange(n, device=DEV) if only is None else only
    pid, at = table[t // P], t % P
    ch = torch.arange(D, device=DEV)
    shift = (ch % 2) * 4
    k = _number((s["k_codes"][pid, :, at][..., ch // 2].long() >> shift) & 15)
    k *= torch.pow(2.0, s["k_scales"][pid, :, at][..., ch // 32].double() - 127)
    unit, inside = ch // (D // 16), ch % (D // 16)
    v = s["v_codes"][pid, :, at // 8, :, at % 8].flatten(2)[..., unit * (D // 32) + inside // 2]
    v = _number((v.long() >> shift) & 15)
    v *= torch.pow(2.0, s["v_scales"][pid, :, at // 8, :, at % 8][..., ch // 32].double() - 127)
    return k, v


def _exact_rows(s):
    off, lens = s["query_offsets"].tolist(), s["lengths"].tolist()
    for b in range(len(lens)):
        yield b, off[b], off[b + 1], lens[b]


def _exact_bits(s, b, n):
    if s["visible"] is None:
        return torch.ones(n, dtype=torch.bool, device=DEV)
    t = torch.arange(n, device=DEV)
    return ((s["visible"][b].long()[t // 32] >> (t % 32)) & 1).bool()


def _exact_softmax(x, ok):
    x = torch.where(ok, x, torch.full_like(x, -1e300))
    p = torch.exp(x - x.max(-1, keepdim=True)[0]) * ok
    z = p.sum(-1, keepdim=True)
    return torch.where(z > 0, p / torch.where(z > 0, z, torch.ones_like(z)), torch.zeros_like(p))


def _exact_attend(s):
    c = s["case"]
    H, G, D = c["heads"], c["group"], c["dim"]
    out = torch.zeros(s["queries"], H * G, D, dtype=torch.float64, device=DEV)
    for b, i, j, n in _exact_rows(s):
        k, v = _exact_kv(s, b, n)
        ok = (torch.arange(n, device=DEV)[None] <= torch.arange(n - (j - i), n, device=DEV)[:, None])
        ok = (ok & _exact_bits(s, b, n)).repeat_interleave(G, 0)
        for h in range(H):
            q = s["q"][i:j, h * G:(h + 1) * G].double().reshape(-1, D)
            p = _exact_softmax(q @ k[:, h].T * s["scale"], ok)
            out[i:j, h * G:(h + 1) * G] = (p @ v[:, h]).reshape(j - i, G, D)
    return out


def _exact_select(s):
    c = s["case"]
    H, G, D, P, width = c["heads"], c["group"], c["dim"], c["page"], c["width"]
    out = torch.full((s["queries"], H, width), -1, dtype=torch.int32, device=DEV)
    for b, i, j, n in _exact_rows(s):
        pid = s["page_table"][b, :-(-n // P)].long()
        box = s["box"][pid].double()                      # [blocks, H, 2, D]
        unit = torch.pow(2.0, s["box_scale"][pid].double() - 127)
        bits = torch.zeros(len(pid) * P, dtype=torch.bool, device=DEV)
        bits[:n] = _exact_bits(s, b, n)
        for r in range(i, j):
            pos = n - (j - r)
            blocks = pos // P + 1
            q = s["q"][r].double().reshape(H, G, D)
            big = q.abs().max(-1, keepdim=True)[0]
            step = torch.pow(2.0, torch.floor(torch.log2(big)) - 6)
            q8 = torch.clamp(torch.round(q / step), -127, 127)
            part = torch.maximum(torch.clamp(q8, min=0), torch.zeros_like(q8))
            x = part @ box[:blocks, :, 0].permute(1, 2, 0) - (part - q8) @ box[:blocks, :, 1].permute(1, 2, 0)
            x = (x * step).amax(1) * unit[:blocks].T       # [H, blocks]
            seen = bits.clone()
            seen[pos + 1:] = False
            seen = seen.reshape(-1, P).any(1)[:blocks]
            at = torch.arange(blocks, device=DEV)
            x = torch.where(((at < s["first"]) | (at >= blocks - s["last"]))[None], 1e300, x)
            m = min(width, int(seen.sum()))
            x = torch.where(seen[None], x, -1e300)
            best = torch.argsort(-x, dim=-1, stable=True)[:, :m]
            out[r, :, :m] = torch.sort(best, dim=-1)[0].to(torch.int32)
    return out


def _exact_sparse(s):
    c = s["case"]
    H, G, D, P = c["heads"], c["group"], c["dim"], c["page"]
    blocks = _exact_select(s)
    out = torch.zeros(s["queries"], H * G, D, dtype=torch.float64, device=DEV)
    for b, i, j, n in _exact_rows(s):
        k, v = _exact_kv(s, b, n)
        k, v = k.permute(1, 2, 0).contiguous(), v.permute(1, 0, 2).contiguous()
        bits = _exact_bits(s, b, n)
        for r in range(i, j):
            pos = n - (j - r)
            t = torch.arange(n, device=DEV)
            ok = torch.zeros(H, n + P, dtype=torch.bool, device=DEV)
            at = blocks[r].long()
            at = (torch.where(at < 0, n // P + 1, at)[..., None] * P + torch.arange(P, device=DEV)).flatten(1)
            ok.scatter_(1, at.clamp(max=n), True)
            ok = ok[:, :n] & bits & (t <= pos)
            q = s["q"][r].double().reshape(H, G, D)
            p = _exact_softmax(torch.matmul(q, k) * s["scale"], ok[:, None])
            out[r] = torch.matmul(p, v).reshape(H * G, D)
    return {"blocks": blocks, "out": out}


def _exact_append(s):
    c = s["case"]
    lo, hi = LIMITS[c["elem"]]
    grid = torch.tensor(GRID, dtype=torch.float64, device=DEV)

    def held(x):
        x = x.double().reshape(*x.shape[:-1], -1, 32)
        big = x.abs().amax(-1, keepdim=True)
        e = torch.ceil(torch.log2(big / 6)).clamp(lo, hi)
        e = torch.where(big <= 6 * torch.pow(2.0, e - 1), e - 1, e).clamp(lo, hi)
        y = x.abs() / torch.pow(2.0, e)
        d = (y[..., None] - grid).abs()
        d = d - 1e-9 * (torch.arange(8, device=DEV) % 2 == 0)  # halfway: the even code
        y = grid[d.argmin(-1)] * torch.pow(2.0, e)
        return torch.where(x < 0, -y, y).flatten(-2)

    got = {"k": held(s["k"]), "v": held(s["v"])}
    return {**got, **{n: None for n in ("k_codes", "k_scales", "v_codes", "v_scales", "box", "box_scale")}}


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "select": _exact_select,
            "sparse": _exact_sparse}[case["kind"]](s)
