"""The 4-bit key/value cache in plain 64-bit arithmetic: quantization, boxes,
block choice and attention, position by position (numpy, for small sizes)."""
from __future__ import annotations

import math

import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
LIMITS = {"bf16": (-125, 125), "f16": (-23, 13)}
UNIT = {"bf16": 2.0 ** -7 / 2, "f16": 2.0 ** -10 / 2}  # half a step of the type at 1


def quantize(x: np.ndarray, elem: str):
    """Codes [..][dim] and exponents [..][dim/32] of rows x (float64)."""
    lo, hi = LIMITS[elem]
    g = x.reshape(*x.shape[:-1], -1, 32)
    g = np.where(np.isnan(g), 0.0, g)
    fin = np.where(np.isinf(g), 0.0, np.abs(g))
    top = fin.max(-1)
    e = np.full(top.shape, lo)
    for i in np.ndindex(top.shape):
        if top[i] > 0:
            n = math.frexp(top[i])[1] - 4  # certainly too small
            while top[i] > 6 * 2.0 ** n:
                n += 1
            e[i] = min(max(n, lo), hi)
    y = np.abs(g) / np.exp2(e)[..., None]
    d = np.abs(np.minimum(y, 6)[..., None] - GRID)
    code = d.argmin(-1)
    # halfway between two: the even one
    nxt = np.minimum(code + 1, 7)
    tie = np.take_along_axis(d, nxt[..., None], -1)[..., 0] == d.min(-1)
    code = np.where(tie & (code % 2 == 1), nxt, code)
    code = code | (np.signbit(g).astype(int) << 3)
    return code.reshape(x.shape).astype(np.uint8), e.astype(int)


def values(code: np.ndarray, e: np.ndarray) -> np.ndarray:
    v = np.where(code & 8, -GRID[code & 7], GRID[code & 7])
    return (v.reshape(*code.shape[:-1], -1, 32) * np.exp2(e.astype(float))[..., None]).reshape(code.shape)


class Cache:
    """The arrays of a cache, written and read one position at a time."""

    def __init__(self, pages, heads, page, dim, elem, seed=0):
        r = np.random.default_rng(seed)
        self.pages, self.heads, self.page, self.dim, self.elem = pages, heads, page, dim, elem
        # What nobody wrote may hold anything, exponent bytes of infinity and NaN included.
        self.k_codes = r.integers(0, 256, (pages, heads, page, dim // 2), dtype=np.uint8)
        self.k_scales = r.choice(np.array([0, 120, 253, 254, 255], np.uint8), (pages, heads, page, dim // 32))
        self.v_codes = r.integers(0, 256, (pages, heads, page // 8, 16, 8, dim // 32), dtype=np.uint8)
        self.v_scales = r.choice(np.array([0, 120, 253, 254, 255], np.uint8),
                                 (pages, heads, page // 8, dim // 32, 8))
        self.box = r.integers(-128, 128, (pages, heads, 2, dim)).astype(np.int8)
        self.box_scale = r.integers(0, 256, (pages, heads), dtype=np.uint8)

    NAMES = ("k_codes", "k_scales", "v_codes", "v_scales", "box", "box_scale")

    def write(self, pid, at, k, v):
        """Row k, v [heads][dim] (float64) at position `at` of page pid; the values then held."""
        kc, ke = quantize(k, self.elem)
        vc, ve = quantize(v, self.elem)
        pack = lambda c: (c[:, 0::2] | (c[:, 1::2] << 4)).astype(np.uint8)  # noqa: E731
        self.k_codes[pid, :, at] = pack(kc)
        self.k_scales[pid, :, at] = ke + 127
        self.v_codes[pid, :, at // 8, :, at % 8] = pack(vc).reshape(self.heads, 16, -1)
        self.v_scales[pid, :, at // 8, :, at % 8] = ve + 127
        return values(kc, ke), values(vc, ve)

    def read(self, pid, at):
        """Key and value [heads][dim] at a position."""
        unpack = lambda b: np.stack((b & 15, b >> 4), -1).reshape(self.heads, -1)  # noqa: E731
        k = values(unpack(self.k_codes[pid, :, at]), self.k_scales[pid, :, at].astype(int) - 127)
        vb = self.v_codes[pid, :, at // 8, :, at % 8].reshape(self.heads, -1)
        v = values(unpack(vb), self.v_scales[pid, :, at // 8, :, at % 8].astype(int) - 127)
        return k, v

    def renew_box(self, pid, count):
        k = np.stack([self.read(pid, t)[0] for t in range(count)])
        hi, lo = k.max(0), k.min(0)
        for h in range(self.heads):
            top = max(np.abs(hi[h]).max(), np.abs(lo[h]).max())
            e = -125
            if top > 0:
                e = math.frexp(top)[1] - 9
                while top > 127 * 2.0 ** e:
                    e += 1
                e = min(max(e, -125), 125)
            self.box[pid, h, 0] = np.ceil(hi[h] * 2.0 ** -e)
            self.box[pid, h, 1] = np.floor(lo[h] * 2.0 ** -e)
            self.box_scale[pid, h] = e + 127


class Batch:
    """Sequences in pages of a pool: lengths, new tokens, holes and filters."""

    def __init__(self, page, lens, new, pages=None, seed=0, holes=0.0, visible=None, extra=1):
        r = np.random.default_rng(seed + 1)
        self.page, self.lens, self.new = page, list(lens), list(new)
        need = [-(-n // page) for n in lens]
        self.width = max(need + [0]) + extra
        self.pages = pages if pages is not None else sum(need) + 3
        order = r.permutation(self.pages)
        self.table = np.full((len(lens), self.width), -1, np.int32)
        n = 0
        for b, k in enumerate(need):
            self.table[b, :k] = order[(n + np.arange(k)) % self.pages]  # a smaller pool: pages shared
            n += k
        if holes:
            gone = r.random(self.table.shape) < holes
            self.table[gone] = r.choice(np.array([-1, -7, self.pages, 2 ** 31 - 1]), int(gone.sum()))
        self.offsets = np.concatenate(([0], np.cumsum(new))).astype(np.int32)
        self.queries = int(self.offsets[-1])
        words = (self.width * page + 31) // 32
        self.visible = None
        if visible is not None:
            bits = np.zeros((len(lens), words * 32), bool)
            for b, n in enumerate(lens):
                bits[b, :n] = visible(b, n, r)
            self.bits = bits
            self.visible = np.packbits(bits.reshape(len(lens), words, 32), axis=-1,
                                       bitorder="little").view(np.uint32)[..., 0].view(np.int32)

    def page_of(self, b, j):
        p = self.table[b, j]
        return p if 0 <= p < self.pages else -1

    def sees(self, b, t):
        return self.visible is None or self.bits[b, t]

    def tokens(self):
        """(row, sequence, position) of every token."""
        for b, n in enumerate(self.new):
            for i in range(n):
                yield self.offsets[b] + i, b, self.lens[b] - n + i


def fill(cache: Cache, batch: Batch, seed=0, magnitude=1.0):
    """Every position of every sequence but the new tokens' written, boxes renewed."""
    r = np.random.default_rng(seed + 2)
    for b, n in enumerate(batch.lens):
        for j in range(-(-n // batch.page)):
            pid = batch.page_of(b, j)
            if pid < 0:
                continue
            count = min(batch.page, n - j * batch.page)
            for t in range(count):
                shape = (cache.heads, cache.dim)
                cache.write(pid, t, magnitude * r.standard_normal(shape), r.standard_normal(shape))
            cache.renew_box(pid, count)


def _int8(q: np.ndarray):
    q = np.where(np.isnan(q), 0.0, q)
    fin = np.where(np.isinf(q), 0.0, np.abs(q)).max()
    e = min(max(math.frexp(fin)[1] - 7, -125), 125) if fin > 0 else -125
    return np.clip(np.rint(q * 2.0 ** -e), -127, 127), e


def select(cache: Cache, batch: Batch, q: np.ndarray, width, first, last):
    """Blocks [queries][kv_heads][width]; q [queries][heads][dim] float64."""
    H = cache.heads
    G = q.shape[1] // H
    out = np.full((q.shape[0], H, width), -1, np.int32)
    for row, b, pos in batch.tokens():
        blocks = pos // batch.page + 1 if pos >= 0 else 0
        for h in range(H):
            rows = [_int8(q[row, h * G + g]) for g in range(G)]
            ranked = []
            for j in range(min(blocks, batch.width)):
                pid = batch.page_of(b, j)
                end = min(pos + 1, (j + 1) * batch.page)
                if pid < 0 or not any(batch.sees(b, t) for t in range(j * batch.page, end)):
                    continue
                box = cache.box[pid, h].astype(np.int64)
                eb = int(cache.box_scale[pid, h]) - 127
                score = max(int(np.maximum(x * box[0], x * box[1]).sum()) * 2.0 ** (e + eb) for x, e in rows)
                forced = j < first or j >= blocks - last
                ranked.append((0 if forced else 1, -score if not forced else 0, j))
            got = sorted(j for _, _, j in sorted(ranked)[:width])
            out[row, h, :len(got)] = got
    return out


def attend(cache: Cache, batch: Batch, q: np.ndarray, scale, blocks=None):
    """(out, lse, bound) for q [queries][heads][dim] float64: the bound is what
    a kernel may be off that keeps its sums in 32 bits, rounds the weights and
    the result to the element type, and recomputes nothing."""
    H, D = cache.heads, cache.dim
    G = q.shape[1] // H
    out = np.zeros(q.shape)
    lse = np.full(q.shape[:2], -np.inf)
    bound = np.zeros(q.shape)
    u = UNIT[cache.elem]
    kv = {}
    for b, n in enumerate(batch.lens):
        ks, vs, at = [], [], []
        for t in range(min(n, batch.width * batch.page)):
            pid = batch.page_of(b, t // batch.page)
            if pid >= 0 and batch.sees(b, t):
                k, v = cache.read(pid, t % batch.page)
                ks.append(k)
                vs.append(v)
                at.append(t)
        kv[b] = (np.array(ks).reshape(-1, H, D), np.array(vs).reshape(-1, H, D), np.array(at, int))
    for row, b, pos in batch.tokens():
        k, v, at = kv[b]
        for h in range(H):
            ok = at <= pos
            if blocks is not None:
                ok &= np.isin(at // batch.page, blocks[row, h])
            kk, vv = k[ok, h], v[ok, h]
            if not len(kk):
                continue
            qs = q[row, h * G:(h + 1) * G]
            s = scale * (qs @ kk.T)
            m = s.max(-1, keepdims=True)
            p = np.exp(s - m)
            z = p.sum(-1, keepdims=True)
            lse[row, h * G:(h + 1) * G] = (m + np.log(z))[:, 0]
            p = p / z
            o = p @ vv
            out[row, h * G:(h + 1) * G] = o
            mass = p @ np.abs(vv)
            # A score's error: dim products summed in 32 bits, scaled, the
            # maximum taken off, and the exponential's own.
            ds = (D + 8) * 2.0 ** -24 * scale * (np.abs(qs) @ np.abs(kk).T).max(-1, keepdims=True) + \
                2.0 ** -21 * (1 + np.abs(s).max(-1, keepdims=True)) + len(kk) * 2.0 ** -24
            b_ = 1.02 * u * (mass + np.abs(o)) + 4 * ds * mass
            if cache.elem == "f16":  # weights and results below the normal range
                b_ += 2.0 ** -25 * (np.abs(vv).sum(0) + 1)
            bound[row, h * G:(h + 1) * G] = b_
    return out, lse, bound
