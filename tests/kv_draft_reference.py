"""Drafts and cross attention over the 4-bit key/value cache in plain 64-bit
arithmetic, beside kv_reference (numpy)."""
from __future__ import annotations

import numpy as np

import kv_reference as ref


# ---- trees --------------------------------------------------------------------

def trees(new, seed=0, bad=0.0):
    """Parents of trees of so many tokens; `bad`: the share that name no token before them."""
    r = np.random.default_rng(seed)
    out = []
    for n in new:
        p = [int(r.integers(max(0, i // 2 - 3), i)) if i else -1 for i in range(n)]
        for i in range(n):
            if r.random() < bad:
                p[i] = int(r.choice([-1, -9, i, i + 1, n, 2 ** 31 - 1, -2 ** 31]))
        out += p
    return np.array(out, np.int32)


def parent_of(p: int, i: int) -> int:
    return p if 0 <= p < i else -1


def tree(new, parents):
    """sees [queries][largest draft] and depths [queries]."""
    sees = np.zeros((len(parents), max(new + [0])), bool)
    depths = np.zeros(len(parents), np.int32)
    at = 0
    for n in new:
        for i in range(n):
            j, d = i, -1
            while j >= 0:
                sees[at + i, j] = True
                j, d = parent_of(int(parents[at + j]), j), d + 1
            depths[at + i] = d
        at += n
    return sees, depths


def words(bits: np.ndarray, width=None) -> np.ndarray:
    """Truth values [rows][n] as i32 words [rows][width]."""
    n = -(-bits.shape[1] // 32) if width is None else width
    full = np.zeros((bits.shape[0], 32 * n), bool)
    full[:, :min(bits.shape[1], 32 * n)] = bits[:, :32 * n]
    full = full.reshape(bits.shape[0], n, 32)
    return np.packbits(full, axis=-1, bitorder="little").view(np.int32).reshape(bits.shape[0], n)


def accept(lens, new, parents, drafted, chosen, width):
    path = np.full((len(new), width), -1, np.int32)
    lengths, answer = np.zeros(len(new), np.int32), np.full(len(new), -1, np.int32)
    at = 0
    for b, n in enumerate(new):
        walk = [0] if n else []
        while walk and len(walk) < width:
            cur = walk[-1]
            nxt = [j for j in range(cur + 1, n) if parent_of(int(parents[at + j]), j) == cur
                   and drafted[at + j] == chosen[at + cur]]
            if not nxt:
                break
            walk.append(nxt[0])
        path[b, :len(walk)] = walk
        lengths[b] = max(0, lens[b] - n + len(walk))
        if walk:
            answer[b] = chosen[at + walk[-1]]
        at += n
    return path, lengths, answer


def keep(cache: ref.Cache, batch: ref.Batch, path):
    """The path's rows moved, all read before any is written, and boxes renewed."""
    moves, P = [], batch.page
    for b, n in enumerate(batch.new):
        start, count = batch.lens[b] - n, 0
        for i, at in enumerate(path[b]):
            if i >= n or at < 0 or at >= n or (i and at <= path[b][i - 1]):
                break
            count += 1
            src, dst = start + int(at), start + i
            if dst < 0 or src // P >= batch.width:
                continue
            sp, dp = batch.page_of(b, src // P), batch.page_of(b, dst // P)
            if sp >= 0 and dp >= 0:
                s = src % P
                moves.append((dp, dst % P, cache.k_codes[sp, :, s].copy(), cache.k_scales[sp, :, s].copy(),
                              cache.v_codes[sp, :, s // 8, :, s % 8].copy(),
                              cache.v_scales[sp, :, s // 8, :, s % 8].copy()))
        batch_stop = min(start + count, batch.width * P) if n else 0
        moves.append((b, max(start, 0), batch_stop))
    for m in moves:
        if len(m) == 6:
            dp, t, kc, ks, vc, vs = m
            cache.k_codes[dp, :, t], cache.k_scales[dp, :, t] = kc, ks
            cache.v_codes[dp, :, t // 8, :, t % 8], cache.v_scales[dp, :, t // 8, :, t % 8] = vc, vs
    for m in moves:
        if len(m) == 3:
            b, first, stop = m
            for j in range(first // P, -(-stop // P)):
                pid = batch.page_of(b, j)
                if pid >= 0:
                    cache.renew_box(pid, min(P, stop - j * P))


# ---- attention ----------------------------------------------------------------

def dense(cache: ref.Cache, batch: ref.Batch, b: int, n: int):
    """Keys and values [n][heads][dim] of sequence b's first n positions, and which have a page."""
    if n == 0:
        return np.zeros((0, cache.heads, cache.dim)), np.zeros((0, cache.heads, cache.dim)), np.zeros(0, bool)
    t = np.arange(n)
    pid = np.array([batch.page_of(b, j) for j in range(batch.width)] + [-1], int)
    pid = pid[np.minimum(t // batch.page, batch.width)]
    at, safe = t % batch.page, np.maximum(pid, 0)
    unpack = lambda x: np.stack((x & 15, x >> 4), -1).reshape(n, cache.heads, cache.dim)  # noqa: E731
    k = ref.values(unpack(cache.k_codes[safe, :, at]), cache.k_scales[safe, :, at].astype(int) - 127)
    vc = cache.v_codes[safe, :, at // 8, :, at % 8].reshape(n, cache.heads, cache.dim // 2)
    v = ref.values(unpack(vc), cache.v_scales[safe, :, at // 8, :, at % 8].astype(int) - 127)
    return k, v, pid >= 0


def attend(cache: ref.Cache, batch: ref.Batch, q: np.ndarray, scale, sees=None, blocks=None):
    """(out, lse, bound) as kv_reference.attend's, of a draft's tokens (`sees` [queries][n],
    missing columns clear) or, without, of tokens that are no part of their sequence."""
    H, D = cache.heads, cache.dim
    G = q.shape[1] // H
    out, lse, bound = np.zeros(q.shape), np.full(q.shape[:2], -np.inf), np.zeros(q.shape)
    u, row = ref.UNIT[cache.elem], 0
    for b, (n, m) in enumerate(zip(batch.lens, batch.new)):
        k, v, there = dense(cache, batch, b, n)
        if batch.visible is not None:
            seen = np.zeros(n, bool)
            w = min(n, batch.bits.shape[1])
            seen[:w] = batch.bits[b, :w]
            there = there & seen
        for i in range(m):
            ok = there.copy()
            if sees is not None:
                t = np.arange(n) - (n - m)
                named = (t >= 0) & (t < sees.shape[1])
                named[named] = sees[row + i, t[named]]
                ok &= (t < 0) | named
            for h in range(H):
                see = ok if blocks is None else ok & np.isin(np.arange(n) // batch.page, blocks[row + i, h])
                kk, vv = k[see, h], v[see, h]
                if not len(kk):
                    continue
                qs = q[row + i, h * G:(h + 1) * G]
                s = scale * (qs @ kk.T)
                top = s.max(-1, keepdims=True)
                p = np.exp(s - top)
                z = p.sum(-1, keepdims=True)
                lse[row + i, h * G:(h + 1) * G] = (top + np.log(z))[:, 0]
                p = p / z
                o = p @ vv
                mass = p @ np.abs(vv)
                # dim products summed in 32 bits, scaled, the maximum taken off, the
                # exponential's own; the weights and the result rounded to the type
                ds = (D + 8) * 2.0 ** -24 * scale * (np.abs(qs) @ np.abs(kk).T).max(-1, keepdims=True) + \
                    2.0 ** -21 * (1 + np.abs(s).max(-1, keepdims=True)) + len(kk) * 2.0 ** -24
                e = 1.02 * u * (mass + np.abs(o)) + 4 * ds * mass
                if cache.elem == "f16":
                    e += 2.0 ** -25 * (np.abs(vv).sum(0) + 1)
                out[row + i, h * G:(h + 1) * G], bound[row + i, h * G:(h + 1) * G] = o, e
        row += m
    return out, lse, bound


def scatter(cache: ref.Cache, seed=0, low=122, high=128):
    """Every page written with random codes under scales of [2^(low-127), 2^(high-128)]."""
    r = np.random.default_rng(seed)
    for name in ("k_codes", "v_codes"):
        getattr(cache, name)[:] = r.integers(0, 256, getattr(cache, name).shape)
    for name in ("k_scales", "v_scales"):
        getattr(cache, name)[:] = r.integers(low, high, getattr(cache, name).shape)
