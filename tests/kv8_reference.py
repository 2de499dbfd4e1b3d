"""Plain 64-bit forms of the paged 8-bit cache, the attention over it and the
8-bit product, in numpy and written from include/moe_hip.h's description."""
import math

import numpy as np


def quantise(x):
    """[..., values] f32 -> codes int8, scales f32 [...], every step rounded to
    f32 (a quotient or product of two f32 rounded once from 64 bits is that)."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        top = np.abs(x).max(-1)
        bad, some = ~np.isfinite(top), np.isfinite(top) & (top >= np.float32(2.0 ** -100))
        t = np.where(some, top, np.float32(1)).astype(np.float64)
        inv = (127.0 / t).astype(np.float32)
        y = (x.astype(np.float64) * inv.astype(np.float64)[..., None]).astype(np.float32)
        code = np.where(some[..., None], np.rint(y), 0).astype(np.int8)  # (rint: halves to even)
        scale = np.where(some, (t / 127.0).astype(np.float32), np.where(bad, np.float32(np.nan), np.float32(0)))
    return code, scale.astype(np.float32)


class Cache8:
    """A pool's codes and scales, read and written by the documented addresses,
    and every sequence's values as they were stored."""

    def __init__(self, n_pages, n_kv, qd, vd, page, table):
        self.n_pages, self.n_kv, self.qd, self.vd, self.page, self.table = n_pages, n_kv, qd, vd, page, table
        tiles = n_pages * n_kv * (page // 64)
        self.codes = np.zeros((tiles, 64 * (qd + vd)), np.uint8)
        self.scales = np.zeros((tiles, 2, 4), np.float32)
        self.values = {}  # (sequence, position) -> (k [kv, qd], v [kv, vd])

    def _bytes(self, p, keys):
        """Offsets in a tile of position p's codes."""
        if keys:
            d = np.arange(self.qd)
            return (p // 16) * 16 * self.qd + d // 16 * 256 + p % 16 * 16 + d % 16
        d = np.arange(self.vd)
        return 64 * self.qd + d // 16 * 1024 + p % 16 // 4 * 256 + d % 16 * 16 + p // 16 * 4 + p % 4

    def tile(self, seq, pos, kv):
        return (int(self.table[seq, pos // self.page]) * self.n_kv + kv) * (self.page // 64) + pos % self.page // 64

    def put(self, seq, block):
        """Block `block` of a sequence, from the values of its positions so far."""
        there = [p for p in range(16 * block, 16 * block + 16) if (seq, p) in self.values]
        for keys, d in ((True, self.qd), (False, self.vd)):
            x = np.zeros((self.n_kv, 16, d), np.float32)
            for p in there:
                x[:, p % 16] = self.values[seq, p][0 if keys else 1]
            code, scale = quantise(x.reshape(self.n_kv, 16 * d))
            code = code.reshape(self.n_kv, 16, d)
            for kv in range(self.n_kv):
                t = self.tile(seq, 16 * block, kv)
                self.scales[t, 0 if keys else 1, block % 4] = scale[kv]
                for p in range(16):
                    self.codes[t, self._bytes(16 * (block % 4) + p, keys)] = code[kv, p].view(np.uint8)

    def store(self, rows, k, v):
        """rows: (sequence, position) or None of each row."""
        touched = set()
        for r, at in enumerate(rows):
            if at is None:
                continue
            s, p = at
            for q in [q for q in self.values if q[0] == s and q[1] >= p]:
                del self.values[q]
            self.values[s, p] = (k[r].reshape(self.n_kv, self.qd), v[r].reshape(self.n_kv, self.vd))
            touched.add((s, p // 16))
        for s, b in touched:
            self.put(s, b)

    def get(self, seq, pos, kv, keys):
        t = self.tile(seq, pos, kv)
        code = self.codes[t, self._bytes(pos % 64, keys)].view(np.int8).astype(np.float64)
        with np.errstate(all="ignore"):
            return code * np.float64(self.scales[t, 0 if keys else 1, pos % 64 // 16])

    def span(self, seq, n, keys):
        """Positions 0 .. n - 1, [n, kv, width], and which of them a page holds."""
        d = self.qd if keys else self.vd
        out, there = np.zeros((n, self.n_kv, d)), np.zeros(n, bool)
        for p in range(n):
            if p // self.page >= self.table.shape[1] or not 0 <= self.table[seq, p // self.page] < self.n_pages:
                continue
            there[p] = True
            for kv in range(self.n_kv):
                out[p, kv] = self.get(seq, p, kv, keys)
        return out, there


def attend(cache, q, seq, pos, heads, scale, window=0, out=None):
    """[rows, heads * vd] in 64 bits; rows that are none keep `out`'s."""
    n_seq = cache.table.shape[0]
    rep = heads // cache.n_kv
    out = np.zeros((len(seq), heads * cache.vd)) if out is None else out.astype(np.float64)
    last = {}
    for s, p in zip(seq, pos):
        if p >= 0 and 0 <= s < n_seq:
            last[s] = max(last.get(s, 0), p + 1)
    spans = {s: (cache.span(s, n, True), cache.span(s, n, False)) for s, n in last.items()}
    for r, (s, p) in enumerate(zip(seq, pos)):
        if p < 0 or not 0 <= s < n_seq:
            continue
        (k, there), (v, _) = spans[s]
        at = np.arange(p + 1)
        at = at[there[: p + 1] & ((at > p - window) if window > 0 else (at >= 0))]
        for h in range(heads):
            o = np.zeros(cache.vd)
            if len(at):
                with np.errstate(all="ignore"):
                    x = k[at, h // rep] @ q[r, h * cache.qd:(h + 1) * cache.qd].astype(np.float64) * scale
                    w = np.exp(x - x.max())
                    o = (w[:, None] * v[at, h // rep]).sum(0) / w.sum()
            out[r, h * cache.vd:(h + 1) * cache.vd] = o
    return out


def product(x, w):
    """y = x W^T in 8 bits: sums as whole numbers, the rest in 64 bits."""
    (cx, sx), (cw, sw) = quantise(x), quantise(w)
    with np.errstate(all="ignore"):
        return (cx.astype(np.int64) @ cw.astype(np.int64).T) * (sx.astype(np.float64)[:, None] * sw.astype(np.float64))
