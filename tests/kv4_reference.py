"""Plain 64-bit forms of the paged 4-bit cache and the attention over it, in
numpy and written from include/moe_hip.h's description, position by position."""
import math

import numpy as np


def quantise(x):
    """[..., 32 n] f32 -> codes uint8 0..15, scales f16 [..., n], every step
    rounded to f32 as quant::quantize does (src/quant.rs:304-365)."""
    v = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, 32)
    with np.errstate(all="ignore"):
        d = (np.nanmax(np.abs(np.where(np.isnan(v), 0, v)), -1) / np.float32(7)).astype(np.float32)
        h = np.where(d < 65520, d, np.inf).astype(np.float16)  # no value here lies on a tie of a subnormal
        inv = np.where(d > 0, np.float32(1) / h.astype(np.float32), np.float32(0)).astype(np.float32)
        y = (v * inv[..., None]).astype(np.float64)
        code = np.sign(y) * np.floor(np.abs(y) + 0.5) + 8
        code = np.where(np.isnan(code), 8, np.clip(code, 0, 15)).astype(np.uint8)
    return code.reshape(x.shape), h


def value(code, h):
    """The value a code and a scale stand for, in 64 bits."""
    with np.errstate(all="ignore"):
        return np.repeat(h.astype(np.float64), 32, -1) * (code.astype(np.float64) - 8)


class Pool:
    """A pool's bytes (numpy), read and written by the documented addresses."""

    def __init__(self, n_pages, n_kv, qd, vd, page, raw=None):
        self.n_pages, self.n_kv, self.qd, self.vd, self.page = n_pages, n_kv, qd, vd, page
        self.tile = 18 * (qd + vd)
        size = n_pages * n_kv * (page // 32) * self.tile
        self.raw = np.zeros(size, np.uint8) if raw is None else raw
        assert self.raw.size == size

    def _at(self, slot, kv):
        pg, off = divmod(int(slot), self.page)
        return ((pg * self.n_kv + kv) * (self.page // 32) + off // 32) * self.tile, off % 32

    def _bytes(self, p, keys):
        """Offsets in a tile of [block][j] code bytes and [block] scales of position p."""
        d = self.qd if keys else self.vd
        code, scale = np.zeros((d // 32, 16), np.int64), np.zeros(d // 32, np.int64)
        for b in range(d // 32):
            w = 2 * b + p // 16
            words = 2 * (d // 32)
            width = min(4, words - w // 4 * 4)  # words a lane has in this chunk
            for j in range(16):
                lane, byte = (16 * (j // 4) + p % 16, j % 4) if keys else (16 * (p % 16 // 4) + j, p % 4)
                code[b, j] = (0 if keys else 16 * self.qd) + w // 4 * 1024 + lane * 4 * width + w % 4 * 4 + byte
            base = 16 * (self.qd + self.vd) if keys else 18 * self.qd + 16 * self.vd
            scale[b] = base + 2 * (32 * b + 8 * (p % 16 // 4) + 4 * (p // 16) + p % 4)
        return code, scale

    def put(self, slot, kv, code, h, keys):
        at, p = self._at(slot, kv)
        cb, sb = self._bytes(p, keys)
        c = code.reshape(-1, 32)
        self.raw[at + cb] = c[:, :16] | c[:, 16:] << 4
        two = np.ascontiguousarray(h).view(np.uint8).reshape(-1, 2)
        self.raw[at + sb], self.raw[at + sb + 1] = two[:, 0], two[:, 1]

    def get(self, slot, kv, keys):
        at, p = self._at(slot, kv)
        cb, sb = self._bytes(p, keys)
        b = self.raw[at + cb]
        code = np.concatenate([b & 15, b >> 4], -1).reshape(-1)
        h = np.stack([self.raw[at + sb], self.raw[at + sb + 1]], -1).copy().view(np.float16)[..., 0]
        return value(code, h)

    def store(self, slots, k, v):
        for r, slot in enumerate(slots):
            if not 0 <= slot < self.n_pages * self.page:
                continue
            for x, keys, d in ((k, True, self.qd), (v, False, self.vd)):
                code, h = quantise(x[r].reshape(self.n_kv, d))
                for kv in range(self.n_kv):
                    self.put(slot, kv, code[kv], h[kv], keys)

    def mean(self, page):
        with np.errstate(all="ignore"):
            m = np.stack([np.mean([self.get(page * self.page + i, kv, True) for i in range(self.page)], 0)
                          for kv in range(self.n_kv)])
            return np.clip(m, -65504, 65504).astype(np.float32).astype(np.float16)


def attend(pool, table, q, seq, pos, heads, scale, window=0, lists=None, out=None):
    """[rows, heads * vd] in 64 bits; rows that are none keep `out`'s."""
    n_kv, qd, vd, P = pool.n_kv, pool.qd, pool.vd, pool.page
    rep = heads // n_kv
    out = np.zeros((len(seq), heads * vd)) if out is None else out.astype(np.float64)
    cache = {}

    def read(s, page, kv):
        if (s, page, kv) not in cache:
            slot = int(table[s, page]) * P
            cache[s, page, kv] = [np.stack([pool.get(slot + i, kv, keys) for i in range(P)]) for keys in (True, False)]
        return cache[s, page, kv]

    for r, (s, top) in enumerate(zip(seq, pos)):
        if top < 0 or not 0 <= s < table.shape[0]:
            continue
        lo = max(0, top + 1 - window) if window else 0
        for kv in range(n_kv):
            pages = range(lo // P, top // P + 1)
            if lists is not None:
                pages, before = [], -1
                for p in lists[r, kv]:
                    if p > before:
                        pages.append(int(p))
                    before = int(p)
            ks, vs = [], []
            for p in pages:
                if p >= table.shape[1] or not 0 <= table[s, p] < pool.n_pages:
                    continue
                at = np.arange(p * P, (p + 1) * P)
                see = (at >= lo) & (at <= top)
                if see.any():
                    k, v = read(s, p, kv)
                    ks.append(k[see])
                    vs.append(v[see])
            for h in range(kv * rep, (kv + 1) * rep):
                if not ks:
                    out[r, h * vd:(h + 1) * vd] = 0
                    continue
                with np.errstate(all="ignore"):
                    w = np.concatenate(ks) @ q[r, h * qd:(h + 1) * qd].astype(np.float64) * scale
                    w = np.exp(w - w.max())
                    out[r, h * vd:(h + 1) * vd] = (w / w.sum()) @ np.concatenate(vs)
    return out


def select(means, table, q, seq, pos, heads, page, n_sel, sinks, recent):
    """[rows, n_kv, n_sel] int32."""
    n_pages, n_kv, qd = means.shape
    rep = heads // n_kv
    out = np.full((len(seq), n_kv, n_sel), -1, np.int32)
    for r, (s, top) in enumerate(zip(seq, pos)):
        if top < 0 or not 0 <= s < table.shape[0]:
            continue
        cur = top // page
        for kv in range(n_kv):
            def score(p):
                if p < sinks or p > cur - recent:
                    return math.inf
                if not 0 <= table[s, p] < n_pages:
                    return -math.inf
                with np.errstate(all="ignore"):
                    v = [float(q[r, h * qd:(h + 1) * qd].astype(np.float64) @ means[table[s, p], kv].astype(np.float64))
                         for h in range(kv * rep, (kv + 1) * rep)]
                v = [x for x in v if not math.isnan(x)]
                return max(v) if v else -math.inf
            pick = sorted(sorted(range(cur + 1), key=lambda p: (-score(p), p))[:n_sel])
            out[r, kv, :len(pick)] = pick
    return out


def advance(length, add, table, ring, state, page, max_rows):
    """moe_pages_advance sequence by sequence, in place; the rows as lists."""
    n, cap = len(length), table.shape[1] * page
    head, count = int(state[0]), int(state[1])
    status, start, seq, pos, slot = [0] * n, [0], [], [], []
    rows = wanted = taken = 0
    back = []
    new = length.copy()
    for i in range(n):
        have = min(max(int(length[i]), 0), cap)
        a = int(add[i])
        new[i] = have
        got = 0
        if a < 0:
            back += [int(x) for x in table[i, :-(-have // page)]]
            new[i] = 0
        elif have + a > cap:
            status[i] = 2
        else:
            rows += a
            need = -(-(have + a) // page) - -(-have // page)
            if a > 0 and rows > max_rows:
                status[i] = 3
            else:
                wanted += need
                if need > 0 and wanted > count:
                    status[i] = 1
                else:
                    for j in range(-(-have // page), -(-(have + a) // page)):
                        table[i, j] = ring[(head + taken) % len(ring)]
                        taken += 1
                    got, new[i] = a, have + a
        for p in range(have, have + got):
            seq.append(i)
            pos.append(p)
            slot.append(int(table[i, p // page]) * page + p % page)
        start.append(len(seq))
    for j, x in enumerate(back):
        ring[(head + count + j) % len(ring)] = x
    pad = max_rows - len(seq)
    return dict(length=new, state=np.array([(head + taken) % len(ring), count - taken + len(back)], np.int32),
                row_start=start, seq=seq + [-1] * pad, pos=pos + [-1] * pad, slot=slot + [-1] * pad, status=status)
