"""The paged 4-bit key/value cache and the attention over it, as cases that can be timed and compared.

Four kinds of case:

  pages    PageTable.advance: block tables and slot maps from request lengths
  store    KvCache.store, then KvCache.load of the rows just written
  attend   KvCache.attend: causal attention over the cache, many sequences at
           once, one new row each (decode) or runs of rows (prompts, chunks)
  sparse   KvCache.select, then KvCache.attend over the pages it chose

The cache.  32 values of a head share an f16 scale d = max|v| / 7 and are held
as codes round(v / d) + 8 in 0..15.  A page is `page` positions of all kv
heads, a multiple of 32; a tile is 32 positions of one kv head,

  [page][kv head][page / 32 tiles][tile: 18 (qd + vd) bytes]

and a tile holds, in this order, the keys' codes (16 qd bytes), the values'
codes (16 vd), the keys' scales (2 qd) and the values' scales (2 vd):

  codes    words of 4 bytes, word w of lane l (64 lanes): words 4c..4c+3 of all
           lanes are chunk c, 16 bytes a lane (8 in the last chunk of an odd
           number of blocks).  Block b (32 dims), positions 0..15 or 16..31
           (half): w = 2 b + half.
           keys:   lane 16 (j / 4) + p % 16, byte j % 4, j = 0..15: dims j (low
                   four bits) and j + 16 of position p
           values: lane 16 (p % 16 / 4) + j, byte p % 4: dims j and j + 16 of
                   position p
  scales   f16 [block][p % 16 / 4][half][p % 4]

A page that is full has the mean of its keys in `means` [page][kv head][qd],
f16.
"""
import math

import torch

own = False

DEV = "cuda:0"

# (query heads, kv heads, key width, value width)
TINY = (8, 2, 64, 64)          # tiny Mixtral
LATENT = (16, 16, 192, 128)    # V2-Lite's expanded latent cache
GROUPED = (32, 8, 128, 128)    # four query heads to a kv head
HEADS = [TINY, LATENT, GROUPED, (32, 4, 128, 128), (6, 2, 96, 96), (40, 1, 64, 32), (4, 2, 256, 256)]


# ------------------------------------------------------------------ the cases


def _heads(h):
    return {"heads": h[0], "kv_heads": h[1], "qd": h[2], "vd": h[3]}


def listed():
    return [
        # A decode step's tables: every sequence one token further.
        {"name": "pages_decode", "kind": "pages", "seqs": 32, "page": 64, "max_pages": 64, "rows": 32, "prompts": 0,
         "released": 0},
        # A large server's step: thousands of sequences, most of them decoding, some with a prompt (more rows than
        # there is room for), some finished.
        {"name": "pages_large", "kind": "pages", "seqs": 4096, "page": 64, "max_pages": 256, "rows": 100000,
         "prompts": 128, "released": 100},
        # A decode step's rows.
        dict(_heads(GROUPED), name="store_decode", kind="store", seqs=32, new=1, past=1500, page=64),
        # Prompts of a latent-attention model, a length off every tile.
        dict(_heads(LATENT), name="store_prompts", kind="store", seqs=3, new=333, past=45, page=32),
        # The largest write: a batch of long prompts.
        dict(_heads(GROUPED), name="store_large", kind="store", seqs=8, new=2047, past=0, page=64),
        # The smallest call: a few sequences of a small model decode.
        dict(_heads(TINY), name="attend_small", kind="attend", seqs=4, new=1, past=96, page=64, window=0, pad=0),
        # Batched decode of a latent-attention model; the launch is sized for more rows than there are.
        dict(_heads(LATENT), name="attend_decode", kind="attend", seqs=32, new=1, past=1200, page=64, window=0, pad=4),
        # One user far into a long context: the position axis is all the parallelism there is.
        dict(_heads(GROUPED), name="attend_one_long", kind="attend", seqs=1, new=1, past=100001, page=64, window=0,
             pad=0),
        # A prompt of ordinary length.
        dict(_heads(GROUPED), name="attend_prompt", kind="attend", seqs=1, new=2000, past=0, page=64, window=0, pad=0),
        # The largest decode step: many sequences, long contexts.
        dict(_heads(GROUPED), name="attend_batch_long", kind="attend", seqs=64, new=1, past=12000, page=128, window=0,
             pad=0),
        # Long contexts read through the pages that each query chooses: 16 of up to 500.
        dict(_heads(GROUPED), name="sparse_decode", kind="sparse", seqs=32, new=1, past=32000, page=64, select=16,
             sinks=1, recent=2),
        # A chunk of a prompt far into one sequence: every row chooses for itself.
        dict(_heads(GROUPED), name="sparse_chunk", kind="sparse", seqs=1, new=61, past=70000, page=64, select=32,
             sinks=1, recent=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["pages", "store", "attend", "attend", "attend", "sparse", "sparse"])
    page = rng.choice([32, 64, 64, 128])
    if kind == "pages":
        seqs = _log(rng, 1, 4000)
        prompts = rng.randint(0, max(1, seqs // 16))
        return {"kind": "pages", "seqs": seqs, "page": page, "max_pages": rng.randint(8, 250),
                "rows": seqs + _log(rng, 1, 400) * prompts, "prompts": prompts, "released": rng.randint(0, seqs // 8)}
    h = rng.choice(HEADS)
    c = dict(_heads(h), kind=kind, page=page)
    if kind == "store":
        seqs = _log(rng, 1, 64)
        return dict(c, seqs=seqs, new=_log(rng, 1, 8000 // seqs), past=rng.randint(0, 1000))
    if kind == "sparse":
        seqs = _log(rng, 1, 24)
        sel = rng.randint(5, 32)
        return dict(c, seqs=seqs, new=_log(rng, 1, max(1, 40 // seqs)), past=_log(rng, 1000, 600000 // seqs // page * 32),
                    select=sel, sinks=rng.randint(0, 2), recent=rng.randint(1, 3))
    c.update(window=_log(rng, 16, 512) if rng.random() < 0.25 else 0, pad=rng.choice([0, 0, 3]))
    how = rng.randrange(3)
    if how == 0:    # decode
        seqs = _log(rng, 1, 64)
        c.update(seqs=seqs, new=1, past=_log(rng, 1, min(60000, 500000 // seqs)))
    elif how == 1:  # prompts
        c.update(seqs=rng.randint(1, 4), new=_log(rng, 2, 1500), past=0)
    else:           # chunks of prompts behind a longer past
        c.update(seqs=rng.randint(1, 8), new=_log(rng, 2, 128), past=_log(rng, 1, 6000))
    return c


def _pasts(c):
    """How far each sequence is: from half of `past` to all of it."""
    n, p = c["seqs"], c["past"]
    return [p - (p // 2) * ((5 * i) % n) // n for i in range(n)]


def work(c):
    if c["kind"] == "pages":
        # lengths, what is added and the state in; rows, tables' new entries and the new state out
        return {"bytes": 24 * c["seqs"] + 16 * c["rows"] + 4 * c["rows"] // c["page"], "flops": 0}
    h, kv, qd, vd, new = c["heads"], c["kv_heads"], c["qd"], c["vd"], c["new"]
    rows = c["seqs"] * new
    if c["kind"] == "store":
        # rows in, codes and scales out and in again, rows out
        return {"bytes": rows * kv * (qd + vd) * (4 + 18 / 32 + 18 / 32 + 4), "flops": 0}
    qo = 4 * rows * h * (qd + vd)
    if c["kind"] == "sparse":
        pages = sum((p + new) // c["page"] for p in _pasts(c))
        at = rows * c["select"] * c["page"]
        return {"bytes": qo + pages * kv * qd * 2 + min(at, sum(p + new for p in _pasts(c))) * kv * (qd + vd) * 18 / 32,
                "flops": 2 * h * qd * pages * new + 2 * at * h * (qd + vd)}
    w = c["window"]
    seen = sum(min(p + new, w + new - 1) if w else p + new for p in _pasts(c))
    pairs = sum(sum(min(p + i + 1, w) if w else p + i + 1 for i in range(new)) for p in _pasts(c))
    return {"bytes": qo + seen * kv * (qd + vd) * 18 / 32, "flops": 2 * pairs * h * (qd + vd)}


# ----------------------------------------------------------- the cache's layout


def _tables(d, keys, at):
    """Byte of a tile at which [position 0..31][block][j 0..15] lies, and f16 at which [position][block]'s scale does."""
    nb = d // 32
    p = torch.arange(32, device=DEV).view(32, 1, 1)
    b = torch.arange(nb, device=DEV).view(1, nb, 1)
    j = torch.arange(16, device=DEV).view(1, 1, 16)
    w = 2 * b + p // 16
    lane, byte = (16 * (j // 4) + p % 16, j % 4) if keys else (16 * (p % 16 // 4) + j, p % 4)
    width = torch.where(w // 4 < nb // 2, 16, 8)
    code = at[0] + w // 4 * 1024 + lane * width + w % 4 * 4 + byte
    scale = at[1] // 2 + (b * 32 + p % 16 // 4 * 8 + p // 16 * 4 + p % 4)[..., 0]
    return code, scale


def _layout(c):
    qd, vd = c["qd"], c["vd"]
    return (_tables(qd, True, (0, 16 * (qd + vd))), _tables(vd, False, (16 * qd, 18 * qd + 16 * vd)))


def _values(tiles, table, d):
    """[..., tile bytes] -> [..., 32, d] f32."""
    code, scale = table
    b = tiles[..., code]
    v = torch.cat([b & 15, b >> 4], -1).float() - 8.0
    v = v * tiles.view(torch.float16)[..., scale].float()[..., None]
    return v.reshape(*tiles.shape[:-1], 32, d)


def _quantise(x):
    """[..., d] f32 -> bytes [..., d / 32, 16], scales f16 [..., d / 32]."""
    v = x.reshape(*x.shape[:-1], -1, 32)
    # Every step is rounded to 32 bits (a quotient by way of 64): the stored code is defined by them.
    d = (v.abs().amax(-1).double() / 7.0).float()
    h = d.half()
    inv = torch.where(d > 0, (1.0 / h.double()).float(), torch.zeros_like(d))
    y = (v * inv[..., None]).double()
    q = (torch.sign(y) * torch.floor(y.abs() + 0.5)).clamp(-8, 7).to(torch.uint8) + 8 & 15
    return q[..., :16] | q[..., 16:] << 4, h


# ------------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _prepare_pages(c, seed):
    g = _gen(seed)
    n, P, mp = c["seqs"], c["page"], c["max_pages"]
    ints = lambda lo, hi, k: torch.randint(lo, hi, (k,), generator=g, device=DEV, dtype=torch.int32)  # noqa: E731
    length = ints(0, mp * P // 2, n)
    add = torch.ones_like(length)
    order = torch.randperm(n, generator=g, device=DEV)
    k = c["prompts"]
    room = max(2, 2 * (c["rows"] - n) // max(k, 1))
    add[order[:k]] = ints(1, room + 1, k)
    add[order[k:k + c["released"]]] = -1
    add[order[k + c["released"]:][: n // 20]] = 0
    pages = (length + P - 1) // P
    first = torch.cumsum(pages, 0) - pages
    free = c["rows"] // P + n // 2
    n_pages = n * ((mp + 1) // 2) + free
    ids = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    col = torch.arange(mp, device=DEV)
    table = torch.where(col < pages[:, None], ids[(first[:, None] + col).clamp(max=n_pages - 1)], -1).to(torch.int32)
    # the free pages' ring starts somewhere and wraps
    head = int(torch.randint(0, n_pages, (1,), generator=g, device=DEV))
    ring = torch.full((n_pages,), -1, dtype=torch.int32, device=DEV)
    ring[(head + torch.arange(free, device=DEV)) % n_pages] = ids[n_pages - free:]
    new = lambda k, t=torch.int32: torch.empty(k, dtype=t, device=DEV)  # noqa: E731
    return {"case": c, "length": length, "add": add, "table": table, "ring": ring,
            "state": torch.tensor([head, free], dtype=torch.int32, device=DEV),
            "out": {"length": new(n), "state": new(2), "row_start": new(n + 1), "status": new(n), "seq": new(c["rows"]),
                    "pos": new(c["rows"]), "slot": new(c["rows"], torch.int64)}}


def _prepare_cache(c, seed):
    """A cache filled up to each sequence's past and new rows: sequences' pages scattered over the pool."""
    g = _gen(seed)
    P, kv, qd, vd, new = c["page"], c["kv_heads"], c["qd"], c["vd"], c["new"]
    n, pasts = c["seqs"], _pasts(c)
    pages = [(p + new + P - 1) // P for p in pasts]
    mp = max(pages) + 1
    n_pages = sum(pages) + 3
    ids = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((n, mp), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, k in enumerate(pages):
        table[i, :k] = ids[at:at + k]
        at += k
    tiles = n_pages * kv * (P // 32)
    tb = 18 * (qd + vd)
    pool = torch.empty((tiles, tb), dtype=torch.uint8, device=DEV)
    # Codes as N(0, 1) values get them (the largest of 32 at 7), scales about a third.
    nc = 16 * (qd + vd)
    step = max(1, (1 << 27) // nc)
    for t in range(0, tiles, step):
        k = min(step, tiles - t)
        z = lambda: (torch.randn((k, nc), generator=g, device=DEV) * 3.1).round_().clamp_(-7, 7).add_(8).to(torch.uint8)  # noqa: E731
        pool[t:t + k, :nc] = z() | z() << 4
    pool.view(torch.float16)[:, nc // 2:] = (torch.rand((tiles, tb // 2 - nc // 2), generator=g, device=DEV) * 0.2 + 0.25).half()
    pos = torch.cat([torch.arange(p, p + new) for p in pasts] + [torch.full((c.get("pad", 0),), -1)])
    seq = torch.cat([torch.full((new,), i) for i in range(n)] + [torch.zeros(c.get("pad", 0), dtype=torch.int64)])
    st = {"case": c, "pool": pool, "table": table, "pos": pos.to(DEV, torch.int32), "seq": seq.to(DEV, torch.int32),
          "max_pos": max(pasts) + new - 1, "pages": n_pages}
    return st, g


def prepare(case, seed):
    c = dict(case)
    if c["kind"] == "pages":
        return _prepare_pages(c, seed)
    st, g = _prepare_cache(c, seed)
    rows, kv, qd, vd, P = len(st["pos"]), c["kv_heads"], c["qd"], c["vd"], c["page"]
    normal = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    if c["kind"] == "store":
        # Keys and values of differing size, some rows far larger.
        big = torch.exp(normal(rows, 1))
        st["k"], st["v"] = normal(rows, kv * qd) * big, normal(rows, kv * vd) * big
        page = st["table"][st["seq"].long(), (st["pos"] // P).long()].long()
        st["slot"] = page * P + st["pos"] % P
        st["means"] = torch.zeros((st["pages"], kv, qd), dtype=torch.float16, device=DEV)
        st["k_out"], st["v_out"] = torch.empty_like(st["k"]), torch.empty_like(st["v"])
        return st
    # Queries sharp enough that some positions matter more than most.
    st["q"] = normal(rows, c["heads"] * qd) * 2.0
    st["scale"] = qd ** -0.5
    st["out"] = torch.zeros((rows, c["heads"] * vd), device=DEV)
    if c["kind"] == "sparse":
        st["means"] = (normal(st["pages"], kv, qd) * 0.3).half()
        st["lists"] = torch.empty((rows, kv, c["select"]), dtype=torch.int32, device=DEV)
    return st


# ------------------------------------------------------------- the plain forms


def _plain_pages(st):
    c, o = st["case"], st["out"]
    P, R = c["page"], c["rows"]
    L, a = st["length"].long(), st["add"].long()
    table, ring = st["table"], st["ring"]
    n, mp = table.shape
    n_pages = ring.numel()
    head, count = st["state"][0].long(), st["state"][1].long()
    gone = a < 0
    status = torch.zeros_like(L)
    fits = ~gone & (L + a <= mp * P)
    status = torch.where(~gone & ~fits, 2, status)
    rows = torch.where(fits, a, 0)
    roomy = fits & ~((rows > 0) & (torch.cumsum(rows, 0) > R))
    status = torch.where(fits & ~roomy, 3, status)
    old = (L + P - 1) // P
    need = torch.where(roomy, (L + a + P - 1) // P - old, 0)
    fed = roomy & ~((need > 0) & (torch.cumsum(need, 0) > count))
    status = torch.where(roomy & ~fed, 1, status)
    need = torch.where(fed, need, 0)
    first = torch.cumsum(need, 0) - need
    rows = torch.where(fed, a, 0)
    ends = torch.cumsum(rows, 0)
    r = torch.arange(R, device=DEV)
    s = torch.searchsorted(ends, r, right=True).clamp(max=n - 1)
    there = r < ends[-1]
    pos = L[s] + r - (ends - rows)[s]
    col = torch.arange(mp, device=DEV)
    fresh = (col >= old[:, None]) & (col < (old + need)[:, None])
    new_table = torch.where(fresh, ring[(head + first[:, None] + col - old[:, None]) % n_pages], table)
    # pages of the sequences that are gone go to the ring's end
    back = torch.where(gone, old, 0)
    upto = torch.cumsum(back, 0)
    k = (torch.arange(n_pages, device=DEV) - head - count) % n_pages
    who = torch.searchsorted(upto, k, right=True).clamp(max=n - 1)
    given = table[who, (k - (upto - back)[who]).clamp(0, mp - 1)]
    ring.copy_(torch.where(k < upto[-1], given, ring))
    table.copy_(new_table)
    slot = table[s, (pos // P).clamp(0, mp - 1)].long() * P + pos % P
    o["seq"].copy_(torch.where(there, s, -1))
    o["pos"].copy_(torch.where(there, pos, -1))
    o["slot"].copy_(torch.where(there, slot, -1))
    o["row_start"][0] = 0
    o["row_start"][1:] = ends
    o["status"].copy_(status)
    o["length"].copy_(torch.where(gone, 0, torch.where(fed, L + a, L)))
    took = need.sum()
    o["state"][0] = (head + took) % n_pages
    o["state"][1] = count - took + upto[-1]
    return [table, ring, o]


def _tile_of(c, slot):
    """[rows] slots -> tile index [rows, kv heads], position in the tile [rows]."""
    P, kv = c["page"], c["kv_heads"]
    head = torch.arange(kv, device=DEV)
    return (slot[:, None] // P * kv + head) * (P // 32) + (slot % P // 32)[:, None], slot % 32


def _plain_store(st):
    c = st["case"]
    kv, qd, vd, P = c["kv_heads"], c["qd"], c["vd"], c["page"]
    slot, pool = st["slot"], st["pool"]
    rows = slot.numel()
    lay = _layout(c)
    tile, p = _tile_of(c, slot)
    flat, halves = pool.view(-1), pool.view(torch.float16).view(-1)
    for name, (code, scale), d in (("k", lay[0], qd), ("v", lay[1], vd)):
        b, h = _quantise(st[name].view(rows, kv, d))
        flat[(tile * pool.shape[1])[..., None, None] + code[p][:, None]] = b
        halves[(tile * (pool.shape[1] // 2))[..., None] + scale[p][:, None]] = h
    # means of the pages whose last position was written (the others keep theirs)
    full = (slot % P == P - 1)[:, None, None]
    keys = _values(pool.view(st["pages"], kv, P // 32, -1)[slot // P], lay[0], qd)
    mean = keys.double().sum((2, 3)) / P
    mean = mean.clamp(-65504.0, 65504.0).float().half()
    # rows of one page would write one mean over another: only the last position's row may
    keep = torch.full((st["pages"],), -1, device=DEV).scatter_reduce(
        0, slot // P, torch.where(full[:, 0, 0], torch.arange(rows, device=DEV), -1), "amax")
    st["means"].copy_(torch.where((keep >= 0)[:, None, None], mean[keep.clamp(min=0)], st["means"]))
    for name, table, d in (("k", lay[0], qd), ("v", lay[1], vd)):
        x = _values(pool[tile], table, d)
        at = p[:, None, None, None].expand(-1, kv, 1, d)
        st[name + "_out"].copy_(x.gather(2, at).view(rows, kv * d))
    return [st["k_out"], st["v_out"], st["means"]]


def _softmax_product(s, v):
    e = torch.exp(s - s.amax(-1, keepdim=True))
    return torch.matmul(e, v) / e.sum(-1, keepdim=True)


def _plain_attend(st):
    c = st["case"]
    n, new, kv, qd, vd, P, h = (c[k] for k in ("seqs", "new", "kv_heads", "qd", "vd", "page", "heads"))
    rep = h // kv
    lay = _layout(c)
    tiles = st["pool"].view(st["pages"], kv, P // 32, -1)[st["table"][:, :-1].clamp(min=0).long()]
    tiles = tiles.transpose(1, 2)  # [seq, kv, page, tile, bytes]
    k = _values(tiles, lay[0], qd).reshape(n, kv, -1, qd)
    kt = k.transpose(2, 3).contiguous()
    del k
    pos = st["pos"][: n * new].view(n, 1, 1, new, 1)
    q = st["q"][: n * new].view(n, new, kv, rep, qd).permute(0, 2, 3, 1, 4).reshape(n, kv, rep * new, qd)
    s = torch.matmul(q, kt) * st["scale"]
    del kt
    at = torch.arange(s.shape[-1], device=DEV)
    seen = at <= pos
    if c["window"]:
        seen = seen & (at > pos - c["window"])
    s = torch.where(seen, s.view(n, kv, rep, new, -1), -math.inf).view(n, kv, rep * new, -1)
    v = _values(tiles, lay[1], vd).reshape(n, kv, -1, vd)
    o = _softmax_product(s, v).view(n, kv, rep, new, vd).permute(0, 3, 1, 2, 4)
    st["out"][: n * new] = o.reshape(n * new, h * vd)
    return [st["out"]]


def _plain_sparse(st):
    c = st["case"]
    kv, qd, vd, P, h, m = (c[k] for k in ("kv_heads", "qd", "vd", "page", "heads", "select"))
    rep, rows = h // kv, c["seqs"] * c["new"]
    lay = _layout(c)
    table = st["table"].clamp(min=0).long()[st["seq"].long()]  # [row, page]
    q = st["q"].view(rows, kv, rep, qd)
    # The choice between near scores is a border: 64 bits.
    means = st["means"][table].double()  # [row, page, kv, qd]
    score = torch.matmul(q.double(), means.permute(0, 2, 3, 1).contiguous()).amax(2)
    j = torch.arange(table.shape[1], device=DEV)
    cur = (st["pos"] // P)[:, None, None]
    score = torch.where((j < c["sinks"]) | (j > cur - c["recent"]), math.inf, score)
    score = torch.where(j <= cur, score, -math.inf)
    pick = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :m]
    pick = torch.sort(torch.where(pick <= cur, pick, 1 << 30), dim=-1).values
    lists = st["lists"]
    if pick.shape[-1] < m:
        lists.fill_(-1)
    lists[..., : pick.shape[-1]] = torch.where(pick < 1 << 30, pick, -1)
    page = table.gather(1, lists.clamp(min=0).long().view(rows, -1)).view(rows, kv, m)
    tiles = st["pool"].view(st["pages"], kv, P // 32, -1)[page, torch.arange(kv, device=DEV)[:, None]]
    k = _values(tiles, lay[0], qd).reshape(rows, kv, m * P, qd)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * st["scale"]
    at = (lists.long()[..., None] * P + torch.arange(P, device=DEV)).view(rows, kv, 1, m * P)
    s = torch.where((at >= 0) & (at <= st["pos"][:, None, None, None]), s, -math.inf)
    v = _values(tiles, lay[1], vd).reshape(rows, kv, m * P, vd)
    st["out"].copy_(_softmax_product(s, v).view(rows, h * vd))
    return [lists, st["out"]]


# ------------------------------------------------------------- the framework's


def _own(st):
    """The handles a program keeps beside its buffers."""
    from moe_amd.paged import KvCache, PageTable, Rows

    c = st["case"]
    if c["kind"] == "pages":
        o = st["out"]
        return (PageTable(st["table"], st["length"], st["ring"], st["state"], c["page"]),
                PageTable(st["table"], o["length"], st["ring"], o["state"], c["page"]),
                Rows(o["row_start"], o["seq"], o["pos"], o["slot"], o["status"]))
    return KvCache(st["pool"].view(-1), st["table"], n_kv=c["kv_heads"], qd=c["qd"], vd=c["vd"], page=c["page"],
                   means=st.get("means"))


def _run_own(st):
    c = st["case"]
    if "own" not in st:
        st["own"] = _own(st)
    if c["kind"] == "pages":
        now, then, rows = st["own"]
        now.advance(st["add"], rows, out=then)
        return [st["table"], st["ring"], st["out"]]
    cache = st["own"]
    if c["kind"] == "store":
        cache.store(st["k"], st["v"], st["slot"])
        cache.load(st["slot"], st["k_out"], st["v_out"])
        return [st["k_out"], st["v_out"], st["means"]]
    if c["kind"] == "attend":
        cache.attend(st["q"], st["seq"], st["pos"], st["out"], max_pos=st["max_pos"], scale=st["scale"],
                     window=c["window"])
        return [st["out"]]
    cache.select(st["q"], st["seq"], st["pos"], st["lists"], max_pos=st["max_pos"], sinks=c["sinks"],
                 recent=c["recent"])
    cache.attend(st["q"], st["seq"], st["pos"], st["out"], max_pos=st["max_pos"], scale=st["scale"],
                 pages=st["lists"])
    return [st["lists"], st["out"]]


def run(state):
    if own:
        return _run_own(state)
    return {"pages": _plain_pages, "store": _plain_store, "attend": _plain_attend,
            "sparse": _plain_sparse}[state["case"]["kind"]](state)


# ------------------------------------------------------------------- 64 bits


def _exact_read(st, head, pages, keys):
    """Positions of the pages of one kv head in 64 bits, [positions, width], byte by byte from the layout's words."""
    c = st["case"]
    P, kv, qd, vd = c["page"], c["kv_heads"], c["qd"], c["vd"]
    d = qd if keys else vd
    p = torch.arange(P, device=DEV)
    start = ((pages[:, None] * kv + head) * (P // 32) + p // 32) * (18 * (qd + vd))  # [page, position]
    start = start.reshape(-1, 1)
    p = (p % 32).repeat(len(pages))[:, None]
    dim = torch.arange(d, device=DEV)
    block, j = dim // 32, dim % 16
    word = 2 * block + (p >= 16).long()
    lane, byte = (j // 4 * 16 + p % 16, j % 4) if keys else ((p % 16) // 4 * 16 + j, p % 4)
    last = word >= d // 64 * 4  # the short chunk of an odd number of blocks
    at = torch.where(last, d // 64 * 1024 + lane * 8 + (word & 1) * 4, (word >> 2) * 1024 + lane * 16 + (word & 3) * 4)
    flat = st["pool"].view(-1)
    b = flat[start + (0 if keys else 16 * qd) + at + byte].long()
    code = torch.where(dim % 32 < 16, b % 16, b // 16) - 8
    at = start + (16 * (qd + vd) if keys else 18 * qd + 16 * vd) + 2 * (block * 32 + (p % 16) // 4 * 8 + p // 16 * 4 + p % 4)
    return code.double() * st["pool"].view(torch.float16).view(-1)[at // 2].double()


def _exact_rows(st, rows, i, choose):
    """Attention of one sequence's rows; choose(row, kv head) -> its logical pages, or None for all."""
    c = st["case"]
    h, kv, qd, vd, P = (c[k] for k in ("heads", "kv_heads", "qd", "vd", "page"))
    rep, win = h // kv, c.get("window", 0)
    out = torch.zeros((len(rows), h, vd), dtype=torch.float64, device=DEV)
    pos = st["pos"].tolist()
    last = pos[rows[-1]]
    for g in range(kv):
        every = torch.arange(last // P + 1, device=DEV)
        if choose is None:
            k, v = (_exact_read(st, g, st["table"][i, every].long(), keys) for keys in (True, False))
            q = st["q"][rows].view(len(rows), h, qd)[:, g * rep:(g + 1) * rep].double()
            s = torch.einsum("rhd,pd->rhp", q, k) * float(st["scale"])
            at = torch.arange(len(every) * P, device=DEV)
            top = torch.tensor([pos[r] for r in rows], device=DEV)[:, None, None]
            hide = (at > top) | ((at <= top - win) if win else (at < 0))
            out[:, g * rep:(g + 1) * rep] = torch.softmax(s.masked_fill(hide, -math.inf), -1) @ v
            continue
        for a, r in enumerate(rows):
            some = choose(r, g)
            k, v = (_exact_read(st, g, st["table"][i, some].long(), keys) for keys in (True, False))
            at = (some[:, None] * P + torch.arange(P, device=DEV)).reshape(-1)
            s = st["q"][r].view(h, qd)[g * rep:(g + 1) * rep].double() @ k.T * float(st["scale"])
            out[a, g * rep:(g + 1) * rep] = torch.softmax(s.masked_fill(at > pos[r], -math.inf), -1) @ v
    return out.view(len(rows), h * vd)


def exact(case, seed):
    c = dict(case)
    if c["kind"] == "pages":
        return None
    st = prepare(c, seed)
    n, new = c["seqs"], c["new"]
    if c["kind"] == "store":
        got = []
        for x, d in ((st["k"], c["qd"]), (st["v"], c["vd"])):
            # A code is defined with each of its steps rounded to 32 bits (a product or quotient of two 32-bit numbers,
            # rounded once from 64, is that): max / 7, the scale's 16 bits, its reciprocal, the value times it.
            v = x.double().view(len(x), -1, 32)
            h = (v.abs().max(-1, keepdim=True).values / 7).float().half().double()
            y = (v * (1 / h).float().double()).float().double()
            code = torch.where(y < 0, -torch.floor(0.5 - y), torch.floor(y + 0.5))
            got.append((code.clamp(-8, 7) * h).view(len(x), -1))
        means = st["means"].double()
        table, P = st["table"].tolist(), c["page"]
        for i, past in enumerate(_pasts(c)):
            for page in range(past // P, (past + new) // P):  # filled by these rows
                for g in range(c["kv_heads"]):
                    keys = _exact_read(st, g, torch.tensor([table[i][page]], device=DEV), True)
                    lo, hi = max(past, page * P), (page + 1) * P
                    r = i * new + lo - past
                    keys[lo - page * P:] = got[0][r:r + hi - lo].view(hi - lo, -1, c["qd"])[:, g]
                    means[table[i][page], g] = keys.mean(0)
        return [got[0], got[1], means]
    out = torch.zeros_like(st["out"], dtype=torch.float64)
    lists = {}
    if c["kind"] == "sparse":
        h, kv, qd, P = c["heads"], c["kv_heads"], c["qd"], c["page"]
        pos, seq = st["pos"].tolist(), st["seq"].tolist()
        for r in range(n * new):
            last = pos[r] // P
            m = st["means"][st["table"][seq[r], :last + 1].long()].double()
            s = torch.einsum("ghd,pgd->ghp", st["q"][r].view(kv, h // kv, qd).double(), m).max(1).values.cpu()
            for g in range(kv):
                forced = [p for p in range(last + 1) if p < c["sinks"] or p > last - c["recent"]]
                by = sorted((p for p in range(last + 1) if p not in set(forced)), key=lambda p: (-float(s[g, p]), p))
                lists[r, g] = torch.tensor(sorted((forced + by)[:c["select"]]), device=DEV)
    for i in range(n):
        rows = list(range(i * new, (i + 1) * new))
        # The scores of a sequence's rows at once where they fit.
        step = len(rows) if lists else max(1, (1 << 28) // (c["heads"] // c["kv_heads"] * (st["max_pos"] + c["page"])))
        for a in range(0, len(rows), step):
            part = rows[a:a + step]
            out[part] = _exact_rows(st, part, i, (lambda r, g: lists[r, g]) if lists else None)
    return [None, out] if lists else [out]
